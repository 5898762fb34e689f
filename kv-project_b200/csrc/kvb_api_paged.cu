// kvb_api_paged.cu - kvb_page_attend (include/kvb.h): validation, tensor maps and launch of the attention over the
// 8-bit paged cache (kvb_paged_decode.cuh).
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "kvb_host.h"
#include "kvb_pages_host.h"
#include "kvb_paged_decode.cuh"

namespace {

constexpr int64_t kCountBytes = kvb::PD_MAX_CTAS * 8 * 4;      // per warp

// floats of one partial: up to 16 query rows
int64_t part_floats(int d) { return 16 * (int64_t(d) + 6); }

// ceil(2^64 / d) for kvb::pd_div; 0 for 1
uint64_t reciprocal(int d) { return d == 1 ? 0 : UINT64_MAX / uint64_t(d) + 1; }

// Codes as (d, page, n_pages * Hkv) bytes: box d x min(page, 32) x 1, swizzled over the d bytes of a row.
kvb_status make_map(CUtensorMap* m, const kvb_pages* p, const void* codes) {
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return fail(KVB_ECUDA, "page_attend: cuTensorMapEncodeTiled unavailable");
    const cuuint64_t dims[3] = {cuuint64_t(p->d), cuuint64_t(p->page), cuuint64_t(p->n_pages * p->Hkv)};
    const cuuint64_t strides[2] = {cuuint64_t(p->d), cuuint64_t(p->d) * p->page};
    const cuuint32_t box[3] = {cuuint32_t(p->d), cuuint32_t(std::min(p->page, kvb::PD_UNIT)), 1};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(codes), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, p->d == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? KVB_OK : fail(KVB_ECUDA, "page_attend: no tensor map for the codes");
}

template <typename T, int D, int NT>
kvb_status launch(kvb::PagedDecodeParams a, cudaStream_t s) {
    constexpr int SM = kvb::PdShape<D, NT>::SMEM;
    const auto kern = kvb::paged_decode_kernel<T, D, NT>;
    static std::atomic<uint64_t> done{0};
    if (kvb_status st = kvbh::allow_smem("page_attend", reinterpret_cast<const void*>(kern), SM, done)) return st;
    a.by_rep = reciprocal(a.rep);
    a.page_log2 = 31 - __builtin_clz(unsigned(a.P.page));
    const unsigned grid = unsigned(std::min(resolve_ctas(0), kvb::PD_MAX_CTAS));
    // A launch's work has to fit 32 bits whatever the lengths are: fewer sequences, and where one alone can be too much, fewer
    // row groups a launch.
    const int rows = a.rep * a.Tq, groups = (rows + 8 * NT - 1) / (8 * NT);
    const int64_t one = (int64_t(a.P.max_blocks) * a.P.page / kvb::PD_UNIT + 1 + kvb::PD_FIXED) * a.P.Hkv;
    const int per_launch = int(std::max<int64_t>(1, std::min<int64_t>(groups, INT32_MAX / one)));
    const int seqs = int(std::max<int64_t>(1, std::min<int64_t>(kvb::PD_MAX_SEQS, INT32_MAX / (one * per_launch))));
    const int n = a.n;
    const char* q = static_cast<const char*>(a.q);
    char* out = static_cast<char*>(a.out);
    const int64_t per = int64_t(a.Hq) * a.Tq;
    const int32_t* slots = a.slots;
    float* lse = a.lse;
    for (int i = 0; i < n; i += seqs) {
        a.n = std::min(n - i, seqs);
        a.q = q + i * per * D * 2;
        a.out = out + i * per * D * 2;
        a.lse = lse ? lse + i * per : nullptr;
        a.slots = slots + i;
        for (int first = 0; first < groups; first += per_launch) {
            a.groups = std::min(groups - first, per_launch);
            a.by_groups = reciprocal(a.groups);
            a.row0 = first * 8 * NT;
            if (kvb_status st = launch_chained("page_attend", kern, grid, kvb::PdShape<D, NT>::THREADS, SM, s, a)) return st;
        }
    }
    return KVB_OK;
}

// One column group of 8 query rows where they fit, two (the codes' conversion shared by 16 rows) where they do not.
template <typename T, int D>
kvb_status launch_rows(const kvb::PagedDecodeParams& a, cudaStream_t s) {
    return a.rep * a.Tq <= 8 ? launch<T, D, 1>(a, s) : launch<T, D, 2>(a, s);
}

}  // namespace

extern "C" {

size_t kvb_page_attend_workspace(const kvb_pages* p, int n, int Hq, int Tq) {
    if (kvbh::check_pages("page_attend", p) || n < 0 || Hq <= 0 || Tq <= 0) return 0;
    return size_t(kCountBytes + 2 * kvb::PD_MAX_CTAS * part_floats(p->d) * 4);
}

kvb_status kvb_page_attend(const kvb_pages* p, const void* q, int dtype, int Hq, int Tq, const int32_t* slots, int n,
                           float scaling, void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    if (kvb_status st = kvbh::check_pages("page_attend", p)) return st;
    if (n > 0 && (!q || !slots || !out || !workspace)) return fail(KVB_EINVAL, "page_attend: null argument");
    if (Hq <= 0 || Hq % p->Hkv != 0 || Hq > 65535) return fail(KVB_EINVAL, "page_attend: Hq a multiple of Hkv, at most 65535");
    if (n < 0 || Tq <= 0 || Tq > (1 << 20)) return fail(KVB_EINVAL, "page_attend: n >= 0, 1 <= Tq <= 2^20");
    if (int64_t(Hq / p->Hkv) * Tq > INT32_MAX) return fail(KVB_EINVAL, "page_attend: query heads per KV head times Tq below 2^31");
    if (dtype != KVB_F16 && dtype != KVB_BF16) return fail(KVB_EUNSUPPORTED, "page_attend: q of float16 or bfloat16");
    if (!std::isfinite(scaling)) return fail(KVB_EINVAL, "page_attend: scaling must be finite");
    if (p->n_pages * p->Hkv > INT32_MAX) return fail(KVB_EINVAL, "page_attend: n_pages * Hkv < 2^31");
    if (n == 0) return KVB_OK;
    if (!aligned(q, 16) || !aligned(out, 4) || !aligned(lse, 4))
        return fail(KVB_EINVAL, "page_attend: q needs 16-byte alignment, out and lse 4-byte");
    if (workspace_bytes < kvb_page_attend_workspace(p, n, Hq, Tq) || !aligned(workspace, 256))
        return fail(KVB_EINVAL, "page_attend: workspace of %zu bytes, 256-byte aligned", kvb_page_attend_workspace(p, n, Hq, Tq));
    kvb::PagedDecodeParams a{};
    if (kvb_status st = make_map(&a.tm_k, p, p->kc)) return st;
    if (kvb_status st = make_map(&a.tm_v, p, p->vc)) return st;
    a.P = kvbh::view_of(p);
    a.q = q;
    a.slots = slots;
    a.n = n;
    a.Hq = Hq;
    a.Tq = Tq;
    a.rep = Hq / p->Hkv;
    a.lam = scaling * 1.44269504088896340736f;
    a.out = out;
    a.lse = lse;
    a.count = static_cast<uint32_t*>(workspace);
    a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCountBytes);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == KVB_F16) return p->d == 128 ? launch_rows<__half, 128>(a, s) : launch_rows<__half, 64>(a, s);
    return p->d == 128 ? launch_rows<__nv_bfloat16, 128>(a, s) : launch_rows<__nv_bfloat16, 64>(a, s);
}

}  // extern "C"

KVB_STATUS_WORDS(status_words_paged)
