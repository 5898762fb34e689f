// kvb_api_prefill.cu - kvb_prefill_attention (include/kvb.h): validation, tensor maps and launch of the causal
// attention of packed prompts (kvb_prefill.cuh).
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "kvb_host.h"
#include "kvb_common.cuh"
#include "kvb_prefill.cuh"

namespace {

constexpr int kMaxCtas = 256;
constexpr size_t kCountBytes = 2 * kMaxCtas * 8 * 4;          // per piece and warp

// Rows of `heads` heads of d 16-bit channels as a 3D tensor (d, heads, rows): box 64 x box_heads x box_rows, 128-byte
// swizzle.
kvb_status make_map(CUtensorMap* m, const char* name, const void* base, int bf16, int d, int heads, int64_t rows,
                    int64_t head_stride, int64_t row_stride, int box_heads, int box_rows) {
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return fail(KVB_ECUDA, "prefill_attention: cuTensorMapEncodeTiled unavailable");
    const cuuint64_t dims[3] = {cuuint64_t(d), cuuint64_t(heads), cuuint64_t(rows)};
    // the stride of a dimension of one entry is never used, but has to be a valid one
    const cuuint64_t strides[2] = {cuuint64_t(heads > 1 ? head_stride : d) * 2, cuuint64_t(rows > 1 ? row_stride : d) * 2};
    const cuuint32_t box[3] = {64, cuuint32_t(box_heads), cuuint32_t(box_rows)};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base),
                          dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(KVB_EINVAL, "prefill_attention: no tensor map for %s (strides %lld, %lld)", name,
                                       static_cast<long long>(head_stride), static_cast<long long>(row_stride));
    return KVB_OK;
}

template <typename T, int D>
kvb_status launch(const kvb::PrefillParams& a, cudaStream_t s) {
    constexpr int SM = kvb::PfShape<D>::SMEM;
    const auto kern = kvb::prefill_kernel<T, D>;
    static std::atomic<uint64_t> done{0};
    if (kvb_status st = kvbh::allow_smem("prefill_attention", reinterpret_cast<const void*>(kern), SM, done)) return st;
    // without pieces no more CTAs than items (at most so many) have work
    const int64_t items = a.part ? kMaxCtas : a.Hkv * (a.nq / (2 * a.tt) + a.n);
    const int ctas = std::min(resolve_ctas(0), kMaxCtas);
    // Launched plainly: the kernel fills an SM, so that placing it early (programmatic serialization) saves the launch's 1 to 2
    // us only.
    kern<<<unsigned(std::min<int64_t>(items, ctas)), kvb::PF_THREADS, SM, s>>>(a);
    return launch_check("prefill_attention");
}

}  // namespace

extern "C" {

size_t kvb_prefill_workspace(int d) {
    return d == 64 || d == 128 ? kCountBytes + size_t(resolve_ctas(0)) * 2 * 2 * (d + 2) * 128 * 4 : 0;
}

kvb_status kvb_prefill_attention(const void* q, const void* k, const void* v, int dtype, int64_t nq, int64_t nk, int Hq,
                                 int Hkv, int d, int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head,
                                 int64_t v_row, int64_t v_head, const int32_t* cu_q, const int32_t* cu_k, int n,
                                 float scaling, void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    if (n < 0 || nq < 0 || nk < 0 || nq > INT32_MAX || nk > INT32_MAX)
        return fail(KVB_EINVAL, "prefill_attention: n >= 0 and row counts in [0, 2^31)");
    if (Hkv <= 0 || Hq <= 0 || Hq % Hkv != 0 || Hq > 65535)
        return fail(KVB_EINVAL, "prefill_attention: Hq a multiple of Hkv, at most 65535");
    if (dtype != KVB_F16 && dtype != KVB_BF16) return fail(KVB_EUNSUPPORTED, "prefill_attention: float16 or bfloat16");
    if (d != 64 && d != 128) return fail(KVB_EUNSUPPORTED, "prefill_attention: d 64 or 128");
    if (Hq / Hkv > 128) return fail(KVB_EUNSUPPORTED, "prefill_attention: at most 128 query heads per KV head");
    if (n == 0 || nq == 0) return KVB_OK;
    if (!q || (!k && nk) || (!v && nk) || !cu_q || !cu_k || !out) return fail(KVB_EINVAL, "prefill_attention: null argument");
    for (int64_t st : {q_row, q_head, k_row, k_head, v_row, v_head})
        if (st < 0 || st % 8 != 0) return fail(KVB_EINVAL, "prefill_attention: row and head strides multiples of 8 elements");
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 32))
        return fail(KVB_EINVAL, "prefill_attention: q, k and v need 16-byte alignment, out 32-byte");
    if (!std::isfinite(scaling)) return fail(KVB_EINVAL, "prefill_attention: scaling must be finite");
    if (workspace && (workspace_bytes < kvb_prefill_workspace(d) || !aligned(workspace, 256)))
        return fail(KVB_EINVAL, "prefill_attention: workspace of %zu bytes, 256-byte aligned (or none)", kvb_prefill_workspace(d));
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    if (kvb_status st = kvbh::cuda_check(cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &capture), "prefill_attention")) return st;
    if (capture != cudaStreamCaptureStatusNone)      // see the head of kvb_prefill.cuh
        return fail(KVB_EUNSUPPORTED, "prefill_attention: not in a stream capture");
    kvb::PrefillParams a{};
    a.count = static_cast<uint32_t*>(workspace);
    a.part = workspace ? reinterpret_cast<float*>(static_cast<char*>(workspace) + kCountBytes) : nullptr;
    a.rep = Hq / Hkv;
    a.tt = 128 / a.rep;
    const int bf16 = dtype == KVB_BF16;
    // without keys nothing is loaded from k and v: their maps then describe q
    const bool none = nk == 0;
    if (kvb_status st = make_map(&a.tm_q, "q", q, bf16, d, Hq, nq, q_head, q_row, a.rep, a.tt)) return st;
    if (kvb_status st = none ? make_map(&a.tm_k, "k", q, bf16, d, Hq, nq, q_head, q_row, 1, 128)
                             : make_map(&a.tm_k, "k", k, bf16, d, Hkv, nk, k_head, k_row, 1, 128)) return st;
    if (kvb_status st = none ? make_map(&a.tm_v, "v", q, bf16, d, Hq, nq, q_head, q_row, 1, 128)
                             : make_map(&a.tm_v, "v", v, bf16, d, Hkv, nk, v_head, v_row, 1, 128)) return st;
    a.v = v;
    a.v_row = v_row;
    a.v_head = v_head;
    a.cu_q = cu_q;
    a.cu_k = cu_k;
    a.nq = nq;
    a.nk = nk;
    a.n = n;
    a.Hq = Hq;
    a.Hkv = Hkv;
    // a scaling of zero becomes one too small to matter, so that -inf stays -inf
    a.lam = std::max(std::fabs(scaling) * 1.44269504088896340736f, 1e-37f);
    a.negate = scaling < 0;
    a.out = out;
    a.lse = lse;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (bf16) return d == 128 ? launch<__nv_bfloat16, 128>(a, s) : launch<__nv_bfloat16, 64>(a, s);
    return d == 128 ? launch<__half, 128>(a, s) : launch<__half, 64>(a, s);
}

}  // extern "C"

KVB_STATUS_WORDS(status_words_prefill)
