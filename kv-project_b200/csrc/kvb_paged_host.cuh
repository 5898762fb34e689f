// kvb_paged_host.cuh - launching the attention over 8-bit pages (kvb_paged_decode.cuh): tensor maps, workspace layout, how a
// call's work is divided over launches.
#pragma once

#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "kvb_host.h"
#include "kvb_pages_host.h"
#include "kvb_paged_decode.cuh"

namespace kvbh {

constexpr int64_t kCountBytes = kvb::PD_MAX_CTAS * 8 * 4;      // per warp

// floats of one partial: up to 16 query rows
inline int64_t part_floats(int d) { return 16 * (int64_t(d) + 6); }

// ceil(2^64 / d) for kvb::pd_div; 0 for 1
inline uint64_t reciprocal(int d) { return d == 1 ? 0 : UINT64_MAX / uint64_t(d) + 1; }

// Codes as (d, page, n_pages * Hkv) bytes: box d x min(page, tokens) x 1, swizzled over the d bytes of a row or not at all.
inline kvb_status make_map(const char* who, CUtensorMap* m, const kvb_pages* p, const void* codes, int tokens, bool swizzled) {
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return fail(KVB_ECUDA, "%s: cuTensorMapEncodeTiled unavailable", who);
    const cuuint64_t dims[3] = {cuuint64_t(p->d), cuuint64_t(p->page), cuuint64_t(p->n_pages * p->Hkv)};
    const cuuint64_t strides[2] = {cuuint64_t(p->d), cuuint64_t(p->d) * p->page};
    const cuuint32_t box[3] = {cuuint32_t(p->d), cuuint32_t(std::min(p->page, tokens)), 1};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(codes), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, !swizzled ? CU_TENSOR_MAP_SWIZZLE_NONE : p->d == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? KVB_OK : fail(KVB_ECUDA, "%s: no tensor map for the codes", who);
}

template <typename T, int D, int NT, int MODE>
kvb_status paged_launch(const char* who, kvb::PagedDecodeParams a, cudaStream_t s) {
    constexpr int SM = kvb::PdShape<D, NT>::SMEM;
    const auto kern = kvb::paged_decode_kernel<T, D, NT, MODE>;
    static std::atomic<uint64_t> done{0};
    if (kvb_status st = allow_smem(who, reinterpret_cast<const void*>(kern), SM, done)) return st;
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
        a.seq0 = i;
        a.q = q + i * per * D * 2;
        a.out = out + i * per * D * 2;
        a.lse = lse ? lse + i * per : nullptr;
        a.slots = slots + i;
        for (int first = 0; first < groups; first += per_launch) {
            a.groups = std::min(groups - first, per_launch);
            a.by_groups = reciprocal(a.groups);
            a.row0 = first * 8 * NT;
            if (kvb_status st = launch_chained(who, kern, grid, kvb::PdShape<D, NT>::THREADS, SM, s, a)) return st;
        }
    }
    return KVB_OK;
}

// One column group of 8 query rows where they fit (`rows`: the most of a KV head), two (the codes' conversion shared by 16
// rows) where they do not.
template <int MODE>
kvb_status paged_launch_any(const char* who, const kvb::PagedDecodeParams& a, int dtype, int64_t rows, cudaStream_t s) {
    if (dtype == KVB_F16) {
        if (a.P.d == 128) return rows <= 8 ? paged_launch<__half, 128, 1, MODE>(who, a, s) : paged_launch<__half, 128, 2, MODE>(who, a, s);
        return rows <= 8 ? paged_launch<__half, 64, 1, MODE>(who, a, s) : paged_launch<__half, 64, 2, MODE>(who, a, s);
    }
    if (a.P.d == 128) return rows <= 8 ? paged_launch<__nv_bfloat16, 128, 1, MODE>(who, a, s) : paged_launch<__nv_bfloat16, 128, 2, MODE>(who, a, s);
    return rows <= 8 ? paged_launch<__nv_bfloat16, 64, 1, MODE>(who, a, s) : paged_launch<__nv_bfloat16, 64, 2, MODE>(who, a, s);
}

// What both entry points check and fill in; `who` names the caller.
inline kvb_status paged_params(const char* who, const kvb_pages* p, const void* q, int dtype, int Hq, int Tq, const int32_t* slots, int n,
                               float scaling, void* out, float* lse, void* workspace, kvb::PagedDecodeParams& a) {
    if (n > 0 && (!q || !slots || !out || !workspace)) return fail(KVB_EINVAL, "%s: null argument", who);
    if (Hq <= 0 || Hq % p->Hkv != 0 || Hq > 65535) return fail(KVB_EINVAL, "%s: Hq a multiple of Hkv, at most 65535", who);
    if (n < 0 || Tq <= 0 || Tq > (1 << 20)) return fail(KVB_EINVAL, "%s: n >= 0, 1 <= Tq <= 2^20", who);
    if (int64_t(Hq / p->Hkv) * Tq > INT32_MAX) return fail(KVB_EINVAL, "%s: query heads per KV head times Tq below 2^31", who);
    if (dtype != KVB_F16 && dtype != KVB_BF16) return fail(KVB_EUNSUPPORTED, "%s: q of float16 or bfloat16", who);
    if (!std::isfinite(scaling)) return fail(KVB_EINVAL, "%s: scaling must be finite", who);
    if (p->n_pages * p->Hkv > INT32_MAX) return fail(KVB_EINVAL, "%s: n_pages * Hkv < 2^31", who);
    if (n == 0) return KVB_OK;
    if (!aligned(q, 16) || !aligned(out, 4) || !aligned(lse, 4))
        return fail(KVB_EINVAL, "%s: q needs 16-byte alignment, out and lse 4-byte", who);
    a.P = view_of(p);
    a.q = q;
    a.slots = slots;
    a.n = n;
    a.Hq = Hq;
    a.Tq = Tq;
    a.rep = Hq / p->Hkv;
    a.by_rep = reciprocal(a.rep);
    a.page_log2 = 31 - __builtin_clz(unsigned(p->page));
    a.lam = scaling * 1.44269504088896340736f;
    a.out = out;
    a.lse = lse;
    return KVB_OK;
}

inline kvb_status paged_maps(const char* who, const kvb_pages* p, kvb::PagedDecodeParams& a) {
    if (kvb_status st = make_map(who, &a.tm_k, p, p->kc, kvb::PD_UNIT, true)) return st;
    return make_map(who, &a.tm_v, p, p->vc, kvb::PD_UNIT, true);
}

inline void paged_workspace(void* workspace, kvb::PagedDecodeParams& a) {
    a.count = static_cast<uint32_t*>(workspace);
    a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCountBytes);
}

inline size_t paged_part_bytes(int d) { return size_t(kCountBytes + 2 * kvb::PD_MAX_CTAS * part_floats(d) * 4); }

}  // namespace kvbh
