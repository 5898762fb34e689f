// kvb_rowattn.cuh - attention over 8-bit pages one query row at a time, in float32.
//
//   s_j = scaling q . k_j,  m = max s_j,  l = sum e^(s_j - m),  o = sum e^(s_j - m) v_j / l,  lse = m + ln l
//
// over the keys the row sees, in one pass with the running maximum and sum of the softmax (the sums are
// rescaled when the maximum grows).  One warp per (row, query head): a round takes 32 keys, a lane computes
// its own key's product and then owns d / 32 output channels.  A row that sees no key gives zeros and -inf.
#pragma once

#include "kvb_common.cuh"
#include "kvb_pages_view.cuh"

namespace kvb {

constexpr int RA_WARPS = 4;

// keys: row(j, c) and value(j, c) as floats, j below `n`
template <int D, typename Keys>
__device__ __forceinline__ void row_attention(const float* q, const Keys& keys, int n, float lam, float (&o)[D / 32], float& m,
                                              float& l) {
    const int lane = threadIdx.x & 31;
    constexpr int C = D / 32;
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] = 0.f;
    for (int j0 = 0; j0 < n; j0 += 32) {
        const int j = j0 + lane;
        float s = -INFINITY;
        if (j < n) {
            s = 0.f;
            for (int c = 0; c < D; ++c) s = __fmaf_rn(q[c], keys.k(j, c), s);
            s *= lam;
        }
        const float mn = fmaxf(m, warp_max(s));
        const float ref = mn == -INFINITY ? 0.f : mn;      // every logit so far is -inf
        const float f = m == -INFINITY ? 1.f : exp2f(m - ref);
        const float p = j < n ? exp2f(s - ref) : 0.f;
        l = l * f + warp_sum(p);
        m = mn;
#pragma unroll
        for (int c = 0; c < C; ++c) o[c] *= f;
        for (int i = 0; i < min(32, n - j0); ++i) {
            const float pi = __shfl_sync(0xffffffffu, p, i);
#pragma unroll
            for (int c = 0; c < C; ++c) o[c] = __fmaf_rn(pi, keys.v(j0 + i, lane * C + c), o[c]);
        }
    }
}

constexpr float RA_LN2 = 0.693147180559945309f;

template <typename T, int D>
__device__ __forceinline__ void store_row(const float (&o)[D / 32], float m, float l, T* out, float* lse) {
    const int lane = threadIdx.x & 31;
    const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) out[lane * (D / 32) + c] = from_f32<T>(o[c] * inv);
    if (lse && lane == 0) *lse = l == 0.f ? -INFINITY : m * RA_LN2 + logf(l);
}

struct PagedAttendParams {
    PagesView P;
    const void* q;                 // (n, Hq, Tq, d)
    const int32_t* slots;
    int n, Hq, Tq;
    float lam;
    void* out;                     // (n, Tq, Hq, d)
    float* lse;                    // (n, Tq, Hq) or null
};

struct PagedKeys {
    const PagesView& P;
    const int32_t* row;
    int h;
    __device__ __forceinline__ float at(const uint8_t* codes, const float* scales, int j, int c) const {
        const int64_t ph = int64_t(row[j / P.page]) * P.Hkv + h;
        return float(int(codes[(ph * P.page + j % P.page) * P.d + c]) - 128) * scales[ph];
    }
    __device__ __forceinline__ float k(int j, int c) const { return at(P.kc, P.ks, j, c); }
    __device__ __forceinline__ float v(int j, int c) const { return at(P.vc, P.vs, j, c); }
};

// grid (ceil(n Tq / RA_WARPS), Hq)
template <typename T, int D>
__global__ void __launch_bounds__(RA_WARPS * 32) paged_rows_kernel(const __grid_constant__ PagedAttendParams A) {
    __shared__ float sq[RA_WARPS][D];
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, hq = blockIdx.y;
    const int64_t r = int64_t(blockIdx.x) * RA_WARPS + w;
    if (r >= int64_t(A.n) * A.Tq) return;
    const int i = int(r / A.Tq), t = int(r % A.Tq), slot = A.slots[i];
    if (slot < 0 || slot >= A.P.n_slots) {
        if (lane == 0) raise_status(KVB_DEV_BOUNDS);
        return;
    }
    const T* q = static_cast<const T*>(A.q) + ((int64_t(i) * A.Hq + hq) * A.Tq + t) * D;
    for (int c = lane; c < D; c += 32) sq[w][c] = to_f32(q[c]);
    __syncwarp();
    const int seen = max(0, min(A.P.lens[slot], A.P.max_blocks * A.P.page) - A.Tq + t + 1);
    const PagedKeys keys{A.P, A.P.table + int64_t(slot) * A.P.max_blocks, hq / (A.Hq / A.P.Hkv)};
    bool bad = false;
    for (int b = lane; b < blocks_of(seen, A.P.page); b += 32) bad |= keys.row[b] < 0 || keys.row[b] >= A.P.n_pages;
    if (__any_sync(0xffffffffu, bad)) {
        if (lane == 0) raise_status(KVB_DEV_BOUNDS);
        return;
    }
    float o[D / 32], m, l;
    row_attention<D>(sq[w], keys, seen, A.lam, o, m, l);
    store_row<T, D>(o, m, l, static_cast<T*>(A.out) + (r * A.Hq + hq) * D, A.lse ? A.lse + r * A.Hq + hq : nullptr);
}

}  // namespace kvb
