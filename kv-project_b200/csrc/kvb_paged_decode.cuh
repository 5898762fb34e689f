// kvb_paged_decode.cuh - attention of a few queries per sequence over the 8-bit paged cache.
//
//   s_j = lam q . (kc_j - 128) ks,  o = sum_j 2^(s_j - m) (vc_j - 128) vs / l,  l = sum_j 2^(s_j - m)
//
// with lam = scaling log2(e), over the keys that the query sees (query t of Tq: j <= len - Tq + t).
//
// The floor is the codes read once: 2 d bytes per token and KV head.  One persistent CTA per SM; a unit of work is
// 32 tokens of one (sequence, KV head, row group), and every CTA takes an equal run of units in (sequence, head,
// group, token) order, found from the lengths inside the kernel: any mixture of lengths is balanced, nothing is
// planned before the launch.  Units go to the eight warps in turn; each warp copies its own units' codes with TMA through
// its own ring (192 KB in flight per SM at d = 128, about 4 us of its share of the bandwidth; one warp copying for all
// was slower than the copies: 178 us for 537 MB without any arithmetic) and keeps its own running softmax.  Page numbers
// and scales are fetched 32 units ahead, a lane a unit.  At the end of a run the warps' states are joined in shared
// memory; a run that is only a part of a (sequence, head, group) leaves a partial, and the CTA that completes the last
// part joins the partials in the order of the tokens (each warp its rows), so the result does not depend on timing.
//
// A step of 8 sequences of 32768 tokens, 8 heads, d 128 (537 MB), with the write of its rows: 97 us in a loop, 5.5 TB/s;
// about 7 TB/s at the margin, the rest is the start (4 us), the first copies' latency and the join.  At 8 x 16384 (269 MB,
// all of the DRAM traffic): ALU pipe 39 % busy (the codes' permutes), tensor pipe 17 %, issue slots 41 %, no bank conflicts
// in the loads.
//
// Per 16 tokens, with the query rows (rep heads x Tq queries, 8 per MMA column group) as the N operand:
//   S (tokens x rows) = K Q^T: a code byte becomes the fp16 pattern 0x6400 | byte = 1024 + code (one byte permute per
//     two codes), less 1152: exact operands.  The sums begin at -1152 sum q, so they are rounded at its size where a
//     query's entries have one sign.  The channels are dealt to the lanes so that a lane reads 16-byte pieces of a row;
//     with the 128-byte (64-byte for d = 64) swizzle these reads meet no bank twice.
//   l takes p = 2^(s - m); the weight of the value product is w = 2^(s + log2 vs - mw), the value scale in the exponent, with
//     a reference of its own, so that pages whose scales lie far apart lose neither mass nor values (a page of zeros has
//     log2 vs = -inf: mass, no values).  The references are only raised when passed by 2^8; out = 2^(mw - m) O / l.
//   O^T (channels x rows) += V^T W^T: the tokens of a lane's codes are interleaved by byte permutes, W goes through
//     movmatrix and is rounded to fp16 (2^-11; it is the MMA's operand type).
// Queries are scaled by a power of two per row, their largest entry to [8, 16), before they become fp16: entries down to
// 2^-20 of it (bfloat16; float16 2^-17) are exact, those below lose bits to the subnormal range and are gone at 2^-28.
#pragma once
#include <cuda.h>

#include <climits>

#include "kvb_common.cuh"
#include "kvb_pages_view.cuh"

namespace kvb {

constexpr int PD_UNIT = 32;                   // tokens
constexpr int PD_MAX_SEQS = 512;              // sequences of one launch (their offsets are in shared memory)
constexpr int PD_MAX_CTAS = 256;
// what a (sequence, head, group) costs beside its units, in units: 48 ragged sequences take 123 us with 6, 88 with 12, 70
// with 16 to 32
constexpr int PD_FIXED = 16;
constexpr int PD_LEAST = 4;                   // a CTA's least share
constexpr float PD_LAZY = 8.f;

struct PagedDecodeParams {
    CUtensorMap tm_k, tm_v;                   // codes as (d, page, n_pages * Hkv), box d x min(page, 32) x 1
    PagesView P;
    const void* q;                            // (n, Hq, Tq, d)
    const int32_t* slots;
    int n, Hq, Tq, rep, groups;               // groups of 8 NT query rows per (sequence, KV head), from the row row0 on
    int row0;
    uint64_t by_rep, by_groups;               // for pd_div
    int page_log2;
    float lam;
    void* out;                                // (n, Tq, Hq, d)
    float* lse;                               // (n, Tq, Hq) or null
    float* part;                              // [2 grid][8 NT x (6 + d)]
    uint32_t* count;                          // [grid][8 warps]
};

template <int D, int NT>
struct PdShape {
    static constexpr int WARPS = 8;                             // 12 with two stages each: 104 against 103 us (8 x 32768), 109 against 89 (ragged)
    static constexpr int THREADS = 32 * WARPS;
    static constexpr int ROWS = 8 * NT;
    static constexpr int SIDE = PD_UNIT * D;                    // bytes of one side of a unit
    static constexpr int STAGE = 2 * SIDE;
    static constexpr int STAGES = 3 * (128 / D);             // per warp
    static constexpr int JOIN = WARPS * 8 * (64 + 4) * 4;    // the warps' O rows, 8 query rows and 64 channels at a time
    static constexpr int PAIRS = NT * (D / 64);              // (row, 64 channels) that a warp joins
    static constexpr int PART = ROWS * (D + 6);              // m, l, mw of the rows, twice (see the joining), then O
    static constexpr int SMEM = 1024 + WARPS * STAGES * STAGE + JOIN;
};

// The work of a call: per (sequence, KV head, row group) its units, and PD_FIXED more in the shares that the CTAs get
// (preparing the queries and joining the warps costs about as much time as that many units).
struct PdPlan {
    const int* pre;                           // [n + 1] units before each sequence, for one head and group
    int n, hg;                                // sequences; KV heads x groups
    int quota, extra, ctas;                   // shares: the first `extra` CTAs get quota + 1

    __device__ __forceinline__ int share(int c) const { return c * quota + min(c, extra); }
    __device__ __forceinline__ int holder(int v) const {
        const int big = extra * (quota + 1);
        return v < big ? v / (quota + 1) : extra + (v - big) / quota;
    }
    // units before the place `v` of the shares
    __device__ __forceinline__ int units_before(int v) const {
        int lo = 0, hi = n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if ((pre[mid] + mid * PD_FIXED) * hg <= v) lo = mid;
            else hi = mid;
        }
        const int u = pre[lo + 1] - pre[lo], local = v - (pre[lo] + lo * PD_FIXED) * hg, vh = min(local / (u + PD_FIXED), hg);
        return pre[lo] * hg + vh * u + max(local - vh * (u + PD_FIXED) - PD_FIXED, 0);
    }
};

struct PdPiece {
    int seq, vh, a, b, units;                 // sequence, head * groups + group, unit range, units of the sequence
    int v0;                                   // where the (sequence, head, group) begins in the shares
};

// The piece that begins at unit `cur` of all work.
__device__ __forceinline__ PdPiece pd_piece(const PdPlan& W, int cur, int end) {
    int lo = 0, hi = W.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (W.pre[mid] * W.hg <= cur) lo = mid;
        else hi = mid;
    }
    PdPiece p;
    p.seq = lo;
    p.units = W.pre[lo + 1] - W.pre[lo];
    const int local = cur - W.pre[lo] * W.hg;
    p.vh = local / p.units;
    p.a = local - p.vh * p.units;
    p.b = min(p.units, p.a + (end - cur));
    p.v0 = (W.pre[lo] + lo * PD_FIXED) * W.hg + p.vh * (p.units + PD_FIXED);
    return p;
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ uint32_t pd_prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

// bytes -> two fp16 values 1024 + code
template <uint32_t SEL>
__device__ __forceinline__ uint32_t pd_raw2(uint32_t w) { return pd_prmt(w, 0x64646464u, SEL); }

// bytes -> two fp16 values code - 128 (exact)
template <uint32_t SEL>
__device__ __forceinline__ uint32_t pd_half2(uint32_t w) {
    const uint32_t x = pd_raw2<SEL>(w);
    uint32_t y;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0x64806480u));      // 1152
    return y;
}

template <typename T>
__device__ __forceinline__ float2 pd_pair(uint32_t w);
template <>
__device__ __forceinline__ float2 pd_pair<__half>(uint32_t w) { return unpack_half2(w); }
template <>
__device__ __forceinline__ float2 pd_pair<__nv_bfloat16>(uint32_t w) {
    return float2{__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
}

// log2 of a float32 power of two scale that brings |x| <= amax into [8, 16); 0 for 0
__device__ __forceinline__ int pd_exponent(float amax) {
    const int e = int(__float_as_uint(amax) >> 23) & 255;
    return amax > 0.f ? min(3 - (e - 127), 126) : 0;
}

// n / d for by = ceil(2^64 / d), 0 for d = 1.  The kernel's parts run once or twice a call, so what their instructions cost
// is mostly their number: a division by a variable is 20 and more.
__device__ __forceinline__ int pd_div(int n, uint64_t by) { return by ? int(__umul64hi(uint64_t(uint32_t(n)), by)) : n; }

template <typename T, int D, int NT>
__global__ void __launch_bounds__(PdShape<D, NT>::THREADS, 1) paged_decode_kernel(const __grid_constant__ PagedDecodeParams A) {
    using S = PdShape<D, NT>;
    constexpr int KS = D / 16;                                   // MMA steps over the channels, and channel tiles
    extern __shared__ uint8_t pd_raw[];
    __shared__ int pre[PD_MAX_SEQS + 1], s_slot[PD_MAX_SEQS], s_len[PD_MAX_SEQS];
    __shared__ uint64_t full[S::WARPS][S::STAGES];
    __shared__ float s_m[S::WARPS][S::ROWS], s_l[S::WARPS][S::ROWS], s_w[S::WARPS][S::ROWS];
    __shared__ int warp_sum[S::WARPS];
    __shared__ int s_abort;
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pd_raw) + 1023) & ~uintptr_t(1023));
    float* join = reinterpret_cast<float*>(base + S::WARPS * S::STAGES * S::STAGE);      // [warp][8 rows][64 + 4]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t* ring = base + warp * S::STAGES * S::STAGE;
    const PagesView& P = A.P;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::WARPS * S::STAGES; ++i) mbar_init(&full[0][i], 1);
        s_abort = 0;
        fence_mbar_init();
        pre[0] = 0;
    }
    chain_kernels();
    // units before each sequence: an inclusive scan, S::THREADS sequences at a time; an empty sequence is one unit
    // without keys, whose rows still have to be written
    int before = 0;
    for (int i0 = 0; i0 < A.n; i0 += S::THREADS) {
        const int i = i0 + threadIdx.x;
        int u = 0;
        if (i < A.n) {
            const int slot = A.slots[i];
            int len = 0;
            if (slot >= 0 && slot < P.n_slots) len = min(max(P.lens[slot], 0), P.max_blocks * P.page);
            else raise_status(KVB_DEV_BOUNDS);
            s_slot[i] = slot;
            s_len[i] = len;
            u = max(1, (len + PD_UNIT - 1) / PD_UNIT);
        }
        int x = u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 31) warp_sum[warp] = x;
        __syncthreads();
        int sum = 0;
        for (int w = 0; w < S::WARPS; ++w) {
            if (w == warp) x += sum;
            sum += warp_sum[w];
        }
        if (i < A.n) pre[i + 1] = before + x;
        before += sum;
    }
    __syncthreads();
    PdPlan W;
    W.pre = pre;
    W.n = A.n;
    W.hg = P.Hkv * A.groups;
    const int64_t work = (int64_t(pre[A.n]) + int64_t(A.n) * PD_FIXED) * W.hg;
    if (work > INT_MAX) {                                        // the host's launches hold less, but for one group of 2^31 units
        if (threadIdx.x == 0) raise_status(KVB_DEV_BOUNDS);
        return;
    }
    W.ctas = max(1, min(int(gridDim.x), int(work) / PD_LEAST));
    W.quota = int(work) / W.ctas;
    W.extra = int(work) - W.quota * W.ctas;
    const int cta = blockIdx.x;
    if (cta >= W.ctas) return;
    const int u0 = W.units_before(W.share(cta)), u1 = W.units_before(W.share(cta + 1));
    volatile int* abort = &s_abort;
    auto wait = [&](uint64_t* bar, uint32_t count) {
        if (*abort) return false;
        if (mbar_wait(bar, count & 1)) return true;
        *abort = 1;
        return false;
    };

    auto row_at = [&](int seq, int h, int r) {
        const int tok = pd_div(r, A.by_rep);
        return (int64_t(seq) * A.Tq + tok) * A.Hq + h * A.rep + r - tok * A.rep;
    };
    auto finite_ref = [](float m) { return m == -INFINITY ? 0.f : m; };
    // 2^(mw - m) / l; rows that see nothing give 0, NaN stays
    auto scale_of = [&](float m, float mw, float sum) { return sum > 0.f ? ex2(mw - finite_ref(m)) / sum : (sum == sum ? 0.f : sum); };
    auto store_pair = [&](int64_t row, int ch, float a, float b, float inv) {
        *reinterpret_cast<uint32_t*>(static_cast<T*>(A.out) + row * D + ch) = pack_f32<T>(a * inv, b * inv);
    };
    auto store_lse = [&](int64_t row, float top, float sum) {
        if (A.lse) A.lse[row] = sum == 0.f ? -INFINITY : top * 0.693147180559945309f + logf(sum);
    };

    // the query rows of a piece: lane (g, t) holds row g of 8, channels (D / 4) t ..
    const int g = lane >> 2, t = lane & 3;
    uint4 raw[NT][KS / 2];
    auto load_q = [&](const PdPiece& p) {
        const int h = pd_div(p.vh, A.by_groups), row0 = A.row0 + (p.vh - h * A.groups) * S::ROWS;
#pragma unroll
        for (int x = 0; x < NT; ++x) {
            const int r = row0 + 8 * x + g, tok = pd_div(r, A.by_rep);
#pragma unroll
            for (int i = 0; i < KS / 2; ++i) raw[x][i] = uint4{0, 0, 0, 0};
            if (r < A.rep * A.Tq) {
                const T* q = static_cast<const T*>(A.q) + ((int64_t(p.seq) * A.Hq + h * A.rep + r - tok * A.rep) * A.Tq + tok) * D + (D / 4) * t;
#pragma unroll
                for (int i = 0; i < KS / 2; ++i) raw[x][i] = __ldg(reinterpret_cast<const uint4*>(q + 8 * i));
            }
        }
    };
    PdPiece p{};
    if (u0 < u1) {
        p = pd_piece(W, u0, u1);
        load_q(p);
    }

    // ---------------- copies: the warp's unit k is the CTA's unit warp + S::WARPS k; lane i looks after the units k = i mod 32 ----------------
    struct Place {
        int row[2], off;                                         // rows of the tensor maps (< 0: nothing there), token in the page
    };
    const int box = min(P.page, PD_UNIT);
    const int mine = max(0, (u1 - u0 - warp + S::WARPS - 1) / S::WARPS);                 // units of this warp
    auto place = [&](int k) {
        Place x{{-1, -1}, 0};
        if (k >= mine) return x;
        const PdPiece p = pd_piece(W, u0 + warp + k * S::WARPS, u1);
        const int h = pd_div(p.vh, A.by_groups), t0 = p.a * PD_UNIT, len = s_len[p.seq];
        x.off = t0 & (P.page - 1);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (i * box >= PD_UNIT || t0 + i * box >= len) continue;
            const int id = P.table[int64_t(s_slot[p.seq]) * P.max_blocks + ((t0 + i * box) >> A.page_log2)];
            if (id >= 0 && id < P.n_pages) x.row[i] = id * P.Hkv + h;
            else raise_status(KVB_DEV_BOUNDS);
        }
        return x;
    };
    auto scales_of = [&](const Place& x) {                       // ks and vs of the tokens 0 .. and 16 ..; ks < 0: no page
        float4 f{-1.f, -1.f, 0.f, 0.f};
        if (x.row[0] >= 0) {
            f.x = P.ks[x.row[0]], f.z = P.vs[x.row[0]];
            if (box == PD_UNIT) f.y = f.x, f.w = f.z;
        }
        if (x.row[1] >= 0) f.y = P.ks[x.row[1]], f.w = P.vs[x.row[1]];
        return f;
    };
    auto log_scale = [](float v) { return v > 0.f ? __log2f(v) : -INFINITY; };
    Place at = place(lane), ahead{};                             // of the units being copied, and of the 32 after
    float4 sc_now{0.f, 0.f, 0.f, 0.f}, sc_next{0.f, 0.f, 0.f, 0.f};      // ks, log2 vs of the units being computed; scales of the next
    int copied = 0;
    auto copy = [&]() {                                          // the warp's next unit
        if (copied >= mine) return;
        if ((copied & 31) == 0 && copied > 0) at = ahead;
        if (lane == (copied & 31)) {
            const int st = copied % S::STAGES;
            uint64_t* bar = &full[warp][st];
            mbar_arrive_expect_tx(bar, uint32_t((at.row[0] >= 0) + (at.row[1] >= 0)) * 2 * box * D);
            uint8_t* dst = ring + st * S::STAGE;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (at.row[i] >= 0) {
                    tma_load_3d(dst + i * box * D, &A.tm_k, 0, at.off, at.row[i], bar);
                    tma_load_3d(dst + S::SIDE + i * box * D, &A.tm_v, 0, at.off, at.row[i], bar);
                }
        }
        if ((copied & 31) == 0) {                                // needed a unit or more later
            sc_next = scales_of(at);
            ahead = place(copied + 32 + lane);
        }
        ++copied;
    };
    for (int i = 0; i < S::STAGES; ++i) copy();
    {
        int first = 1, unit = 0;
        for (int cur = u0; cur < u1;) {
            const int h = pd_div(p.vh, A.by_groups), row0 = A.row0 + (p.vh - h * A.groups) * S::ROWS, len = s_len[p.seq];
            const int nrows = min(A.rep * A.Tq - row0, S::ROWS);
            // ---- the group's query rows as B operands
            uint32_t qf[NT][KS][2];
            float lam[NT][2], bias[NT][2];                       // bias: -1152 sum q, what the codes' pattern adds
#pragma unroll
            for (int x = 0; x < NT; ++x) {
                float amax = 0.f;
#pragma unroll
                for (int i = 0; i < KS / 2; ++i) {
                    const uint32_t ws[4] = {raw[x][i].x, raw[x][i].y, raw[x][i].z, raw[x][i].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float2 f = pd_pair<T>(ws[k]);
                        amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
                    }
                }
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                const int e = pd_exponent(amax);
                const float up = __uint_as_float(uint32_t(127 + e) << 23);
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < KS / 2; ++i) {
                    const uint32_t ws[4] = {raw[x][i].x, raw[x][i].y, raw[x][i].z, raw[x][i].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float2 f = pd_pair<T>(ws[k]);
                        const uint32_t qh = pack_half2(f.x * up, f.y * up);
                        qf[x][2 * i + (k >> 1)][k & 1] = qh;
                        const float2 r = unpack_half2(qh);
                        sum += r.x + r.y;
                    }
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                const float down = A.lam * __uint_as_float(uint32_t(127 - e) << 23);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    lam[x][k] = __shfl_sync(0xffffffffu, down, 4 * (2 * t + k));
                    bias[x][k] = -1152.f * __shfl_sync(0xffffffffu, sum, 4 * (2 * t + k));
                }
            }
            float o[NT][KS][4], m[NT][2], mw[NT][2], l[NT][2];
#pragma unroll
            for (int x = 0; x < NT; ++x) {
                m[x][0] = m[x][1] = mw[x][0] = mw[x][1] = -INFINITY;
                l[x][0] = l[x][1] = 0.f;
#pragma unroll
                for (int c = 0; c < KS; ++c) o[x][c][0] = o[x][c][1] = o[x][c][2] = o[x][c][3] = 0.f;
            }
            // the first unit of the piece that is this warp's (units go to the warps in turn over the CTA's whole run)
            const int lead = (cur - u0) % S::WARPS;
            for (int k = warp < lead ? warp - lead + S::WARPS : warp - lead; k < p.b - p.a; k += S::WARPS, ++unit) {
                const int st = unit % S::STAGES;
                if (!__all_sync(0xffffffffu, wait(&full[warp][st], unit / S::STAGES))) continue;
                if ((unit & 31) == 0) sc_now = float4{sc_next.x, sc_next.y, log_scale(sc_next.z), log_scale(sc_next.w)};
                const int src = unit & 31;
                const float ks[2] = {__shfl_sync(0xffffffffu, sc_now.x, src), __shfl_sync(0xffffffffu, sc_now.y, src)};
                const float lv[2] = {__shfl_sync(0xffffffffu, sc_now.z, src), __shfl_sync(0xffffffffu, sc_now.w, src)};
                const int t0 = (p.a + k) * PD_UNIT;
                const uint8_t* kt = ring + st * S::STAGE;
                const bool edge = t0 + PD_UNIT > len - A.Tq + 1;
                // ---- S = K Q^T for the two halves of 16 tokens; past the sequence's end the codes are whatever the page
                // holds (any byte is a finite value) and are masked below
                float s[2][NT][4];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float s2[2][NT][4];                          // two chains of MMAs
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int x = 0; x < NT; ++x)
#pragma unroll
                            for (int i = 0; i < 4; ++i) s2[c][x][i] = c ? 0.f : bias[x][i & 1];
#pragma unroll
                    for (int c = 0; c < D / 64; ++c) {
                        uint4 a, b;
                        if (D == 128) {
                            const int ch = ((2 * t + c) ^ g) * 16;
                            a = *reinterpret_cast<const uint4*>(kt + (16 * half + g) * 128 + ch);
                            b = *reinterpret_cast<const uint4*>(kt + (16 * half + g + 8) * 128 + ch);
                        } else {
                            const int ch = (t ^ ((g >> 1) & 3)) * 16;
                            a = *reinterpret_cast<const uint4*>(kt + (16 * half + g) * 64 + ch);
                            b = *reinterpret_cast<const uint4*>(kt + (16 * half + g + 8) * 64 + ch);
                        }
                        const uint32_t wa[4] = {a.x, a.y, a.z, a.w}, wb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t f[4] = {pd_raw2<0x4140>(wa[i]), pd_raw2<0x4140>(wb[i]), pd_raw2<0x4342>(wa[i]),
                                                   pd_raw2<0x4342>(wb[i])};
#pragma unroll
                            for (int x = 0; x < NT; ++x) mma16816(s2[i & 1][x], f, qf[x][4 * c + i][0], qf[x][4 * c + i][1]);
                        }
                    }
#pragma unroll
                    for (int x = 0; x < NT; ++x)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[half][x][i] = s2[0][x][i] + s2[1][x][i];
                }
                // ---- weights; lane (g, t) holds tokens g, g + 8 and rows 2t, 2t + 1 of either half
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float off = ks[half] < 0.f ? -INFINITY : 0.f;          // tokens without a page are left out
#pragma unroll
                    for (int x = 0; x < NT; ++x)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[half][x][i] = __fmaf_rn(s[half][x][i], lam[x][i & 1] * ks[half], off);
                }
                if (edge) {
#pragma unroll
                    for (int x = 0; x < NT; ++x)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            // keys from this unit on that the row 2t + k sees
                            const int lim = len - A.Tq + pd_div(row0 + 8 * x + 2 * t + k, A.by_rep) + 1 - t0;
#pragma unroll
                            for (int half = 0; half < 2; ++half)
#pragma unroll
                                for (int i = k; i < 4; i += 2)
                                    if (16 * half + g + 8 * (i >> 1) >= lim) s[half][x][i] = -INFINITY;
                        }
                }
                bool grow = false;
                float top[NT][2], topw[NT][2];
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float a = fmaxf(s[0][x][i], s[0][x][i + 2]), b = fmaxf(s[1][x][i], s[1][x][i + 2]);
                        top[x][i] = fmaxf(a, b);
                        topw[x][i] = fmaxf(a + lv[0], b + lv[1]);
                        grow |= top[x][i] > m[x][i] + PD_LAZY || topw[x][i] > mw[x][i] + PD_LAZY;
                    }
                if (__any_sync(0xffffffffu, grow)) {
                    auto quad_max = [](float y) {                // over the lanes of a row
                        y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 4));
                        y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 8));
                        return fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 16));
                    };
#pragma unroll
                    for (int x = 0; x < NT; ++x)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float y = quad_max(top[x][i]), yw = quad_max(topw[x][i]);
                            if (y > m[x][i] + PD_LAZY) {
                                l[x][i] *= ex2(m[x][i] - y);
                                m[x][i] = y;
                            }
                            if (yw > mw[x][i] + PD_LAZY) {
                                const float f = ex2(mw[x][i] - yw);
                                mw[x][i] = yw;
#pragma unroll
                                for (int c = 0; c < KS; ++c) {
                                    o[x][c][i] *= f;
                                    o[x][c][2 + i] *= f;
                                }
                            }
                        }
                }
                uint32_t wf[2][NT][2];
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    // w = p 2^e; e from the references' difference, which is the final factor's too, so that roundings of large
                    // logits cancel
                    const float r[2] = {finite_ref(m[x][0]), finite_ref(m[x][1])};
                    const float dr[2] = {r[0] - finite_ref(mw[x][0]), r[1] - finite_ref(mw[x][1])};
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const float e[2] = {lv[half] + dr[0], lv[half] + dr[1]};
                        float w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float u = s[half][x][i] - r[i & 1];
                            w[i] = ex2(u + e[i & 1]);
                            l[x][i & 1] += ex2(u);
                        }
                        wf[half][x][0] = movmatrix_trans(pack_half2(w[0], w[1]));
                        wf[half][x][1] = movmatrix_trans(pack_half2(w[2], w[3]));
                    }
                }
                // ---- O^T += V^T W^T: lane (g, t) holds channels (D / 8) g .. of the tokens 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint8_t* vt = kt + S::SIDE + half * 16 * D;
                    uint32_t wv[4][D / 32];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int tok = 2 * t + (i & 1) + 8 * (i >> 1);
                        if (D == 128) {
                            const uint4 x = *reinterpret_cast<const uint4*>(vt + tok * 128 + ((g ^ (tok & 7)) * 16));
                            wv[i][0] = x.x, wv[i][1] = x.y, wv[i][D / 32 - 2] = x.z, wv[i][D / 32 - 1] = x.w;
                        } else {
                            const uint2 x = *reinterpret_cast<const uint2*>(vt + tok * 64 + (((g >> 1) ^ ((tok >> 1) & 3)) * 16) + (g & 1) * 8);
                            wv[i][0] = x.x, wv[i][1] = x.y;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            const uint32_t sel = b ? 0x7362u : 0x5140u;
                            const uint32_t lo = pd_prmt(wv[0][i], wv[1][i], sel), hi = pd_prmt(wv[2][i], wv[3][i], sel);
                            const uint32_t f[4] = {pd_half2<0x4140>(lo), pd_half2<0x4342>(lo), pd_half2<0x4140>(hi), pd_half2<0x4342>(hi)};
#pragma unroll
                            for (int x = 0; x < NT; ++x) mma16816(o[x][2 * i + b], f, wf[half][x][0], wf[half][x][1]);
                        }
                    }
                }
                __syncwarp();                                    // every lane has read the stage: refill it
                copy();
            }
            const int next = cur + p.b - p.a;
            PdPiece pn{};
            if (next < u1) {                                     // the next piece's queries arrive during the joining
                pn = pd_piece(W, next, u1);
                load_q(pn);
            }
            // ---- join the warps.  Warp w joins the rows w and 8 + w, 64 channels at a time; where there are at most four
            // rows of 128 channels, row w % 4 and the half w / 4 of its channels, all at once.  Column c of the buffer is
            // channel (D / 8) (c / 8) + 8 y + c % 8 of the half y.
            const bool few = D == 128 && NT == 1 && nrows <= 4;
            const bool whole = p.a == 0 && p.b == p.units;
            // the CTAs c0 .. c1 hold its units
            const int c0 = whole ? 0 : W.holder(p.v0 + PD_FIXED), c1 = whole ? 0 : W.holder(p.v0 + PD_FIXED + p.units - 1);
            if (!first) asm volatile("bar.sync 1, %0;" ::"n"(32 * S::WARPS) : "memory");       // the last join's reads are done
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float v = l[x][k];
                    v += __shfl_xor_sync(0xffffffffu, v, 4);
                    v += __shfl_xor_sync(0xffffffffu, v, 8);
                    v += __shfl_xor_sync(0xffffffffu, v, 16);
                    if (g == 0) {
                        s_m[warp][8 * x + 2 * t + k] = m[x][k];
                        s_l[warp][8 * x + 2 * t + k] = v;
                        s_w[warp][8 * x + 2 * t + k] = mw[x][k];
                    }
                }
            float* part = A.part + int64_t(2 * blockIdx.x + (first ? 0 : 1)) * S::PART;
            const int ml = few ? warp >> 2 : 0;                  // which copy of m, l and mw
            const bool used = (few ? warp & 3 : warp) < nrows;
            auto row_of = [&](int x) { return few ? warp & 3 : 8 * x + warp; };
            auto channel_of = [&](int y) { return (D / 8) * (lane >> 2) + 8 * (few ? warp >> 2 : y) + 2 * (lane & 3); };
            auto put = [&](int x, int y, int slot) {             // O of the rows 2t, 2t + 1, half y
                float* to = join + warp * 8 * 68 + slot * 68 + 8 * g;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    *reinterpret_cast<float2*>(to + 2 * c) = float2{o[x][4 * y + c][0], o[x][4 * y + c][2]};
                    *reinterpret_cast<float2*>(to + 68 + 2 * c) = float2{o[x][4 * y + c][1], o[x][4 * y + c][3]};
                }
            };
#pragma unroll
            for (int x = 0; x < NT; ++x) {
                const int r = row_of(x);
                const int64_t row = whole ? row_at(p.seq, h, row0 + r) : 0;
                float top = -INFINITY, topw = -INFINITY, sum = 0.f, inv = 0.f, f[S::WARPS];
#pragma unroll
                for (int y = 0; y < D / 64; ++y) {
                    if (few && y > 0) break;
                    if (x + y > 0) asm volatile("bar.sync 1, %0;" ::"n"(32 * S::WARPS) : "memory");
                    if (!few) put(x, y, 2 * t);
                    else if (t < 2)
#pragma unroll
                        for (int k = 0; k < D / 64; ++k) put(x, k, 4 * k + 2 * t);
                    asm volatile("bar.sync 1, %0;" ::"n"(32 * S::WARPS) : "memory");
                    if (y == 0) {
#pragma unroll
                        for (int w = 0; w < S::WARPS; ++w) top = fmaxf(top, s_m[w][r]), topw = fmaxf(topw, s_w[w][r]);
                        const float ref = finite_ref(top), refw = finite_ref(topw);
#pragma unroll
                        for (int w = 0; w < S::WARPS; ++w) {
                            f[w] = ex2(s_w[w][r] - refw);
                            sum = __fmaf_rn(s_l[w][r], ex2(s_m[w][r] - ref), sum);
                        }
                        inv = scale_of(top, topw, sum);
                    }
                    float2 acc{0.f, 0.f};
#pragma unroll
                    for (int w = 0; w < S::WARPS; ++w) {
                        const float2 v = *reinterpret_cast<const float2*>(join + (w * 8 + warp) * 68 + 2 * lane);
                        acc.x = __fmaf_rn(v.x, f[w], acc.x);
                        acc.y = __fmaf_rn(v.y, f[w], acc.y);
                    }
                    if (whole) {
                        if (r < nrows) store_pair(row, channel_of(y), acc.x, acc.y, inv);
                    } else if (r < nrows) {
                        *reinterpret_cast<float2*>(part + 6 * S::ROWS + r * D + channel_of(y)) = acc;
                    }
                }
                if (lane == 0 && r < nrows) {
                    if (whole) {
                        if (ml == 0) store_lse(row, top, sum);
                    } else {
                        part[3 * ml * S::ROWS + r] = top;
                        part[(3 * ml + 1) * S::ROWS + r] = sum;
                        part[(3 * ml + 2) * S::ROWS + r] = topw;
                    }
                }
            }
            if (!whole && used) {
                // each warp for its rows: the last CTA to arrive joins the CTAs' partials.  The loops are kept short: code
                // that runs once per call is fetched as it runs (with 24 partials unrolled the joining took 3.9 us)
                uint32_t* count = A.count + c0 * S::WARPS + warp;
                uint32_t seen = 0;
                __syncwarp();
                if (lane == 0) seen = atomic_add_acq_rel(count, 1u);
                seen = __shfl_sync(0xffffffffu, seen, 0);
                if (seen > uint32_t(c1 - c0)) {
                    if (lane == 0) raise_status(KVB_DEV_WORKSPACE);
                } else if (seen == uint32_t(c1 - c0)) {
                    if (lane == 0) *count = 0;
                    // the partial of c is its first one, unless the (sequence, head, group) begins inside c's run
                    const float* slot0 = A.part + int64_t(2 * c0 + (W.share(c0) < p.v0 ? 1 : 0)) * S::PART;
                    auto slot_of = [&](int c) { return c == c0 ? slot0 : A.part + int64_t(2 * c) * S::PART; };
                    float top[NT], topw[NT], sum[NT];
                    float2 acc[NT][D / 64];
#pragma unroll
                    for (int x = 0; x < NT; ++x) {
                        top[x] = topw[x] = -INFINITY;
                        sum[x] = 0.f;
#pragma unroll
                        for (int y = 0; y < D / 64; ++y) acc[x][y] = float2{0.f, 0.f};
                    }
                    for (int cc = c0; cc <= c1; cc += 32) {      // 32 partials: a lane has the m, l and mw of one
                        const int cnt = min(32, c1 - cc + 1);
                        const float* mine_p = slot_of(min(cc + lane, c1)) + 3 * ml * S::ROWS;
                        float f[NT], ms[NT], lv[NT];             // f: mw until the first loads of O are on their way
#pragma unroll
                        for (int x = 0; x < NT; ++x) {
                            ms[x] = lane < cnt ? __ldcg(mine_p + row_of(x)) : -INFINITY;
                            lv[x] = lane < cnt ? __ldcg(mine_p + S::ROWS + row_of(x)) : 0.f;
                            f[x] = lane < cnt ? __ldcg(mine_p + 2 * S::ROWS + row_of(x)) : -INFINITY;
                        }
                        constexpr int B = 16 / NT;               // partials whose loads are in flight together
#pragma unroll 1
                        for (int k0 = 0; k0 < cnt; k0 += B) {
                            float2 v[B][NT][D / 64];
                            const float* q = A.part + int64_t(2 * (cc + k0)) * S::PART + 6 * S::ROWS;
#pragma unroll
                            for (int k = 0; k < B; ++k) {
                                const float* qk = k == 0 && cc + k0 == c0 ? slot0 + 6 * S::ROWS : q + 2 * k * S::PART;
#pragma unroll
                                for (int x = 0; x < NT; ++x)
#pragma unroll
                                    for (int y = 0; y < D / 64; ++y) {
                                        v[k][x][y] = float2{0.f, 0.f};
                                        if (k0 + k < cnt && !(few && y > 0))
                                            v[k][x][y] = __ldcg(reinterpret_cast<const float2*>(qk + row_of(x) * D + channel_of(y)));
                                    }
                            }
                            if (k0 == 0) {
#pragma unroll
                                for (int x = 0; x < NT; ++x) {
                                    const float to = fmaxf(top[x], warp_max(ms[x])), ref = finite_ref(to);
                                    sum[x] = __fmaf_rn(sum[x], ex2(top[x] - ref), kvb::warp_sum(lv[x] * ex2(ms[x] - ref)));
                                    top[x] = to;
                                    const float tow = fmaxf(topw[x], warp_max(f[x])), refw = finite_ref(tow), old = ex2(topw[x] - refw);
                                    topw[x] = tow;
                                    f[x] = ex2(f[x] - refw);
#pragma unroll
                                    for (int y = 0; y < D / 64; ++y) acc[x][y].x *= old, acc[x][y].y *= old;
                                }
                            }
#pragma unroll
                            for (int k = 0; k < B; ++k)
#pragma unroll
                                for (int x = 0; x < NT; ++x) {
                                    const float fk = __shfl_sync(0xffffffffu, f[x], (k0 + k) & 31);
#pragma unroll
                                    for (int y = 0; y < D / 64; ++y) {
                                        acc[x][y].x = __fmaf_rn(v[k][x][y].x, fk, acc[x][y].x);
                                        acc[x][y].y = __fmaf_rn(v[k][x][y].y, fk, acc[x][y].y);
                                    }
                                }
                        }
                    }
#pragma unroll
                    for (int x = 0; x < NT; ++x) {
                        if (row_of(x) >= nrows) continue;
                        const int64_t row = row_at(p.seq, h, row0 + row_of(x));
                        const float inv = scale_of(top[x], topw[x], sum[x]);
#pragma unroll
                        for (int y = 0; y < D / 64; ++y)
                            if (!(few && y > 0)) store_pair(row, channel_of(y), acc[x][y].x, acc[x][y].y, inv);
                        if (lane == 0 && ml == 0) store_lse(row, top[x], sum[x]);
                    }
                }
            }
            cur = next;
            p = pn;
            first = 0;
        }
    }
    if (*abort) {                                                // copies in flight land before shared memory is released
        if (lane == 0) {
            raise_status(KVB_DEV_TIMEOUT);
            for (int k = max(0, copied - S::STAGES); k < copied; ++k) mbar_wait(&full[warp][k % S::STAGES], (k / S::STAGES) & 1, 10000000ull);
        }
    }
    __syncthreads();
}

}  // namespace kvb
