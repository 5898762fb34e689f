// kvb_shared_tc.cuh - the pages that several sequences hold, attended once for all of them, on the 5th-generation tensor cores
// (kvb_rows_tc.cuh).
//
//   s_j = lam q . (kc_j - 128) ks,  p_j = 2^(s_j - m),  l = sum p_j,  o = sum p_j (vc_j - 128) vs / l
//
// over the tokens of a segment (kvb_page_share).  A work item is a group of 256 rows (row = (member, query, head in the group)) of
// one (segment, KV head), a unit 64 tokens.  One warp looks the pages up, 32 units ahead, a lane a unit, and copies codes with TMA
// through a ring; four warps turn them into operands in shared memory: keys into the queries' type, values into float16, code -
// 128 being exact in both.  A page's key scale multiplies the logits of its tokens and its value scale their weights,
// w = p vs 2^(m - mw), which become float16 (2^-11) with a reference mw of their own, so that pages whose scales lie far apart lose
// neither mass nor values.
//
// What a segment gives is a part of its members' rows (O normalised, maximum, sum) for the kernel of the sequences' own
// tokens to join (PD_OWN of kvb_paged_decode.cuh).
//
// The conversion is a loop that is not unrolled: with all of it in line, it and the softmax together left the instruction cache
// at every unit (64 sequences behind 16384 tokens 80 us, 75 with the loop; 32 behind four prompts 61 and 54).  Neither HBM nor the
// tensor cores bound it (20 % busy in the first case, issue slots 42 %, waits for instructions 1.4 of 9 cycles a warp) but the
// converting warps, of which the registers leave one an SM partition: of a unit's 2750 cycles there (3200 with 256 rows) 1000 are keys, 700
// values, the rest fences, barriers and the wait for codes; the softmax takes 1400.  The start (page look-ups, queries, first instructions) is
// 10 of the about 45 us of this kernel in the first case.  Two rounds of the loop at a time: 75.6 us and 56.7.
#pragma once
#include "kvb_rows_tc.cuh"

namespace kvb {

constexpr int ST_WARPS = CM_SOFTMAX + 8;      // softmax; S; O of either tile; copies; conversion
constexpr int ST_K = 2, ST_V = 3, ST_CODES = 3;                  // stages of operands and of codes
constexpr int ST_SCALES = 64;                 // units whose scales are at hand

struct SharedTcParams {
    CUtensorMap tm_k, tm_v;                   // codes as (d, page, n_pages * Hkv), box d x min(page, 64) x 1
    PagesView P;
    SharedView shared;
    const void* q;                            // (n, Hq, Tq, d)
    int Hq, Tq, rep;
    uint64_t by_rep, by_rows;                 // for pd_div: by rep, by rep Tq
    int page_log2;
    float lam;                                // |scaling| log2(e), above 0
    int negate;                               // scaling < 0
    int64_t rows;                             // n Tq Hq
    float* level_o;                           // [levels][rows][d], normalised
    float* level_ml;                          // [levels][rows][2]: maximum, sum
    float* part;                              // two a CTA
    void* cuts;                               // CmCut<SharedItem> a CTA
    int ctas;                                 // that take part
};

template <int D>
struct StShape {
    using S = CmShape<D>;
    static constexpr int CODES = 2 * CM_KEYS * D;               // bytes of a unit
    static constexpr int SMEM = 1024 + 2 * S::QTILE + (ST_K + ST_V) * S::TILE + ST_CODES * CODES + S::XBYTES + ST_SCALES * 8 * 4;
};

// 16 codes -> 16 values code - 128 of type T in two 16-byte chunks
template <typename T>
__device__ __forceinline__ void st_convert(const uint4& w, uint4 (&to)[2]) {
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
    uint32_t r[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __half>::value) {
            r[2 * i] = pd_half2<0x4140>(a[i]);
            r[2 * i + 1] = pd_half2<0x4342>(a[i]);
        } else {
            // the low seven bits become the mantissa of 128 + bits; less 128 where the eighth is set, else less 256
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t x = pd_prmt(a[i], 0x43434343u, k ? 0x4342u : 0x4140u);
                const uint32_t lo = x & 0xff7fff7fu, by = (x & 0x00800080u) ^ 0x43804380u;
                asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r[2 * i + k]) : "r"(lo), "r"(by));
            }
        }
    }
    to[0] = uint4{r[0], r[1], r[2], r[3]};
    to[1] = uint4{r[4], r[5], r[6], r[7]};
}

struct SharedItem {
    SharedSegment g;
    int h, row0;
};

// The work of a call; false when there is none.  Whole block.
template <int WARPS>
__device__ __forceinline__ bool shared_plan(const SharedTcParams& A, int* pre, int* shares, int (*warp_sum)[WARPS], PdPlan<true, CM_FIXED>& W) {
    const int n = A.shared.segment_count();
    if (!cm_scan<WARPS>(n, pre, shares, warp_sum, [&](int i, int& u, int& p) {
            const SharedSegment g = A.shared.segment(i);
            const int hg = (g.members * A.rep * A.Tq + 2 * CM_ROWS - 1) / (2 * CM_ROWS) * A.P.Hkv, units = (g.end - g.start + CM_KEYS - 1) / CM_KEYS;
            // a plan's segments fit 32 bits together (the host has seen to it); what is no plan may not
            u = units <= INT_MAX / hg - CM_FIXED ? units * hg : 0;
            p = u + CM_FIXED * hg;
        })) {
        if (threadIdx.x == 0) raise_status(KVB_DEV_BOUNDS);
        return false;
    }
    cm_deal(W, n, pre, shares, A.ctas);
    return shares[n] > 0;
}

// sequence, query and head of row `at` of a segment's KV head h
__device__ __forceinline__ int shared_row(const SharedTcParams& A, const SharedSegment& g, int h, int at, int& tok, int& head) {
    const int member = pd_div(at, A.by_rows), rest = at - member * A.rep * A.Tq;
    tok = pd_div(rest, A.by_rep);
    head = h * A.rep + rest - tok * A.rep;
    return A.shared.member(g, member);
}
// where its part goes
__device__ __forceinline__ int64_t shared_out(const SharedTcParams& A, const SharedSegment& g, int h, int at) {
    int tok, head;
    const int of = shared_row(A, g, h, at, tok, head);
    return g.level * A.rows + (int64_t(of) * A.Tq + tok) * A.Hq + head;
}
// 2^(mw - m) / l; rows that see nothing give 0, NaN stays
__device__ __forceinline__ float shared_inverse(float m, float mw, float sum) {
    return sum > 0.f ? ex2(mw - (m == -INFINITY ? 0.f : m)) / sum : (sum == sum ? 0.f : sum);
}

// ROUNDS times 16 codes, 2048 bytes apart, as operands STEP bytes apart, and to the asynchronous proxy; whole warp.  In a short loop,
// the next codes read before these are stored: unrolled, it and the softmax beside it did not fit the instruction cache, and half
// of the time was waiting for code.
template <typename T, int ROUNDS, int STEP>
__device__ __forceinline__ void st_store(const uint8_t* from, uint8_t* to, uint32_t first, bool swap) {
    uint4 next = *reinterpret_cast<const uint4*>(from);
#pragma unroll 1
    for (int i = 0; i < ROUNDS; ++i) {
        const uint4 codes = next;
        from += 2048;
        if (i + 1 < ROUNDS) next = *reinterpret_cast<const uint4*>(from);
        uint4 x[2];
        st_convert<T>(codes, x);
        // the two halves of the channels in opposite order: their chunks then meet different banks
        *reinterpret_cast<uint4*>(to + first) = swap ? x[1] : x[0];
        *reinterpret_cast<uint4*>(to + (first ^ 16)) = swap ? x[0] : x[1];
        to += STEP;
    }
    fence_proxy_async_smem();
    __syncwarp();
}

template <typename T, int D>
__global__ void __launch_bounds__(32 * ST_WARPS, 1) shared_pages_kernel(const __grid_constant__ SharedTcParams A) {
    using S = CmShape<D>;
    constexpr int BF16 = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    extern __shared__ uint8_t st_raw[];
    __shared__ int pre[PS_MAX_SEQS + 1], shares[PS_MAX_SEQS + 1];        // units and places before each segment
    __shared__ CmBars B;
    __shared__ uint64_t codes_full[ST_CODES], codes_empty[ST_CODES];
    __shared__ int warp_sum[2][ST_WARPS];
    __shared__ uint32_t s_tmem;
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(st_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* const sq = base;                                    // [2 tiles], then key and value operands and codes [stage]
    uint8_t* const sk = sq + 2 * S::QTILE;
    uint8_t* const sv = sk + ST_K * S::TILE;
    uint8_t* const sc = sv + ST_V * S::TILE;
    float* const pass_all = reinterpret_cast<float*>(sc + ST_CODES * StShape<D>::CODES);
    // of a unit's tokens 16 g ..: scaling log2(e) times the key scale (-1: no page), log2 of the value scale
    float4* const scales = reinterpret_cast<float4*>(pass_all + 4 * S::XROWS);
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const PagesView& P = A.P;
    const SharedView& V = A.shared;

    if (threadIdx.x == 0) {
        B.init(4);                                               // the converting warps
        for (int i = 0; i < ST_CODES; ++i) {
            mbar_init(&codes_full[i], 1);
            mbar_init(&codes_empty[i], 4);
        }
        fence_mbar_init();
    }
    chain_kernels();
    PdPlan<true, CM_FIXED> W;
    const int cta = blockIdx.x;
    const bool any = shared_plan<ST_WARPS>(A, pre, shares, warp_sum, W);
    CmCut<SharedItem>* const cuts = static_cast<CmCut<SharedItem>*>(A.cuts);
    if (!any || cta >= W.ctas) {
        if (threadIdx.x == 0) cuts[cta] = CmCut<SharedItem>{};
        return;
    }
    const int u0 = W.units_before(W.share(cta)), u1 = W.units_before(W.share(cta + 1));

    if (warp == CM_SOFTMAX) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(CM_TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    cm_before();
    __syncthreads();
    cm_after();
    const uint32_t tmem = s_tmem;
    // the piece that begins at unit `cur`
    struct Item {
        PdPiece p;
        SharedSegment g;
        int h, row0, nrows;                                      // KV head, first row, rows
        __device__ bool split() const { return nrows <= CM_ROWS; }
        __device__ int tiles() const { return p.b - p.a; }
    };
    auto item_at = [&](int cur) {
        Item x;
        x.p = pd_piece(W, cur, u1);
        x.g = V.segment(x.p.seq);
        const int groups = W.heads(x.p.seq) / P.Hkv;
        x.h = x.p.vh / groups;
        x.row0 = (x.p.vh - x.h * groups) * 2 * CM_ROWS;
        x.nrows = min(x.g.members * A.rep * A.Tq - x.row0, 2 * CM_ROWS);
        return x;
    };
    auto step_at = [&](int cur) {
        const Item x = item_at(cur);
        return CmStep{x.tiles(), x.tiles(), x.g.end - x.g.start - x.p.a * CM_KEYS, x.split()};
    };

    if (warp < CM_SOFTMAX) {
        // ---------------- softmax of tile t: thread = row ----------------
        const int t = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
        const uint32_t lanes = uint32_t(quarter * 32) << 16, ts = tmem + lanes + t * 128, to = tmem + lanes + 256 + t * 128;
        float* const pass = pass_all + quarter * S::XROWS;
        // the warp's 32 rows of the tile, swizzled, zeros past the last; and how many of the segment's tokens the thread's row sees
        auto load_q = [&](const Item& x) {
            constexpr int CHUNKS = D / 8, PER = 32 / CHUNKS;     // 16-byte chunks of a row, rows at a time
            const int c = lane % CHUNKS, tile0 = x.split() ? 0 : t * CM_ROWS;
            uint4 v[32 / PER];
#pragma unroll
            for (int i = 0; i < 32 / PER; ++i) {
                const int row = tile0 + quarter * 32 + i * PER + lane / CHUNKS;
                v[i] = uint4{0, 0, 0, 0};
                if (row < x.nrows) {
                    int tok, head;
                    const int of = shared_row(A, x.g, x.h, x.row0 + row, tok, head);
                    v[i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(A.q) + ((int64_t(of) * A.Hq + head) * A.Tq + tok) * D + 8 * c));
                }
            }
            int limit = x.g.end - x.g.start;
            if (tile0 + r < x.nrows) {
                int tok, head;
                const int of = shared_row(A, x.g, x.h, x.row0 + tile0 + r, tok, head);
                limit = min(x.g.end, V.length_of(of, P) - A.Tq + tok + 1) - x.g.start;
            }
            if (cm_units(x.split(), x.tiles(), t) == 0) return limit;
#pragma unroll
            for (int i = 0; i < 32 / PER; ++i) {
                const int row = quarter * 32 + i * PER + lane / CHUNKS;
                *reinterpret_cast<uint4*>(sq + t * S::QTILE + (c >> 3) * S::QHALF + row * 128 + (((c ^ row) & 7) * 16)) = v[i];
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&B.q_full[t]);
            return limit;
        };
        Item x{};
        int limit = 0;
        if (u0 < u1) {
            x = item_at(u0);
            limit = load_q(x);
        }
        uint32_t sn = 0, it = 0, xn = 0;                         // S of this tile so far; units of the block; parts passed on
        int first = 1;
        bool ok = true;
        for (int cur = u0; cur < u1 && ok;) {
            const bool split = x.split();
            const int units = cm_units(split, x.tiles(), t);
            float m = -INFINITY, mw = -INFINITY, l = 0.f;
            for (int j = 0; j < units; ++j, ++sn) {
                const uint32_t half = sn & 1, cols = ts + CM_KEYS * half;
                const int u = cm_unit(split, t, j);
                if (!(ok = cm_wait(&B.s_full[t][half], sn >> 1))) break;
                cm_after();
                const int left = limit - (x.p.a + u) * CM_KEYS;  // tokens from this unit on that the row sees
                const float4 sk4 = scales[2 * ((it + u) % ST_SCALES)], sv4 = scales[2 * ((it + u) % ST_SCALES) + 1];
                float lamk[4] = {sk4.x, sk4.y, sk4.z, sk4.w}, lv[4] = {sv4.x, sv4.y, sv4.z, sv4.w};
                float v[CM_KEYS];
                cm_ld64(cols, v);
                if (A.negate) {
#pragma unroll
                    for (int i = 0; i < CM_KEYS; ++i) v[i] = -v[i];
                }
                // tokens that the row does not see, or that have no page.  What it sees nothing of (16 tokens are of one page) gives it
                // nothing whatever its scales are: -inf times NaN and -inf + inf would be NaN.
                if (__any_sync(0xffffffffu, left < CM_KEYS || fminf(fminf(lamk[0], lamk[1]), fminf(lamk[2], lamk[3])) < 0.f)) {
#pragma unroll
                    for (int i = 0; i < CM_KEYS; ++i) v[i] = i < left && lamk[i / 16] > 0.f ? v[i] : -INFINITY;
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        if (16 * g >= left) lamk[g] = 1.f, lv[g] = -INFINITY;
                }
                float y = -INFINITY, yw = -INFINITY;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float top[2] = {v[16 * g], v[16 * g + 1]};
#pragma unroll
                    for (int i = 2; i < 14; i += 4) {
                        top[0] = cm_max3(top[0], v[16 * g + i], v[16 * g + i + 1]);
                        top[1] = cm_max3(top[1], v[16 * g + i + 2], v[16 * g + i + 3]);
                    }
                    const float yg = cm_max3(cm_max3(top[0], v[16 * g + 14], v[16 * g + 15]), top[1], -INFINITY) * fabsf(lamk[g]);
                    y = cm_max3(y, yg, -INFINITY);
                    yw = fmaxf(yw, yg + lv[g]);
                }
                const bool grow = y > m + PD_LAZY, groww = yw > mw + PD_LAZY;
                if (__any_sync(0xffffffffu, grow || groww)) {
                    const float f = groww ? ex2(mw - yw) : 1.f;
                    if (groww) mw = yw;
                    l *= grow ? ex2(m - y) : 1.f;
                    if (grow) m = y;
                    if (j > 0 && __any_sync(0xffffffffu, groww)) {               // once the product before is done
                        if (!(ok = cm_wait(&B.pv_done[t][half ^ 1], (sn - 1) >> 1))) break;
                        cm_after();
                        cm_rescale<D>(to, f);
                    }
                }
                const float ref = m == -INFINITY ? 0.f : m, dr = ref - (mw == -INFINITY ? 0.f : mw);
                uint32_t w[CM_KEYS / 2];
                // w = p 2^e, e = lv + dr.  A weight that float32 has to hold as p 2^e with a large e has a p that it cannot: where
                // e passes 100, p is taken 2^(e - 100) times as large and its sum is scaled back.
                float both = 0.f;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const float e2 = lv[g] + dr, up = fmaxf(e2 - 100.f, 0.f), f = ex2(e2 - up);
                    const float2 lam2{fabsf(lamk[g]), fabsf(lamk[g])}, f2{f, f}, ref2{up - ref, up - ref};
                    float2 sum[2];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int i = 8 * g + k;
                        float2 e = cm_fma2(float2{v[2 * i], v[2 * i + 1]}, lam2, ref2);
                        if (i % 4 < CM_FMA) {
                            e = cm_ex2(e);
                        } else {
                            e.x = ex2(e.x);
                            e.y = ex2(e.y);
                        }
                        sum[k & 1] = k < 2 ? e : cm_add2(sum[k & 1], e);
                        e = cm_mul2(e, f2);
                        w[i] = pack_half2(e.x, e.y);
                    }
                    sum[0] = cm_add2(sum[0], sum[1]);
                    both = __fmaf_rn(sum[0].x + sum[0].y, ex2(-up), both);
                }
                if (!(y < INFINITY)) {                           // NaN or +inf among the logits: the row is NaN
                    both = NAN;
                    w[0] = 0x7fff7fffu;
                }
                __syncwarp();
                cm_st32(cols, w);
                l += both;
                cm_wait_st();
                cm_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&B.p_ready[t][half]);
            }
            if (!ok) break;
            it += x.tiles();
            const Item done = x;
            const int next = cur + x.tiles();
            if (next < u1) {                                     // all products with this item's queries are done
                x = item_at(next);
                limit = load_q(x);
            }
            if (units > 0 && !(ok = cm_wait(&B.pv_done[t][(sn - 1) & 1], (sn - 1) >> 1))) break;     // nothing is written
            cm_after();
            const bool whole = done.p.a == 0 && done.p.b == done.p.units, two = split && done.tiles() > 1;
            const int tile0 = split ? 0 : t * CM_ROWS;
            float* const part = A.part + int64_t(2 * cta + (first ? 0 : 1)) * CM_PART<D>;
            if (split && t == 1) {                               // the second tile passes its part on to the first
                for (int c = 0; c < D / 32 && two; ++c, ++xn) {
                    if (xn > 0 && !(ok = cm_wait(&B.x_empty[quarter], xn - 1))) break;
                    float v[32];
                    cm_ld32(to + 32 * c, v);
#pragma unroll
                    for (int i = 0; i < 32; ++i) pass[32 * i + lane] = v[i];
                    pass[1024 + lane] = m;
                    pass[1056 + lane] = l;
                    pass[1088 + lane] = mw;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&B.x_full[quarter]);
                    __syncwarp();
                }
            } else {
                const bool row_ok = tile0 + r < done.nrows;
                const int64_t row = row_ok ? shared_out(A, done.g, done.h, done.row0 + tile0 + r) : 0;
                float f0 = 1.f, f1 = 0.f;
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {               // 32 channels; the sum and maxima with the first
                    float v[32];
                    cm_ld32(to + 32 * c, v);
                    if (two) {
                        if (!(ok = cm_wait(&B.x_full[quarter], xn))) break;
                        if (c == 0) {
                            const float m1 = pass[1024 + lane], l1 = pass[1056 + lane], w1 = pass[1088 + lane];
                            const float most = fmaxf(m, m1), ref = most == -INFINITY ? 0.f : most;
                            const float mostw = fmaxf(mw, w1), refw = mostw == -INFINITY ? 0.f : mostw;
                            f0 = ex2(mw - refw);
                            f1 = ex2(w1 - refw);
                            l = l * ex2(m - ref) + l1 * ex2(m1 - ref);
                            m = most, mw = mostw;
                        }
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = __fmaf_rn(pass[32 * i + lane], f1, v[i] * f0);
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&B.x_empty[quarter]);
                        __syncwarp();
                        ++xn;
                    }
                    if (row_ok) {
                        if (whole) {
                            const float inv = shared_inverse(m, mw, l);
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] *= inv;
                            cm_put(A.level_o + row * D + 32 * c, v);
                        } else {
                            cm_put(part + (tile0 + r) * D + 32 * c, v);
                        }
                    }
                    __syncwarp();
                }
                if (ok && row_ok) {
                    if (whole) {
                        *reinterpret_cast<float2*>(A.level_ml + 2 * row) = float2{m, l};
                    } else {
                        __stcg(part + 2 * CM_ROWS * D + tile0 + r, m);
                        __stcg(part + 2 * CM_ROWS * (D + 1) + tile0 + r, l);
                        __stcg(part + 2 * CM_ROWS * (D + 2) + tile0 + r, mw);
                    }
                }
            }
            __syncwarp();
            cm_before();                                         // O is read: the next product into it comes after the next P
            cur = next;
            first = 0;
        }
    } else if (warp == CM_SOFTMAX) {
        cm_issue_scores<D, BF16, ST_K>(B, tmem, smem_u32(sq), smem_u32(sk), u0, u1, step_at);
    } else if (warp < CM_SOFTMAX + 3) {
        // the second of these has the time: the joining kernel is told what this CTA's end cuts
        if (warp == CM_SOFTMAX + 2 && lane == 0)
            cm_note_cut(W, cta, cuts, [&](const PdPiece& p, SharedItem& x) {
                x.g = V.segment(p.seq);
                const int groups = W.heads(p.seq) / P.Hkv;
                x.h = p.vh / groups;
                x.row0 = (p.vh - x.h * groups) * 2 * CM_ROWS;
                return min(x.g.members * A.rep * A.Tq - x.row0, 2 * CM_ROWS);
            });
        __syncwarp();
        cm_issue_values<D, 0, ST_V>(B, tmem, smem_u32(sv), warp - CM_SOFTMAX - 1, u0, u1, step_at);
    } else if (warp == CM_SOFTMAX + 3) {
        // ---------------- copies of codes: lane i looks after the units i mod 32 of the block ----------------
        const int total = u1 - u0, box = min(P.page, CM_KEYS);
        struct Place {
            int row[4], off;                                     // rows of the tensor maps (< 0: nothing there), token in the page
        };
        auto place = [&](int k) {
            Place x{{-1, -1, -1, -1}, 0};
            if (k >= total) return x;
            const PdPiece p = pd_piece(W, u0 + k, u1);
            const SharedSegment g = V.segment(p.seq);
            const int h = p.vh / (W.heads(p.seq) / P.Hkv), t0 = g.start + p.a * CM_KEYS, slot = V.slot_of(g, P.n_slots);
            x.off = t0 & (P.page - 1);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (i * box >= CM_KEYS || t0 + i * box >= g.end) continue;
                const int id = slot < 0 ? -1 : P.table[int64_t(slot) * P.max_blocks + ((t0 + i * box) >> A.page_log2)];
                if (id >= 0 && id < P.n_pages) x.row[i] = id * P.Hkv + h;
                else raise_status(KVB_DEV_BOUNDS);
            }
            return x;
        };
        Place at = place(lane);
        float ks[4], vs[4];
        auto load_scales = [&](const Place& x) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {                        // of the tokens 16 g ..; key scale < 0: no page
                const int row = box == 64 ? x.row[0] : box == 32 ? x.row[g >> 1] : x.row[g];
                ks[g] = row >= 0 ? P.ks[row] : -1.f;
                vs[g] = row >= 0 ? P.vs[row] : 0.f;
            }
        };
        load_scales(at);
        bool ok = true;
        int k = 0;
        for (; k < total && ok; ++k) {
            if ((k & 31) == 0) {
                // scales of these 32 units; what the places held is 64 units old
                const int to = (k + lane) % ST_SCALES;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    // a scale of zero becomes one too small to matter, so that -inf stays -inf; NaN stays
                    const float x = A.lam * ks[g];
                    ks[g] = ks[g] < 0.f ? -1.f : x < 1e-37f ? 1e-37f : x;
                    vs[g] = vs[g] > 0.f ? __log2f(vs[g]) : -INFINITY;
                }
                scales[2 * to] = float4{ks[0], ks[1], ks[2], ks[3]};
                scales[2 * to + 1] = float4{vs[0], vs[1], vs[2], vs[3]};
                __syncwarp();
            }
            const uint32_t st = k % ST_CODES;
            if (k >= ST_CODES && !(ok = cm_wait(&codes_empty[st], k / ST_CODES - 1))) break;
            if (lane == (k & 31)) {
                uint32_t boxes = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) boxes += at.row[i] >= 0;
                mbar_arrive_expect_tx(&codes_full[st], boxes * 2 * box * D);
                uint8_t* dst = sc + st * StShape<D>::CODES;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (at.row[i] >= 0) {
                        tma_load_3d(dst + i * box * D, &A.tm_k, 0, at.off, at.row[i], &codes_full[st]);
                        tma_load_3d(dst + CM_KEYS * D + i * box * D, &A.tm_v, 0, at.off, at.row[i], &codes_full[st]);
                    }
            }
            __syncwarp();
            if ((k & 31) == 31) {
                at = place(k + 1 + lane);
                load_scales(at);
            }
        }
        // copies in flight land before shared memory is released (without a timeout they were all waited for)
        for (int i = max(0, k - ST_CODES); i < k; ++i) mbar_wait(&codes_full[i % ST_CODES], (i / ST_CODES) & 1, 10000000ull);
        __syncwarp();
    } else {
        // ---------------- conversion: 128 threads, 16 codes at a time ----------------
        const int id = threadIdx.x - 32 * (CM_SOFTMAX + 4), total = u1 - u0;
        constexpr int CHUNKS = D / 16, ROUNDS = CM_KEYS * CHUNKS / 128, ROW_STEP = 128 / CHUNKS * 128;
        // the thread's 16 codes of a round: channels 16 c .. of row id / CHUNKS, rows a multiple of 8 further on; as 16-bit values
        // the two chunks 2 c and 2 c + 1 of a half's row, swizzled by the row
        const int c = id % CHUNKS, row = id / CHUNKS, swap = c >> 2 & 1;
        const uint32_t at = (c >> 2) * S::HALF + row * 128, first = uint32_t((((2 * c + swap) & 7) ^ (row & 7)) * 16);
        bool ok = true;
        for (int k = 0; k < total && ok; ++k) {
            const uint32_t st = k % ST_CODES, kst = k % ST_K, vst = k % ST_V;
            if (!(ok = cm_wait(&codes_full[st], k / ST_CODES))) break;
            const uint8_t* from = sc + st * StShape<D>::CODES + 16 * id;
            if (k >= ST_K && !(ok = cm_wait(&B.k_empty[kst], k / ST_K - 1))) break;
            st_store<T, ROUNDS, ROW_STEP>(from, sk + kst * S::TILE + at, first, swap);
            if (lane == 0) mbar_arrive(&B.k_full[kst]);
            if (k >= ST_V && !(ok = cm_wait(&B.v_empty[vst], k / ST_V - 1))) break;
            st_store<__half, ROUNDS, ROW_STEP>(from + CM_KEYS * D, sv + vst * S::TILE + at, first, swap);
            if (lane == 0) {
                mbar_arrive(&B.v_full[vst]);
                mbar_arrive(&codes_empty[st]);
            }
            __syncwarp();
        }
        __syncwarp();
    }
    cm_before();
    __syncthreads();
    cm_after();
    if (warp == CM_SOFTMAX) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(CM_TMEM));
}

// Joins the items that shared_pages_kernel cut.
template <int D>
__global__ void __launch_bounds__(32 * CJ_WARPS, 4) shared_join_kernel(const __grid_constant__ SharedTcParams A) {
    cm_join<D, true>(static_cast<const CmCut<SharedItem>*>(A.cuts), A.ctas, A.part,
                     [&](const SharedItem& x, int r, int ch, const float (&o)[CJ_CH], float top, float sum, float topw) {
                         const int64_t row = shared_out(A, x.g, x.h, x.row0 + r);
                         const float inv = shared_inverse(top, topw, sum);
                         *reinterpret_cast<float4*>(A.level_o + row * D + ch) = float4{o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
                         if (ch == 0) *reinterpret_cast<float2*>(A.level_ml + 2 * row) = float2{top, sum};
                     });
}

}  // namespace kvb
