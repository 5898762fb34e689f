// kvb_cross_tc.cuh - attention of packed queries to keys of another length (an encoder's states), more than a few rows per
// sequence, on the 5th-generation tensor cores (kvb_rows_tc.cuh).
//
// A work item is a group of 256 query rows (row = token * rep + head in the group: the rep query heads of a KV head and the
// sequence's queries packed together) of one (sequence, KV head); one warp copies its keys and values with TMA through rings of
// four units.  P is rounded to the inputs' type.
//
// Values past a sequence's end belong to the next one: their weight is zero, but zero times NaN is not, so the rows of the
// last 16 that lie past the end are zeroed in shared memory, and steps of 16 keys behind them left out.
//
// Measured (32 query heads over 8 KV heads of 128 channels, bfloat16): 8192 queries over 16384 keys 1.83 to 2.16 ms, 1020 to 1200
// TFLOP/s, with the power limit active and the SM clock between 1600 and 1710 MHz; of that kernel's time on 2048 queries over
// 8192 keys the tensor cores are busy 53 %, the special functions 40 %, the issue slots 48 %, and no single one bounds it: a tile's
// softmax and its products wait for one another where the other tile does not fill in.  Eight packed prompts of 5300 queries
// over 14860 keys 197 us, 870 TFLOP/s: items start and end (queries, sums, cut items).  37 queries of 6 sequences (67 MB) 28 us,
// of which 9 are the joining kernel.
#pragma once
#include "kvb_cross.cuh"
#include "kvb_rows_tc.cuh"

namespace kvb {

constexpr int CM_WARPS = CM_SOFTMAX + 4;
constexpr int CM_STAGES = 4;                  // of keys and of values

template <int D>
struct CrossTcShape {
    using S = CmShape<D>;
    static constexpr int SMEM = 1024 + 2 * S::QTILE + 2 * CM_STAGES * S::TILE + S::XBYTES;
};

struct CrossItem {
    int64_t row;                              // of out: the sequence's first token, the KV head's first query head
    int row0;
};

// The work of a call dealt to `ctas` CTAs; false when there is none.  Whole block.
template <int WARPS>
__device__ __forceinline__ bool cross_plan(const CrossParams& A, int ctas, int* pre, int* shares, int (*warp_sum)[WARPS], PdPlan<true, CM_FIXED>& W) {
    if (!cm_scan<WARPS>(A.n, pre, shares, warp_sum, [&](int i, int& u, int& p) {
            cr_work<2 * CM_ROWS, CM_KEYS, CM_FIXED>(cr_seq(A.cu_q, A.cu_k, A.nq, A.nk, i), A.rep, A.Hkv, u, p);
        })) {
        if (threadIdx.x == 0) raise_status(KVB_DEV_BOUNDS);
        return false;
    }
    cm_deal(W, A.n, pre, shares, ctas);
    return shares[A.n] > 0;
}

template <typename T, int D>
__global__ void __launch_bounds__(32 * CM_WARPS, 1) cross_many_kernel(const __grid_constant__ CrossParams A) {
    using S = CmShape<D>;
    constexpr int BF16 = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    extern __shared__ uint8_t cm_raw[];
    __shared__ int pre[CR_MAX_SEQS + 1], shares[CR_MAX_SEQS + 1];        // units and places before each sequence
    __shared__ CmBars B;
    __shared__ int warp_sum[2][CM_WARPS];
    __shared__ uint32_t s_tmem;
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(cm_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* const sq = base;                                    // [2 tiles], then keys and values [stage]
    uint8_t* const sk = sq + 2 * S::QTILE;
    uint8_t* const sv = sk + CM_STAGES * S::TILE;
    // the warp's number from a shuffle: the compiler then knows it, and what follows from it, to be the same in all lanes
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        B.init(1);
        fence_mbar_init();
    }
    chain_kernels();
    auto seq_at = [&](int i) { return cr_seq(A.cu_q, A.cu_k, A.nq, A.nk, i); };
    PdPlan<true, CM_FIXED> W;
    const int cta = blockIdx.x;
    const bool any = cross_plan<CM_WARPS>(A, A.ctas, pre, shares, warp_sum, W);
    CmCut<CrossItem>* const cuts = static_cast<CmCut<CrossItem>*>(A.cuts);
    if (!any || cta >= W.ctas) {
        if (threadIdx.x == 0) cuts[cta] = CmCut<CrossItem>{};
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
        CrSeq s;
        int h, row0, nrows, tiles;                               // KV head, first row, rows, units with keys
        __device__ bool split() const { return nrows <= CM_ROWS; }
    };
    auto item_at = [&](int cur) {
        Item x;
        x.p = pd_piece(W, cur, u1);
        x.s = seq_at(x.p.seq);
        const int groups = W.heads(x.p.seq) / A.Hkv;
        x.h = x.p.vh / groups;
        x.row0 = (x.p.vh - x.h * groups) * 2 * CM_ROWS;
        x.nrows = min(x.s.ql * A.rep - x.row0, 2 * CM_ROWS);
        x.tiles = x.s.kl > 0 ? x.p.b - x.p.a : 0;
        return x;
    };
    auto step_at = [&](int cur) {
        const Item x = item_at(cur);
        return CmStep{x.p.b - x.p.a, x.tiles, x.s.kl - x.p.a * CM_KEYS, x.split()};
    };

    if (warp < CM_SOFTMAX) {
        // ---------------- softmax of tile t: thread = row ----------------
        const int t = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
        const uint32_t lanes = uint32_t(quarter * 32) << 16, ts = tmem + lanes + t * 128, to = tmem + lanes + 256 + t * 128;
        float* const pass = reinterpret_cast<float*>(sv + CM_STAGES * S::TILE) + quarter * S::XROWS;
        auto load_q = [&](const Item& x) {                       // the warp's 32 rows of the tile, swizzled; zeros past the last
            constexpr int CHUNKS = D / 8, PER = 32 / CHUNKS;     // 16-byte chunks of a row, rows at a time
            const int c = lane % CHUNKS, tile0 = x.split() ? 0 : t * CM_ROWS;
            uint4 v[32 / PER];
#pragma unroll
            for (int i = 0; i < 32 / PER; ++i) {
                const int row = tile0 + quarter * 32 + i * PER + lane / CHUNKS, at = x.row0 + row, tok = pd_div(at, A.by_rep);
                v[i] = uint4{0, 0, 0, 0};
                if (row < x.nrows)
                    v[i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(A.q) + (int64_t(x.s.q0) + tok) * A.q_row +
                                                                 int64_t(x.h * A.rep + at - tok * A.rep) * A.q_head + 8 * c));
            }
#pragma unroll
            for (int i = 0; i < 32 / PER; ++i) {
                const int row = quarter * 32 + i * PER + lane / CHUNKS;
                *reinterpret_cast<uint4*>(sq + t * S::QTILE + (c >> 3) * S::QHALF + row * 128 + (((c ^ row) & 7) * 16)) = v[i];
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&B.q_full[t]);
        };
        Item x{};
        if (u0 < u1) {
            x = item_at(u0);
            if (cm_units(x.split(), x.tiles, t) > 0) load_q(x);
        }
        uint32_t sn = 0, it = 0, xn = 0;                         // S of this tile so far; units of the block; parts passed on
        int first = 1;
        bool ok = true;
        for (int cur = u0; cur < u1 && ok;) {
            const bool split = x.split();
            const int units = cm_units(split, x.tiles, t);
            // a warp without a row lets its S pass: what its part of O then is, nobody reads
            const bool live = __any_sync(0xffffffffu, (split ? 0 : t * CM_ROWS) + r < x.nrows);
            float m = -INFINITY, l = 0.f;
            for (int j = 0; j < units; ++j, ++sn) {
                const uint32_t half = sn & 1, cols = ts + CM_KEYS * half;
                const int u = cm_unit(split, t, j);
                if (!(ok = cm_wait(&B.s_full[t][half], sn >> 1))) break;
                cm_after();
                const int left = x.s.kl - (x.p.a + u) * CM_KEYS; // keys of the sequence from this unit on
                if (live) {
                    float v[CM_KEYS];
                    cm_ld64(cols, v);
                    if (A.negate) {
#pragma unroll
                        for (int i = 0; i < CM_KEYS; ++i) v[i] = -v[i];
                    }
                    if (left < CM_KEYS) {
#pragma unroll
                        for (int i = 0; i < CM_KEYS; ++i) v[i] = i < left ? v[i] : -INFINITY;
                    }
                    float top[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                    for (int i = 4; i < CM_KEYS - 4; i += 8)
#pragma unroll
                        for (int k = 0; k < 4; ++k) top[k] = cm_max3(top[k], v[i + k], v[i + 4 + k]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) top[k] = cm_max3(top[k], v[CM_KEYS - 4 + k], -INFINITY);
                    const float y = cm_max3(cm_max3(top[0], top[1], top[2]), top[3], -INFINITY) * A.lam;
                    const bool grow = y > m + PF_LAZY;
                    if (__any_sync(0xffffffffu, grow)) {
                        const float f = grow ? ex2(m - y) : 1.f;
                        if (grow) m = y;
                        l *= f;
                        if (j > 0) {                                 // once the product before is done
                            if (!(ok = cm_wait(&B.pv_done[t][half ^ 1], (sn - 1) >> 1))) break;
                            cm_after();
                            cm_rescale<D>(to, f);
                        }
                    }
                    const float ref = m == -INFINITY ? 0.f : m;
                    const float2 lam2{A.lam, A.lam}, ref2{-ref, -ref};
                    float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
                    uint32_t w[CM_KEYS / 2];
                    // of four pairs of keys CM_FMA on the FMA pipe: with all on the special-function unit, which the two
                    // warpgroups share, it is what bounds the step.  -inf gives 0 on either.
#pragma unroll
                    for (int i = 0; i < CM_KEYS / 2; ++i) {
                        float2 e = cm_fma2(float2{v[2 * i], v[2 * i + 1]}, lam2, ref2);
                        if (i % 4 < CM_FMA) {
                            e = cm_ex2(e);
                        } else {
                            e.x = ex2(e.x);
                            e.y = ex2(e.y);
                        }
                        sum[i & 1] = cm_add2(sum[i & 1], e);
                        w[i] = pack_f32<T>(e.x, e.y);
                    }
                    if (!(y < INFINITY)) {                           // NaN or +inf among the logits: the row is NaN
                        sum[0].x = NAN;
                        w[0] = 0x7fff7fffu;
                    }
                    __syncwarp();
                    cm_st32(cols, w);
                    const float2 both = cm_add2(sum[0], sum[1]);
                    l += both.x + both.y;
                }
                if (left < CM_KEYS) {                            // value rows past the end, up to the last step's 16
                    const uint32_t st = (it + u) % CM_STAGES;
                    if (!(ok = cm_wait(&B.v_full[st], (it + u) / CM_STAGES))) break;
                    if (r >= left && r < ((left + 15) & ~15)) {
#pragma unroll
                        for (int c = 0; c < 8 * S::HALVES; ++c)
                            *reinterpret_cast<uint4*>(sv + st * S::TILE + (c >> 3) * S::HALF + r * 128 + (c & 7) * 16) = uint4{0, 0, 0, 0};
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                cm_wait_st();
                cm_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&B.p_ready[t][half]);
            }
            if (!ok) break;
            it += x.tiles;
            const Item done = x;
            const int next = cur + x.p.b - x.p.a;
            if (next < u1) {                                     // all products with this item's queries are done
                x = item_at(next);
                if (cm_units(x.split(), x.tiles, t) > 0) load_q(x);
            }
            if (units > 0 && !(ok = cm_wait(&B.pv_done[t][(sn - 1) & 1], (sn - 1) >> 1))) break;     // nothing is written
            cm_after();
            const bool whole = done.p.a == 0 && done.p.b == done.p.units, two = live && split && done.tiles > 1;
            const int tile0 = split ? 0 : t * CM_ROWS;
            float* const part = A.part + int64_t(2 * cta + (first ? 0 : 1)) * CM_PART<D>;
            auto out_row = [&](int r) {                          // row r of the item in out and lse
                const int at = done.row0 + r, tok = pd_div(at, A.by_rep);
                return (int64_t(done.s.q0) + tok) * A.Hq + done.h * A.rep + at - tok * A.rep;
            };
            auto store_lse = [&](int64_t row, float top, float sum) {
                if (A.lse) A.lse[row] = sum == 0.f ? -INFINITY : top * 0.693147180559945309f + logf(sum);
            };
            if (split && t == 1) {                               // the second tile passes its part on to the first
                for (int c = 0; c < D / 32 && two; ++c, ++xn) {
                    if (xn > 0 && !(ok = cm_wait(&B.x_empty[quarter], xn - 1))) break;
                    float v[32];
                    cm_ld32(to + 32 * c, v);
#pragma unroll
                    for (int i = 0; i < 32; ++i) pass[32 * i + lane] = v[i];
                    pass[1024 + lane] = m;
                    pass[1056 + lane] = l;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&B.x_full[quarter]);
                    __syncwarp();
                }
            } else {
                const bool row_ok = tile0 + r < done.nrows;
                const int64_t row = out_row(tile0 + r);
                float f0 = 1.f, f1 = 0.f;
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {               // 32 channels; the sum and maximum with the first
                    float v[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = 0.f;
                    if (done.tiles > 0) cm_ld32(to + 32 * c, v);
                    if (two) {
                        if (!(ok = cm_wait(&B.x_full[quarter], xn))) break;
                        if (c == 0) {
                            const float m1 = pass[1024 + lane], l1 = pass[1056 + lane], most = fmaxf(m, m1), ref = most == -INFINITY ? 0.f : most;
                            f0 = ex2(m - ref);
                            f1 = ex2(m1 - ref);
                            l = l * f0 + l1 * f1;
                            m = most;
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
                            const float inv = cm_inverse(l);
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                uint32_t w[8];
#pragma unroll
                                for (int k = 0; k < 8; ++k) w[k] = pack_f32<T>(v[16 * i + 2 * k] * inv, v[16 * i + 2 * k + 1] * inv);
                                cm_store32(static_cast<T*>(A.out) + row * D + 32 * c + 16 * i, w);
                            }
                        } else {
                            cm_put(part + (tile0 + r) * D + 32 * c, v);
                        }
                    }
                    __syncwarp();
                }
                if (ok && row_ok) {
                    if (whole) {
                        store_lse(row, m, l);
                    } else {
                        __stcg(part + 2 * CM_ROWS * D + tile0 + r, m);
                        __stcg(part + 2 * CM_ROWS * (D + 1) + tile0 + r, l);
                    }
                }
            }
            __syncwarp();
            cm_before();                                         // O is read: the next product into it comes after the next P
            cur = next;
            first = 0;
        }
    } else if (warp == CM_SOFTMAX) {
        cm_issue_scores<D, BF16, CM_STAGES>(B, tmem, smem_u32(sq), smem_u32(sk), u0, u1, step_at);
    } else if (warp < CM_SOFTMAX + 3) {
        // the second of these has the time: the joining kernel is told what this CTA's end cuts
        if (warp == CM_SOFTMAX + 2 && lane == 0)
            cm_note_cut(W, cta, cuts, [&](const PdPiece& p, CrossItem& x) {
                const CrSeq s = seq_at(p.seq);
                const int groups = W.heads(p.seq) / A.Hkv, h = p.vh / groups;
                x.row0 = (p.vh - h * groups) * 2 * CM_ROWS;
                x.row = int64_t(s.q0) * A.Hq + h * A.rep;
                return min(s.ql * A.rep - x.row0, 2 * CM_ROWS);
            });
        __syncwarp();
        cm_issue_values<D, BF16, CM_STAGES>(B, tmem, smem_u32(sv), warp - CM_SOFTMAX - 1, u0, u1, step_at);
    } else {
        // ---------------- copies ----------------
        uint32_t it = 0;
        bool ok = true;
        for (int cur = u0; cur < u1 && ok;) {
            const Item x = item_at(cur);
            for (int j = 0; j < x.tiles && ok; ++j, ++it) {
                const uint32_t st = it % CM_STAGES, use = it / CM_STAGES;
                const int row = x.s.k0 + (x.p.a + j) * CM_KEYS;
                if (it >= CM_STAGES && !(ok = cm_wait(&B.k_empty[st], use - 1))) break;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&B.k_full[st], S::TILE);
                    for (int c = 0; c < S::HALVES; ++c)
                        tma_load_3d(sk + st * S::TILE + c * S::HALF, &A.tm_k, 64 * c, x.h * A.k_heads, row, &B.k_full[st]);
                }
                __syncwarp();
                if (it >= CM_STAGES && !(ok = cm_wait(&B.v_empty[st], use - 1))) {
                    if (lane == 0) mbar_wait(&B.k_full[st], use & 1, 10000000ull);
                    break;
                }
                if (lane == 0) {
                    mbar_arrive_expect_tx(&B.v_full[st], S::TILE);
                    for (int c = 0; c < S::HALVES; ++c)
                        tma_load_3d(sv + st * S::TILE + c * S::HALF, &A.tm_v, 64 * c, x.h * A.v_heads, row, &B.v_full[st]);
                }
                __syncwarp();
            }
            cur += x.p.b - x.p.a;
        }
        // copies in flight land before shared memory is released (without a timeout they were all waited for)
        for (uint32_t k = it > CM_STAGES ? it - CM_STAGES : 0; k < it; ++k) {
            mbar_wait(&B.k_full[k % CM_STAGES], (k / CM_STAGES) & 1, 10000000ull);
            mbar_wait(&B.v_full[k % CM_STAGES], (k / CM_STAGES) & 1, 10000000ull);
        }
        __syncwarp();
    }
    cm_before();
    __syncthreads();
    cm_after();
    if (warp == CM_SOFTMAX) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(CM_TMEM));
}

// Joins the items that cross_many_kernel cut.
template <typename T, int D>
__global__ void __launch_bounds__(32 * CJ_WARPS, 4) cross_join_kernel(const __grid_constant__ CrossParams A) {
    cm_join<D, false>(static_cast<const CmCut<CrossItem>*>(A.cuts), A.ctas, A.part,
                      [&](const CrossItem& x, int r, int ch, const float (&o)[CJ_CH], float top, float sum, float) {
                          const int at = x.row0 + r, tok = pd_div(at, A.by_rep);
                          const int64_t row = x.row + int64_t(tok) * A.Hq + at - tok * A.rep;
                          const float inv = cm_inverse(sum);
                          *reinterpret_cast<uint2*>(static_cast<T*>(A.out) + row * D + ch) =
                              uint2{pack_f32<T>(o[0] * inv, o[1] * inv), pack_f32<T>(o[2] * inv, o[3] * inv)};
                          if (ch == 0 && A.lse) A.lse[row] = sum == 0.f ? -INFINITY : top * 0.693147180559945309f + logf(sum);
                      });
}

}  // namespace kvb
