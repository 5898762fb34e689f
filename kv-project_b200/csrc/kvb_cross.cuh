// kvb_cross.cuh - attention of packed queries to keys of another length (an encoder's states), few queries per sequence.
//
//   s_j = lam q . k_j,  o = sum_j 2^(s_j - m) v_j / l,  l = sum_j 2^(s_j - m),  lam = scaling log2(e), over all keys of the
// sequence.
//
// The floor is the keys and values read once.  One persistent CTA per SM; a unit of work is 4 KB of keys and as much of
// values (16 keys at d = 128) of one (sequence, KV head, group of 16 query rows), and every CTA takes an equal run of units,
// found from the offsets inside the kernel: any mixture of lengths is balanced, nothing is planned before the launch.  Units
// go to the eight warps in turn; each warp copies its own units with TMA through its own ring (192 KB in flight per SM) and
// keeps its own running softmax; the warps are joined in shared memory at the end of a run, the CTAs of a cut run by
// the last one to arrive, in the order of the keys.  The rep query heads of a KV head and the sequence's queries are packed
// into the 16 rows of mma.sync; weights are rounded to the inputs' type (the product's operand).
//
// Values past a sequence's end belong to the next one: their weight is zero, but zero times NaN is not, so a unit that ends
// the sequence has those rows zeroed in shared memory first.
//
// Bound by HBM where there is enough to read: 48 single queries over 257 to 7258 keys (665 MB, 8 KV heads of 128 channels,
// bfloat16) take 115 us, 5.8 TB/s, 0.88 of the rate of a copy; tensor cores 19 % busy, issue slots 22 %.  One query over 1500
// keys takes 10 us: the offsets, the first copies and the joining, one after the other.
#pragma once
#include <cuda.h>

#include "kvb_paged_decode.cuh"
#include "kvb_prefill.cuh"

namespace kvb {

constexpr int CR_MAX_SEQS = 512;              // sequences of one launch
constexpr int CR_WARPS = 8;
constexpr int CR_ROWS = 16;
constexpr int CR_STAGES = 3;                  // per warp

struct CrossParams {
    CUtensorMap tm_k, tm_v;                   // (d, KV heads, nk), box 64 channels x 1 x unit
    const void* q;                            // (nq, Hq, d)
    int64_t q_row, q_head;
    const int32_t* cu_q;
    const int32_t* cu_k;
    int64_t nq, nk;
    int n, Hq, Hkv, rep;
    int k_heads, v_heads;                     // 0: all KV heads read head 0
    uint64_t by_rep;                          // for pd_div
    float lam;                                // scaling log2(e); cross_many_kernel: its magnitude, above 0
    int negate;                               // cross_many_kernel: scaling < 0
    void* out;                                // (nq, Hq, d)
    float* lse;                               // (nq, Hq) or null
    float* part;                              // two a CTA: O, maximum, sum
    uint32_t* count;                          // cross_few_kernel: [grid][8 warps]
    void* cuts;                               // cross_many_kernel: CmCut<CrossItem> a CTA
    int ctas;                                 // that take part
};

template <int D>
struct CrShape {
    static constexpr int KEYS = 2048 / D;                       // of a unit
    static constexpr int HALVES = D / 64;
    static constexpr int HALF = KEYS * 128;                     // bytes of 64 channels of a unit's keys
    static constexpr int SIDE = HALVES * HALF, STAGE = 2 * SIDE;
    static constexpr int JOIN = CR_WARPS * 8 * 68 * 4;          // the warps' O rows, 8 rows and 64 channels at a time
    static constexpr int PART = CR_ROWS * (D + 2);
    static constexpr int SMEM = 1024 + CR_WARPS * CR_STAGES * STAGE + JOIN;
};

// A sequence's rows, none where its offsets do not fit.
struct CrSeq {
    int q0, ql, k0, kl;
};

__device__ __forceinline__ CrSeq cr_seq(const int32_t* cu_q, const int32_t* cu_k, int64_t nq, int64_t nk, int s) {
    CrSeq x;
    x.q0 = cu_q[s];
    x.k0 = cu_k[s];
    const int64_t ql = int64_t(cu_q[s + 1]) - x.q0, kl = int64_t(cu_k[s + 1]) - x.k0;
    x.ql = int(ql);
    x.kl = int(kl);
    if (ql < 0 || kl < 0 || x.q0 < 0 || x.k0 < 0 || x.q0 + ql > nq || x.k0 + kl > nk) {
        raise_status(KVB_DEV_BOUNDS);
        x.ql = x.kl = 0;
    }
    return x;
}

// Units and places of a sequence: groups of ROWS query rows of the KV heads, units of KEYS keys.  None where they do not fit 32
// bits: it is left out.
template <int ROWS, int KEYS, int FIXED>
__device__ __forceinline__ void cr_work(const CrSeq& x, int rep, int Hkv, int& u, int& p) {
    const int64_t hg = (int64_t(x.ql) * rep + ROWS - 1) / ROWS * Hkv;
    const int units = max(1, (x.kl + KEYS - 1) / KEYS);          // without keys one empty unit: its rows are written
    const bool fits = hg <= INT_MAX && (int64_t(units) + FIXED) * hg <= INT_MAX;       // the product itself within 64 bits
    if (!fits) raise_status(KVB_DEV_BOUNDS);
    u = fits ? int(units * hg) : 0;
    p = fits ? int((units + FIXED) * hg) : 0;
}

template <typename T, int D>
__global__ void __launch_bounds__(32 * CR_WARPS, 1) cross_few_kernel(const __grid_constant__ CrossParams A) {
    using S = CrShape<D>;
    constexpr int KS = D / 16, CT = D / 8, NT = S::KEYS / 8;
    extern __shared__ uint8_t cr_raw[];
    __shared__ int pre[CR_MAX_SEQS + 1], shares[CR_MAX_SEQS + 1];        // units and places before each sequence
    __shared__ uint64_t full[CR_WARPS][CR_STAGES];
    __shared__ float s_m[CR_WARPS][CR_ROWS], s_l[CR_WARPS][CR_ROWS];
    __shared__ int warp_sum[2][CR_WARPS];
    __shared__ int s_abort;
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(cr_raw) + 1023) & ~uintptr_t(1023));
    float* join = reinterpret_cast<float*>(base + CR_WARPS * CR_STAGES * S::STAGE);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint8_t* ring = base + warp * CR_STAGES * S::STAGE;

    if (threadIdx.x == 0) {
        for (int i = 0; i < CR_WARPS * CR_STAGES; ++i) mbar_init(&full[0][i], 1);
        s_abort = 0;
        fence_mbar_init();
        pre[0] = shares[0] = 0;
    }
    chain_kernels();
    auto seq_at = [&](int i) { return cr_seq(A.cu_q, A.cu_k, A.nq, A.nk, i); };
    // units and places before each sequence: inclusive scans, a block of threads at a time
    int before_u = 0, before_p = 0;
    for (int i0 = 0; i0 < A.n; i0 += 32 * CR_WARPS) {
        const int i = i0 + threadIdx.x;
        int u = 0, p = 0;
        if (i < A.n) cr_work<CR_ROWS, S::KEYS, PD_FIXED>(seq_at(i), A.rep, A.Hkv, u, p);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int a = __shfl_up_sync(0xffffffffu, u, o), b = __shfl_up_sync(0xffffffffu, p, o);
            if (lane >= o) u += a, p += b;
        }
        __syncthreads();
        if (lane == 31) warp_sum[0][warp] = u, warp_sum[1][warp] = p;
        __syncthreads();
        int sum_u = 0, sum_p = 0;
        for (int w = 0; w < CR_WARPS; ++w) {
            if (w == warp) u += sum_u, p += sum_p;
            sum_u += warp_sum[0][w], sum_p += warp_sum[1][w];
        }
        if (i < A.n) pre[i + 1] = before_u + u, shares[i + 1] = before_p + p;
        before_u += sum_u, before_p += sum_p;
    }
    __syncthreads();
    bool fits = true;                                            // a sum that passed 32 bits shows as one that falls
    for (int i = threadIdx.x; i < A.n; i += 32 * CR_WARPS) fits &= shares[i + 1] >= shares[i] && pre[i + 1] >= pre[i];
    if (!__syncthreads_and(fits)) {
        if (threadIdx.x == 0) raise_status(KVB_DEV_BOUNDS);
        return;
    }
    const int work = shares[A.n];
    if (work == 0) return;
    PdPlan<true> W;
    W.pre = pre;
    W.shares = shares;
    W.n = A.n;
    W.hg = 0;
    W.ctas = max(1, min(int(gridDim.x), work / PD_LEAST));
    W.quota = work / W.ctas;
    W.extra = work - W.quota * W.ctas;
    const int cta = blockIdx.x;
    if (cta >= W.ctas) return;
    const int u0 = W.units_before(W.share(cta)), u1 = W.units_before(W.share(cta + 1));
    volatile int* abort = &s_abort;
    auto finite_ref = [](float m) { return m == -INFINITY ? 0.f : m; };

    // ---------------- copies: the warp's unit k is the CTA's unit warp + 8 k; lane i looks after the units k = i mod 32 ----------------
    const int mine = max(0, (u1 - u0 - warp + CR_WARPS - 1) / CR_WARPS);
    struct Place {
        int row, head;                                           // row < 0: no keys
    };
    auto place = [&](int k) {
        Place x{-1, 0};
        if (k >= mine) return x;
        const PdPiece p = pd_piece(W, u0 + warp + k * CR_WARPS, u1);
        const CrSeq s = seq_at(p.seq);
        if (s.kl == 0) return x;
        x.row = s.k0 + p.a * S::KEYS;
        x.head = p.vh / (W.heads(p.seq) / A.Hkv);
        return x;
    };
    Place at = place(lane), ahead{};
    int copied = 0;
    auto copy = [&]() {                                          // the warp's next unit
        if (copied >= mine) return;
        if ((copied & 31) == 0 && copied > 0) at = ahead;
        if (lane == (copied & 31)) {
            const int st = copied % CR_STAGES;
            uint64_t* bar = &full[warp][st];
            uint8_t* dst = ring + st * S::STAGE;
            mbar_arrive_expect_tx(bar, at.row >= 0 ? uint32_t(S::STAGE) : 0u);
            if (at.row >= 0) {
#pragma unroll
                for (int c = 0; c < S::HALVES; ++c) {
                    tma_load_3d(dst + c * S::HALF, &A.tm_k, 64 * c, at.head * A.k_heads, at.row, bar);
                    tma_load_3d(dst + S::SIDE + c * S::HALF, &A.tm_v, 64 * c, at.head * A.v_heads, at.row, bar);
                }
            }
        }
        if ((copied & 31) == 0) ahead = place(copied + 32 + lane);
        ++copied;
    };
    for (int i = 0; i < CR_STAGES; ++i) copy();

    // lane's addresses of the fragments within a half's tile: chunk c of row r lies at c ^ (r & 7)
    const int k_row = (lane >> 4) * 8 + (lane & 7), k_chunk = lane >> 3 & 1, v_row = (lane >> 3 & 1) * 8 + (lane & 7), v_chunk = lane >> 4;
    int first = 1, unit = 0;
    for (int cur = u0; cur < u1;) {
        const PdPiece p = pd_piece(W, cur, u1);
        const CrSeq sq = seq_at(p.seq);
        const int groups = W.heads(p.seq) / A.Hkv, h = p.vh / groups, row0 = (p.vh - h * groups) * CR_ROWS;
        const int nrows = min(sq.ql * A.rep - row0, CR_ROWS);
        auto row_at = [&](int r) {                               // (token, head) of row r, as a row of out
            const int tok = pd_div(row0 + r, A.by_rep);
            return (int64_t(sq.q0) + tok) * A.Hq + h * A.rep + row0 + r - tok * A.rep;
        };
        // ---- query rows as A operands: lane (g, t) holds rows g, g + 8 and channels 2 t .. of each 8
        uint32_t qf[KS][4];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            const int r = g + 8 * hf, tok = pd_div(row0 + r, A.by_rep);
            const bool ok = r < nrows;
            const T* q = static_cast<const T*>(A.q) + (ok ? (int64_t(sq.q0) + tok) * A.q_row + (h * A.rep + row0 + r - tok * A.rep) * A.q_head + 2 * t : 0);
#pragma unroll
            for (int c = 0; c < KS; ++c) {
                qf[c][hf] = ok ? __ldg(reinterpret_cast<const uint32_t*>(q + 16 * c)) : 0u;
                qf[c][hf + 2] = ok ? __ldg(reinterpret_cast<const uint32_t*>(q + 16 * c + 8)) : 0u;
            }
        }
        float o[CT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int c = 0; c < CT; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;
        const int lead = (cur - u0) % CR_WARPS;
        for (int k = warp < lead ? warp - lead + CR_WARPS : warp - lead; k < p.b - p.a; k += CR_WARPS, ++unit) {
            const int st = unit % CR_STAGES;
            const bool there = !*abort && mbar_wait(&full[warp][st], (unit / CR_STAGES) & 1);
            if (!__all_sync(0xffffffffu, there)) {
                *abort = 1;
                continue;
            }
            const int left = sq.kl - (p.a + k) * S::KEYS;        // keys of the sequence from this unit on
            uint8_t* kt = ring + st * S::STAGE;
            const uint32_t ks = smem_u32(kt), vs = ks + S::SIDE;
            if (left < S::KEYS) {
                // values past the end become zeros (8 lanes a row); async copies to the stage come after these writes
                for (int r = max(left, 0) + (lane >> 3); r < S::KEYS; r += 4)
#pragma unroll
                    for (int c = 0; c < S::HALVES; ++c) *reinterpret_cast<uint4*>(kt + S::SIDE + c * S::HALF + r * 128 + (lane & 7) * 16) = uint4{0, 0, 0, 0};
                fence_proxy_async_smem();
                __syncwarp();
            }
            if (left > 0) {
                float s[NT][4];
#pragma unroll
                for (int c = 0; c < NT; ++c) s[c][0] = s[c][1] = s[c][2] = s[c][3] = 0.f;
#pragma unroll
                for (int c = 0; c < KS; ++c)
#pragma unroll
                    for (int x = 0; x < NT / 2; ++x) {
                        uint32_t b[4];
                        const int row = 16 * x + k_row, chunk = (2 * c + k_chunk) & 7;
                        pf_ldmatrix(b, ks + (c >> 2) * S::HALF + row * 128 + ((chunk ^ (row & 7)) * 16));
                        pf_mma<T>(s[2 * x], qf[c], b[0], b[1]);
                        pf_mma<T>(s[2 * x + 1], qf[c], b[2], b[3]);
                    }
#pragma unroll
                for (int c = 0; c < NT; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[c][i] *= A.lam;
                if (left < S::KEYS) {
#pragma unroll
                    for (int c = 0; c < NT; ++c)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (8 * c + 2 * t + (i & 1) >= left) s[c][i] = -INFINITY;
                }
                bool grow = false;
                float top[2];
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    top[hf] = -INFINITY;
#pragma unroll
                    for (int c = 0; c < NT; ++c) top[hf] = fmaxf(top[hf], fmaxf(s[c][2 * hf], s[c][2 * hf + 1]));
                    grow |= top[hf] > m[hf] + PD_LAZY;
                }
                if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        float y = top[hf];
                        y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 1));
                        y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 2));
                        const float f = y > m[hf] + PD_LAZY ? ex2(m[hf] - y) : 1.f;
                        if (y > m[hf] + PD_LAZY) m[hf] = y;
                        l[hf] *= f;
#pragma unroll
                        for (int c = 0; c < CT; ++c) o[c][2 * hf] *= f, o[c][2 * hf + 1] *= f;
                    }
                }
                const float ref[2] = {finite_ref(m[0]), finite_ref(m[1])};
#pragma unroll
                for (int c = 0; c < NT; ++c) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[c][i] = ex2(s[c][i] - ref[i >> 1]);
                    l[0] += s[c][0] + s[c][1];
                    l[1] += s[c][2] + s[c][3];
                }
#pragma unroll
                for (int x = 0; x < NT / 2; ++x) {
                    const uint32_t pa[4] = {pack_f32<T>(s[2 * x][0], s[2 * x][1]), pack_f32<T>(s[2 * x][2], s[2 * x][3]),
                                            pack_f32<T>(s[2 * x + 1][0], s[2 * x + 1][1]), pack_f32<T>(s[2 * x + 1][2], s[2 * x + 1][3])};
#pragma unroll
                    for (int c = 0; c < CT / 2; ++c) {
                        uint32_t b[4];
                        const int row = 16 * x + v_row, chunk = (2 * c + v_chunk) & 7;
                        pf_ldmatrix_trans(b, vs + (c >> 2) * S::HALF + row * 128 + ((chunk ^ (row & 7)) * 16));
                        pf_mma<T>(o[2 * c], pa, b[0], b[1]);
                        pf_mma<T>(o[2 * c + 1], pa, b[2], b[3]);
                    }
                }
            }
            __syncwarp();                                        // every lane has read the stage: refill it
            copy();
        }
        // ---- join the warps: warp w the rows w and 8 + w, 64 channels at a time
        const bool whole = p.a == 0 && p.b == p.units;
        const int c0 = whole ? 0 : W.holder(p.v0 + PD_FIXED), c1 = whole ? 0 : W.holder(p.v0 + PD_FIXED + p.units - 1);
        __syncthreads();                                         // the last join's reads are done
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 1);
            l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 2);
            if (t == 0) s_m[warp][g + 8 * hf] = m[hf], s_l[warp][g + 8 * hf] = l[hf];
        }
        float* part = A.part + int64_t(2 * blockIdx.x + (first ? 0 : 1)) * S::PART;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            if (8 * hf >= nrows) break;
            const int r = warp + 8 * hf;
            float top = -INFINITY, sum = 0.f, f[CR_WARPS];
#pragma unroll
            for (int y = 0; y < S::HALVES; ++y) {
                if (hf + y > 0) __syncthreads();
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    *reinterpret_cast<float2*>(join + (warp * 8 + g) * 68 + 8 * c + 2 * t) = float2{o[8 * y + c][2 * hf], o[8 * y + c][2 * hf + 1]};
                __syncthreads();
                if (y == 0) {
#pragma unroll
                    for (int w = 0; w < CR_WARPS; ++w) top = fmaxf(top, s_m[w][r]);
                    const float ref = finite_ref(top);
#pragma unroll
                    for (int w = 0; w < CR_WARPS; ++w) {
                        f[w] = ex2(s_m[w][r] - ref);
                        sum = __fmaf_rn(s_l[w][r], f[w], sum);
                    }
                }
                float2 acc{0.f, 0.f};
#pragma unroll
                for (int w = 0; w < CR_WARPS; ++w) {
                    const float2 v = *reinterpret_cast<const float2*>(join + (w * 8 + warp) * 68 + 2 * lane);
                    acc.x = __fmaf_rn(v.x, f[w], acc.x);
                    acc.y = __fmaf_rn(v.y, f[w], acc.y);
                }
                if (r < nrows) {
                    if (whole) {
                        const float inv = sum > 0.f ? 1.f / sum : (sum == sum ? 0.f : sum);
                        *reinterpret_cast<uint32_t*>(static_cast<T*>(A.out) + row_at(r) * D + 64 * y + 2 * lane) = pack_f32<T>(acc.x * inv, acc.y * inv);
                    } else {
                        *reinterpret_cast<float2*>(part + r * D + 64 * y + 2 * lane) = acc;
                    }
                }
            }
            if (lane == 0 && r < nrows) {
                if (!whole) {
                    part[CR_ROWS * D + r] = top;
                    part[CR_ROWS * D + CR_ROWS + r] = sum;
                } else if (A.lse) {
                    A.lse[row_at(r)] = sum == 0.f ? -INFINITY : top * 0.693147180559945309f + logf(sum);
                }
            }
        }
        if (!whole && warp < nrows) {
            // each warp for its rows: the last CTA to arrive joins the CTAs' partials
            uint32_t* count = A.count + c0 * CR_WARPS + warp;
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
#pragma unroll 1
                for (int r = warp; r < nrows; r += 8) {
                    float top = -INFINITY, sum = 0.f;
                    float2 acc[S::HALVES];
#pragma unroll
                    for (int y = 0; y < S::HALVES; ++y) acc[y] = float2{0.f, 0.f};
                    for (int cc = c0; cc <= c1; cc += 32) {      // 32 partials: a lane has the maximum and sum of one
                        const int cnt = min(32, c1 - cc + 1);
                        const float* ml = slot_of(min(cc + lane, c1)) + CR_ROWS * D + r;
                        const float ms = lane < cnt ? __ldcg(ml) : -INFINITY, ls = lane < cnt ? __ldcg(ml + CR_ROWS) : 0.f;
                        const float to = fmaxf(top, warp_max(ms)), ref = finite_ref(to), old = ex2(top - ref), f = ex2(ms - ref);
                        sum = __fmaf_rn(sum, old, kvb::warp_sum(ls * f));
                        top = to;
#pragma unroll
                        for (int y = 0; y < S::HALVES; ++y) acc[y].x *= old, acc[y].y *= old;
#pragma unroll 8
                        for (int k = 0; k < cnt; ++k) {
                            const float* from = slot_of(cc + k) + r * D + 2 * lane;
                            const float fk = __shfl_sync(0xffffffffu, f, k);
#pragma unroll
                            for (int y = 0; y < S::HALVES; ++y) {
                                const float2 v = __ldcg(reinterpret_cast<const float2*>(from + 64 * y));
                                acc[y].x = __fmaf_rn(v.x, fk, acc[y].x);
                                acc[y].y = __fmaf_rn(v.y, fk, acc[y].y);
                            }
                        }
                    }
                    const float inv = sum > 0.f ? 1.f / sum : (sum == sum ? 0.f : sum);
                    const int64_t row = row_at(r);
#pragma unroll
                    for (int y = 0; y < S::HALVES; ++y)
                        *reinterpret_cast<uint32_t*>(static_cast<T*>(A.out) + row * D + 64 * y + 2 * lane) = pack_f32<T>(acc[y].x * inv, acc[y].y * inv);
                    if (lane == 0 && A.lse) A.lse[row] = sum == 0.f ? -INFINITY : top * 0.693147180559945309f + logf(sum);
                }
            }
        }
        cur += p.b - p.a;
        first = 0;
    }
    if (*abort && lane == 0) {                                   // copies in flight land before shared memory is released
        raise_status(KVB_DEV_TIMEOUT);
        for (int k = max(0, copied - CR_STAGES); k < copied; ++k) mbar_wait(&full[warp][k % CR_STAGES], (k / CR_STAGES) & 1, 10000000ull);
    }
    __syncthreads();
}

}  // namespace kvb
