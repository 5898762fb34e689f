// kvb_prefill.cuh - causal attention of packed prompts.
//
//   S = Q K^T,  x = scaling log2(e) S,  m = running row maximum of x,  P = 2^(x - m),  l = sum P,  O = P V,
//   out = O / l,  lse = ln 2 m + ln l, over the keys j <= i + (keys - queries) that a query sees.
//
// One pass over the keys with the running maximum and sum of a softmax.  The `rep` query heads of a KV head are
// packed into the tile's rows (row = token * rep + head in the group), so a tile of 128 rows is 128 / rep tokens of
// one KV head and a short chunk still fills it.  A CTA of four warps computes one tile, or a piece of one; a warp has 32
// rows, so that each fragment of K and V read from shared memory serves two products.  Keys and values come in steps of 64
// through two buffers filled by cp.async, one barrier a step: the copies of the next step leave when everyone has left the
// buffer.  Two CTAs share an SM, so that one's softmax runs beside the other's products.  S and O stay in registers, P
// is rounded to the inputs' type (it is the product's operand) and never leaves them.  O is rescaled only when a
// row's maximum grew by more than 2^8 (P then reaches 256 at most, well inside float16's range; the sums stay in
// float32), which is seldom after the first steps.
//
// The products are mma.sync: a kernel on tcgen05 (operands by TMA, S, P and O in tensor memory) stood here that was more
// than twice as fast, and ended in an illegal access in replayed graphs and, in an earlier form, in some of many plain
// calls, without a cause that reading could name.  This one has nothing that outlives an instruction but the copies
// of cp.async, which are waited for before the buffers are read and before the CTA leaves; no wait for another thread but
// the block's barrier; and every address it forms is that of a row below the sequence's length or of a slot below the
// workspace's.
//
// Masks: logits of keys past a row's limit become -inf by selection, so what lies there does not matter; values
// there would still meet a weight of zero in the product (0 * NaN), so rows past the sequence are filled with zeros, and in
// steps that some row of the tile does not see whole, non-finite entries of the sequence's own later tokens become zeros in
// shared memory, and the rows that do see them get them added back at the end.
//
// Work items are placed in descending order of their steps, a CTA each; the hardware hands them out as CTAs end.  Items
// of more steps than a CTA's fair share (few rows over long keys) come first, cut into equal pieces of at most that many:
// each piece leaves its O, m and l in the workspace, and the warp that completes the last piece of its 32 rows joins them
// in the order of the keys.  Every CTA finds its item from the lengths (bisection on the step count, sums of step counts in
// closed form, a warp's lanes over the sequences), so no plan is built before the launch.
//
// In a loop: 16384 tokens, 32 heads over 8, d 128: 5440 us (404 TFLOP/s); 8 packed prompts of 7208 tokens in all: 376; chunks
// of 500 and 1100 tokens after prefixes of 7000 and 333, 16 heads over 4, d 64: 87; one prompt of 77 tokens: 14.6, of
// which the code's first fetch is most (with one pass over 256 rows of records at the end of an item instead of 8 words: 25).
#pragma once
#include <climits>
#include <type_traits>

#include "kvb_common.cuh"
#include "kvb_pages_view.cuh"

namespace kvb {

constexpr int PF_ROWS = 128;
constexpr int PF_KT = 64;                     // keys per step
constexpr int PF_THREADS = 128;
constexpr int PF_CTAS_PER_SM = 2;
constexpr float PF_LAZY = 8.f;                // log2 of how far a maximum may grow before O is rescaled

struct PrefillParams {
    const void* q;                            // (nq, Hq, d)
    const void* k;                            // (nk, Hkv, d)
    const void* v;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;
    const int32_t* cu_q;
    const int32_t* cu_k;
    int64_t nq, nk;
    int n, Hq, Hkv, rep, tt;                  // tt = 128 / rep tokens per tile
    int by_rep;                               // 65536 / rep + 1: r / rep = r by_rep / 65536 for r < 128
    int ctas;                                 // that run at a time; pieces have 2 ctas slots
    float* part;                              // [2 ctas][d + 2][128]: O by register and thread, m and l by row; null: no item is cut
    uint32_t* count;                          // [2 ctas][4 warps], see pf_arrive
    uint32_t call;                            // number of this call, 1 .. 2^20 - 1
    float lam;                                // |scaling| log2(e), > 0
    int negate;                               // scaling < 0
    void* out;                                // (nq, Hq, d)
    float* lse;                               // (nq, Hq) or null
};

template <int D>
struct PfShape {
    static constexpr int ROW = 2 * D;                           // bytes
    static constexpr int CHUNKS = D / 8;                        // of 16 bytes
    static constexpr int TILE = PF_KT * ROW;
    static constexpr int SMEM = PF_ROWS * ROW + 4 * TILE;
};

struct PfItem {
    int q0, ql, k0, kl;                       // the sequence's rows
    int t0;                                   // first token within it
    int head;                                 // KV head; < 0: no work
    int j0, n;                                // first step and steps of this piece
    int piece, first, pieces;                 // number of this piece and of the item's first; how many the item has
    int jm;                                   // first step that some row does not see whole
};

// ---------------------------------------------------------------------------------------------
// Work items: those of more steps than the fair share, in pieces, then the others in descending order of steps.
// ---------------------------------------------------------------------------------------------
struct PfSeq {
    int q0, ql, k0, kl, tiles;
};

__device__ __forceinline__ PfSeq pf_seq(const PrefillParams& A, int s) {
    PfSeq q{0, 0, 0, 0, 0};
    if (s < A.n) {
        q.q0 = A.cu_q[s];
        q.ql = A.cu_q[s + 1] - q.q0;
        q.k0 = A.cu_k[s];
        q.kl = A.cu_k[s + 1] - q.k0;
        if (q.ql <= 0) q.ql = 0;
        else if (q.q0 < 0 || q.k0 < 0 || q.kl < 0 || int64_t(q.q0) + q.ql > A.nq || int64_t(q.k0) + q.kl > A.nk) {
            raise_status(KVB_DEV_BOUNDS);
            q.ql = q.kl = 0;
        }
        q.tiles = int((int64_t(q.ql) + A.tt - 1) / A.tt);
    }
    return q;
}

// How many of a sequence's tiles have t steps or more: tile p ends at the query min(tt (p + 1), ql), which sees kl - ql +
// that many keys.
__device__ __forceinline__ int pf_count(const PfSeq& q, int t, int tt) {
    if (t <= 0) return q.tiles;
    const int need = PF_KT * (t - 1) + 1;
    if (q.kl < need) return 0;
    const int first = max(need - q.kl + q.ql + tt - 1, 0) / tt - 1;      // ceil(..) - 1
    return q.tiles - min(max(first, 0), q.tiles - 1);
}

__device__ __forceinline__ int pf_warp_sum(int v) { return __reduce_add_sync(0xffffffffu, v); }

// sum over i < n of floor((a i + b) / m), for a, b >= 0 (the Euclidean reduction of a and the divisor).  Intermediate
// values stay below 2^32: n is a count of tiles, whose rows have to fit the GPU's memory.
__device__ __forceinline__ uint32_t pf_floor_sum(uint32_t n, uint32_t m, uint32_t a, uint32_t b) {
    uint32_t sum = 0;
    while (n > 0) {
        const uint32_t qa = a / m, qb = b / m;
        sum += qa * uint32_t(uint64_t(n) * (n - 1) / 2) + qb * n;
        a -= qa * m;
        b -= qb * m;
        const uint32_t y = a * n + b;
        if (y < m) break;
        n = y / m;
        b = y - n * m;
        const uint32_t t = m;
        m = a;
        a = t;
    }
    return sum;
}

// Pieces of up to `keys` keys (a multiple of the step) in the tiles before p, a tile counting one at least unless it sees
// no key.
__device__ __forceinline__ int pf_pieces(const PfSeq& q, int p, int tt, uint32_t keys) {
    const int full = min(p, q.tiles - 1), a = q.kl - q.ql;                     // tiles that end before the sequence does
    const int i0 = a < 0 ? min(-a / tt, full) : 0;                             // those before see no key
    int c = full > i0 ? int(pf_floor_sum(full - i0, keys, tt, uint32_t(a + tt * (i0 + 1)) + keys - 1)) : 0;
    if (p == q.tiles && p > 0) c += int((uint32_t(q.kl) + keys - 1) / keys);
    return c;
}

// The steps j0 .. j1 - 1 of a tile (out: its sequence and head).
__device__ __forceinline__ void pf_steps_of(const PrefillParams& A, int tile, int j0, int j1, PfItem& out) {
    out.t0 = tile * A.tt;
    out.j0 = j0;
    const int keys = min(max(out.kl - out.ql + min(out.t0 + A.tt, out.ql), 0), out.kl);
    out.n = max(min((keys + PF_KT - 1) / PF_KT, j1) - j0, 0);
    out.jm = max(out.kl - out.ql + out.t0 + 1, 0) / PF_KT;
}

constexpr int PF_SHARE = 16;                  // items of fewer steps are never cut

struct PfCuts {
    int share;                                // items of more steps are cut into pieces of at most so many
    int items;                                // how many are,
    int pieces;                               // into how many pieces
};

// The fair share (not below 16 steps), and what it cuts; whole warp.  The share is that of a bound on the number of
// steps, at most a step an item too high; so there are at most 2 ctas pieces, each having half a share or more.
// Item and piece counts fit 32 bits by far: 128 query rows an item.
__device__ __forceinline__ PfCuts pf_cuts(const PrefillParams& A) {
    const int lane = threadIdx.x & 31;
    PfCuts c{INT_MAX, 0, 0};
    if (!A.part) return c;
    float steps = 0.f;
    int most = 0;
    for (int s0 = 0; s0 < A.n; s0 += 32) {
        const PfSeq q = pf_seq(A, s0 + lane);
        if (q.tiles == 0) continue;
        // the tiles from the first that sees a key on end at a + tt (i + 1) keys or before
        const int a = q.kl - q.ql, i0 = a < 0 ? min(-a / A.tt, q.tiles) : 0;
        const float k = float(q.tiles - i0);
        steps += k * (float(a) + float(A.tt) * (float(i0) + 0.5f * (k + 1.f))) * (1.f / PF_KT) + k;
        most = max(most, (q.kl + PF_KT - 1) / PF_KT);
    }
    steps = warp_sum(steps) * float(A.Hkv);
    most = __reduce_max_sync(0xffffffffu, most);
    const float share = fmaxf(float(PF_SHARE), steps * 1.0001f / float(A.ctas) + 1.f);
    if (float(most) <= share) return c;
    c.share = int(share);
    for (int s0 = 0; s0 < A.n; s0 += 32) {
        const PfSeq q = pf_seq(A, s0 + lane);
        const int cut = q.tiles ? pf_count(q, c.share + 1, A.tt) : 0;
        const uint32_t keys = uint32_t(c.share) * PF_KT;
        c.items += cut * A.Hkv;
        if (cut) c.pieces += (pf_pieces(q, q.tiles, A.tt, keys) - pf_pieces(q, q.tiles - cut, A.tt, keys)) * A.Hkv;
    }
    c.items = __reduce_add_sync(0xffffffffu, c.items);
    c.pieces = __reduce_add_sync(0xffffffffu, c.pieces);
    // more pieces than slots would need offsets that do not ascend: then nothing is cut
    return c.pieces <= 2 * A.ctas ? c : PfCuts{INT_MAX, 0, 0};
}

// Piece `idx` of the cut items; whole warp.
__device__ __forceinline__ void pf_piece(const PrefillParams& A, const PfCuts& cuts, int idx, PfItem& out) {
    const int lane = threadIdx.x & 31;
    const uint32_t keys = uint32_t(cuts.share) * PF_KT;
    int r = idx;
    for (int s0 = 0; s0 < A.n; s0 += 32) {
        const PfSeq q = pf_seq(A, s0 + lane);
        const int cut = q.tiles ? pf_count(q, cuts.share + 1, A.tt) : 0;
        const int before = cut ? pf_pieces(q, q.tiles - cut, A.tt, keys) : 0;
        const int per = cut ? pf_pieces(q, q.tiles, A.tt, keys) - before : 0;                  // pieces of one head
        int x = per * A.Hkv;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        const uint32_t after = __ballot_sync(0xffffffffu, x > r);
        if (after == 0) {
            r -= __shfl_sync(0xffffffffu, x, 31);
            continue;
        }
        const int src = __ffs(int(after)) - 1;
        PfSeq c;
        c.q0 = __shfl_sync(0xffffffffu, q.q0, src);
        c.ql = __shfl_sync(0xffffffffu, q.ql, src);
        c.k0 = __shfl_sync(0xffffffffu, q.k0, src);
        c.kl = __shfl_sync(0xffffffffu, q.kl, src);
        c.tiles = __shfl_sync(0xffffffffu, q.tiles, src);
        r -= __shfl_sync(0xffffffffu, x - per * A.Hkv, src);
        const int one = __shfl_sync(0xffffffffu, per, src), skipped = __shfl_sync(0xffffffffu, before, src);
        const int head = r / one;
        r -= head * one;
        // the last tile whose pieces begin at or before r, by 32-way search
        int lo = c.tiles - __shfl_sync(0xffffffffu, cut, src), len = c.tiles - lo, at = 0;
        while (true) {
            const int step = (len + 31) / 32, p = lo + lane * step;
            const int v = p < lo + len ? pf_pieces(c, p, A.tt, keys) - skipped : 0;
            const int k = 31 - __clz(int(__ballot_sync(0xffffffffu, p < lo + len && v <= r) | 1u));
            at = __shfl_sync(0xffffffffu, v, k);
            lo += k * step;
            len = min(step, c.tiles - lo);
            if (step == 1) break;
        }
        out.q0 = c.q0, out.ql = c.ql, out.k0 = c.k0, out.kl = c.kl;
        out.head = head;
        const int e = c.kl - c.ql + min(A.tt * (lo + 1), c.ql), steps = (e + PF_KT - 1) / PF_KT, k = r - at;
        out.pieces = (steps + cuts.share - 1) / cuts.share;
        out.piece = idx;
        out.first = idx - k;
        pf_steps_of(A, lo, int(int64_t(steps) * k / out.pieces), int(int64_t(steps) * (k + 1) / out.pieces), out);
        return;
    }
}

// Item `idx`.  Whole warp; false when there are no more.
__device__ __forceinline__ bool pf_item(const PrefillParams& A, const PfCuts& cuts, int idx, PfItem& out) {
    const int lane = threadIdx.x & 31;
    if (idx < cuts.pieces) {
        pf_piece(A, cuts, idx, out);
        return true;
    }
    idx += cuts.items - cuts.pieces;              // place among all items by their steps
    const PfSeq mine = pf_seq(A, lane);
    auto total = [&](int steps) {                 // items of `steps` steps or more
        int c = mine.tiles ? pf_count(mine, steps, A.tt) : 0;
        for (int s0 = 32; s0 < A.n; s0 += 32) {
            const PfSeq q = pf_seq(A, s0 + lane);
            if (q.tiles) c += pf_count(q, steps, A.tt);
        }
        return pf_warp_sum(c) * A.Hkv;
    };
    if (idx >= total(0)) return false;
    int most = (mine.kl + PF_KT - 1) / PF_KT;
    for (int s0 = 32; s0 < A.n; s0 += 32) most = max(most, (pf_seq(A, s0 + lane).kl + PF_KT - 1) / PF_KT);
    // the largest t with total(t) > idx, and total(t + 1); items of more than the share are the cut ones
    int lo = 0, hi = min(__reduce_max_sync(0xffffffffu, most), cuts.share), above = cuts.items;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2, m = total(mid);
        if (m > idx) lo = mid;
        else {
            hi = mid - 1;
            above = m;
        }
    }
    int r = idx - above;                          // rank among the items of lo steps
    for (int s0 = 0; s0 < A.n; s0 += 32) {
        const PfSeq q = s0 == 0 ? mine : pf_seq(A, s0 + lane);
        const int before = q.tiles ? pf_count(q, lo + 1, A.tt) : 0, c = (q.tiles ? pf_count(q, lo, A.tt) : 0) - before;
        int x = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        const int sum = __shfl_sync(0xffffffffu, x, 31) * A.Hkv;
        if (r >= sum) { r -= sum; continue; }
        const int src = __ffs(int(__ballot_sync(0xffffffffu, x * A.Hkv > r))) - 1;
        out.q0 = __shfl_sync(0xffffffffu, q.q0, src);
        out.ql = __shfl_sync(0xffffffffu, q.ql, src);
        out.k0 = __shfl_sync(0xffffffffu, q.k0, src);
        out.kl = __shfl_sync(0xffffffffu, q.kl, src);
        r -= __shfl_sync(0xffffffffu, x - c, src) * A.Hkv;
        const int step = r / A.Hkv;
        out.head = r - step * A.Hkv;
        out.first = out.piece = 0;
        out.pieces = 1;
        pf_steps_of(A, __shfl_sync(0xffffffffu, q.tiles - before - c, src) + step, 0, INT_MAX, out);
        return true;
    }
    return false;
}

// ---------------------------------------------------------------------------------------------
// Copies, fragments, products
// ---------------------------------------------------------------------------------------------
// 16 bytes to shared memory, zeros where `ok` is false (nothing is read then)
__device__ __forceinline__ void pf_copy16(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void pf_copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Byte offset of a 16-byte chunk of a row: eight rows' chunks of one number meet eight different banks
template <int D>
__device__ __forceinline__ uint32_t pf_at(int row, int chunk) {
    return uint32_t(row * (2 * D) + (((chunk ^ row) & 7) | (chunk & 8)) * 16);
}

__device__ __forceinline__ void pf_ldmatrix(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void pf_ldmatrix_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

template <typename T>
__device__ __forceinline__ void pf_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        mma16816(d, a, b0, b1);
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Whether one of eight values is not finite: x * 0 is NaN for NaN and infinities only.
template <typename T>
__device__ __forceinline__ bool pf_not_finite(const uint4& w) {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const uint32_t zero = 0, a[4] = {w.x, w.y, w.z, w.w};
    const T2 z = *reinterpret_cast<const T2*>(&zero);
    T2 s = z;
#pragma unroll
    for (int i = 0; i < 4; ++i) s = __hfma2(*reinterpret_cast<const T2*>(&a[i]), z, s);
    return __hisnan(s.x) || __hisnan(s.y);
}

// A piece's warp is done with its rows: true for the last of `pieces` to arrive.  The word holds the number of the call
// (20 bits) and how many have arrived (12 bits); the last one leaves zero.  A word that an unfinished call, or a
// workspace that was not zero-filled, left behind names another call: it is counted from the start, and reported.
__device__ __forceinline__ bool pf_arrive(uint32_t* word, uint32_t call, uint32_t pieces) {
    uint32_t seen = *reinterpret_cast<volatile uint32_t*>(word), want, n;
    do {
        want = seen;
        n = (want >> 12) == call ? (want & 0xfffu) + 1 : 1;
        seen = atomicCAS(word, want, n == pieces ? 0u : call << 12 | n);
    } while (seen != want);
    if (want != 0 && (want >> 12) != call) raise_status(KVB_DEV_WORKSPACE);
    return n == pieces;
}

template <typename T, int D>
__global__ void __launch_bounds__(PF_THREADS, PF_CTAS_PER_SM) prefill_kernel(const __grid_constant__ PrefillParams A) {
    using S = PfShape<D>;
    constexpr int NT = PF_KT / 8, CT = D / 8;                    // column tiles of S (keys) and of O (channels)
    constexpr int LOADS = PF_KT * S::CHUNKS / PF_THREADS;        // 16-byte copies of a thread for K, and for V, a step
    constexpr int LSTEP = PF_THREADS / S::CHUNKS;                // rows between them
    extern __shared__ __align__(128) uint8_t pf_smem[];
    __shared__ PfItem s_item;
    __shared__ uint32_t s_bad[4][2];                             // non-finite value rows of the steps jm ..
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t sq = smem_u32(pf_smem), sk = sq + PF_ROWS * S::ROW, sv = sk + 2 * S::TILE;

    if (warp == 0) {
        const PfCuts cuts = pf_cuts(A);
        PfItem x;
        bool more = pf_item(A, cuts, int(blockIdx.x), x);
        if (lane == 0) {
            s_item = x;
            if (!more) s_item.head = -1;
        }
        if (lane < 8) s_bad[lane >> 1][lane & 1] = 0;
        // offsets that do not ascend may hold more rows than the grid was made for
        if (blockIdx.x + 1 == gridDim.x && more && pf_item(A, cuts, int(gridDim.x), x) && lane == 0) raise_status(KVB_DEV_BOUNDS);
    }
    __syncthreads();
    const PfItem& x = s_item;
    if (x.head < 0) return;

    // ---------------- this thread's copies ----------------
    const int lrow = threadIdx.x / S::CHUNKS, lchunk = threadIdx.x % S::CHUNKS;
    const T* kp = static_cast<const T*>(A.k) + (int64_t(x.k0) + x.j0 * PF_KT + lrow) * A.k_row + x.head * A.k_head + lchunk * 8;
    const T* vp = static_cast<const T*>(A.v) + (int64_t(x.k0) + x.j0 * PF_KT + lrow) * A.v_row + x.head * A.v_head + lchunk * 8;
    int left = x.kl - x.j0 * PF_KT - lrow;                       // of the sequence's rows, from the next to be copied on
    const uint32_t ldst = pf_at<D>(lrow, lchunk);                // rows 8 apart have their chunks in the same places
    auto load = [&](int j) {                                     // the next step, to buffer j & 1
        const uint32_t to = ldst + uint32_t(j & 1) * S::TILE;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const bool ok = left > i * LSTEP;                    // past them zeros, and no address that is not a row's
            pf_copy16(sk + to + i * LSTEP * S::ROW, ok ? kp : static_cast<const T*>(A.k), ok);
            pf_copy16(sv + to + i * LSTEP * S::ROW, ok ? vp : static_cast<const T*>(A.v), ok);
            kp += LSTEP * A.k_row;
            vp += LSTEP * A.v_row;
        }
        left -= PF_KT;
    };
    // token of a row of the tile, its query head in `head`; < 0: no row
    auto token = [&](int row, int& head) {
        const int tok = row * A.by_rep >> 16;
        head = x.head * A.rep + row - tok * A.rep;
        return tok < A.tt && unsigned(x.t0 + tok) < unsigned(x.ql) ? x.t0 + tok : -1;
    };
    if (x.n > 0) {
#pragma unroll
        for (int i = 0; i < PF_ROWS / LSTEP; ++i) {
            int head;
            const int row = lrow + i * LSTEP, tok = token(row, head);
            const T* q = static_cast<const T*>(A.q) + (tok < 0 ? 0 : int64_t(x.q0 + tok) * A.q_row + head * A.q_head + lchunk * 8);
            pf_copy16(sq + pf_at<D>(row, lchunk), q, tok >= 0);
        }
        load(0);
    }

    // ---------------- this thread's rows: 32 warp + 16 mt + 8 hf + g ----------------
    int lim[2][2], lo = INT_MAX, hi = 0;                         // keys that a row sees; the warp's least and most
    bool used = false;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            int head;
            const int tok = token(warp * 32 + mt * 16 + hf * 8 + g, head);
            lim[mt][hf] = tok < 0 ? x.kl : min(max(x.kl - x.ql + tok + 1, 0), x.kl);       // rows of no token mask nothing
            if (tok < 0) continue;
            used = true;
            lo = min(lo, lim[mt][hf]);
            hi = max(hi, lim[mt][hf]);
        }
    used = __any_sync(0xffffffffu, used);
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);

    float o[2][CT][4], m[2][2], l[2][2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
        m[mt][0] = m[mt][1] = -INFINITY;
        l[mt][0] = l[mt][1] = 0.f;
#pragma unroll
        for (int c = 0; c < CT; ++c) o[mt][c][0] = o[mt][c][1] = o[mt][c][2] = o[mt][c][3] = 0.f;
    }
    // a lane's addresses of the fragments: those of the even chunk c, 16 rows on a constant further
    const uint32_t q_lane = sq + pf_at<D>(warp * 32 + (lane & 15), lane >> 4), k_lane = pf_at<D>((lane >> 4) * 8 + (lane & 7), lane >> 3 & 1),
                   v_lane = pf_at<D>((lane >> 3 & 1) * 8 + (lane & 7), lane >> 4);
    auto chunk = [](uint32_t at, int c) { return (at ^ ((c & 6) * 16)) + (c & 8) * 16; };

    for (int j = 0; j < x.n; ++j) {
        pf_copies_done();
        __syncthreads();                                         // the step's rows are there, and the other buffer is left
        if (j + 1 < x.n) load(j + 1);
        const uint32_t kt = sk + k_lane + uint32_t(j & 1) * S::TILE, vt = sv + v_lane + uint32_t(j & 1) * S::TILE;
        const int key0 = (x.j0 + j) * PF_KT;
        const bool mend = x.j0 + j >= x.jm;
        if (mend) {                                              // value rows that some row does not see: see the head of this file
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int row = lrow + i * LSTEP;
                T* e = reinterpret_cast<T*>(pf_smem + (sv - sq) + uint32_t(j & 1) * S::TILE + ldst + i * LSTEP * S::ROW);
                if (!pf_not_finite<T>(*reinterpret_cast<const uint4*>(e))) continue;
                for (int c = 0; c < 8; ++c)
                    if (!(fabsf(to_f32(e[c])) < INFINITY)) e[c] = from_f32<T>(0.f);
                atomicOr(&s_bad[x.j0 + j - x.jm][row >> 5], 1u << (row & 31));
            }
            __syncwarp();                                        // the products below want the lanes together
        }
        const bool seen = key0 < hi;                             // by some row of the warp
        uint32_t p[2][NT / 2][4];
        if (seen) {
            float s[2][NT][4];
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int c = 0; c < NT; ++c) s[mt][c][0] = s[mt][c][1] = s[mt][c][2] = s[mt][c][3] = 0.f;
#pragma unroll 4                             // a step's code is fetched as it runs: whole 384 us for the packed prompts below, 376, by two 385
            for (int ks = 0; ks < D / 16; ++ks) {
                uint32_t a[2][4];
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) pf_ldmatrix(a[mt], chunk(q_lane, 2 * ks) + 16 * mt * S::ROW);
#pragma unroll
                for (int c = 0; c < NT / 2; ++c) {
                    uint32_t b[4];
                    pf_ldmatrix(b, chunk(kt, 2 * ks) + 16 * c * S::ROW);
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt) {
                        pf_mma<T>(s[mt][2 * c], a[mt], b[0], b[1]);
                        pf_mma<T>(s[mt][2 * c + 1], a[mt], b[2], b[3]);
                    }
                }
            }
            if (A.negate) {
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int c = 0; c < NT; ++c)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[mt][c][i] = -s[mt][c][i];
            }
            if (key0 + PF_KT > lo) {
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int c = 0; c < NT; ++c)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (key0 + 8 * c + 2 * t + (i & 1) >= lim[mt][i >> 1]) s[mt][c][i] = -INFINITY;
            }
            // the reference so far serves unless a row's maximum grew by 2^8 or has not begun.  NaN and +inf make the row
            // NaN, as they do in the formula.
            bool grow = false;
            float top[2][2];
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    float y = -INFINITY;
#pragma unroll
                    for (int c = 0; c < NT; ++c) y = fmaxf(y, fmaxf(s[mt][c][2 * hf], s[mt][c][2 * hf + 1]));
                    top[mt][hf] = y * A.lam;
                    grow |= top[mt][hf] > m[mt][hf] + PF_LAZY;
                }
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        float y = top[mt][hf];
                        y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 1));
                        y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 2));
                        const float f = y > m[mt][hf] + PF_LAZY ? ex2(m[mt][hf] - y) : 1.f;
                        if (y > m[mt][hf] + PF_LAZY) m[mt][hf] = y;
                        l[mt][hf] *= f;
#pragma unroll
                        for (int c = 0; c < CT; ++c) {
                            o[mt][c][2 * hf] *= f;
                            o[mt][c][2 * hf + 1] *= f;
                        }
                    }
            }
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                const float ref[2] = {m[mt][0] == -INFINITY ? 0.f : m[mt][0], m[mt][1] == -INFINITY ? 0.f : m[mt][1]};
#pragma unroll
                for (int c = 0; c < NT; ++c) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[mt][c][i] = ex2(__fmaf_rn(s[mt][c][i], A.lam, -ref[i >> 1]));
                    l[mt][0] += s[mt][c][0] + s[mt][c][1];
                    l[mt][1] += s[mt][c][2] + s[mt][c][3];
                    p[mt][c >> 1][2 * (c & 1)] = pack_f32<T>(s[mt][c][0], s[mt][c][1]);
                    p[mt][c >> 1][2 * (c & 1) + 1] = pack_f32<T>(s[mt][c][2], s[mt][c][3]);
                }
            }
        }
        if (mend) __syncthreads();
        if (seen) {
#pragma unroll
            for (int ks = 0; ks < NT / 2; ++ks)
#pragma unroll
                for (int c = 0; c < CT / 2; ++c) {
                    uint32_t b[4];
                    pf_ldmatrix_trans(b, chunk(vt, 2 * c) + 16 * ks * S::ROW);
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt) {
                        pf_mma<T>(o[mt][2 * c], p[mt][ks], b[0], b[1]);
                        pf_mma<T>(o[mt][2 * c + 1], p[mt][ks], b[2], b[3]);
                    }
                }
        }
    }
    if (!used) return;                                           // no barrier of the block follows

#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            l[mt][hf] += __shfl_xor_sync(0xffffffffu, l[mt][hf], 1);
            l[mt][hf] += __shfl_xor_sync(0xffffffffu, l[mt][hf], 2);
        }
    if (x.jm < x.j0 + x.n) {                                     // the records are complete since the last step's second barrier
#pragma unroll 1
        for (int b = 0; b < 4 * PF_KT; ++b) {
            const uint32_t rows = s_bad[b >> 6][b >> 5 & 1] >> (b & 31);
            if (rows == 0) {                                     // none in the rest of the word
                b |= 31;
                continue;
            }
            b += __ffs(int(rows)) - 1;
            const int key = x.jm * PF_KT + b;
            const T* row = static_cast<const T*>(A.v) + (int64_t(x.k0) + key) * A.v_row + x.head * A.v_head + 2 * t;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int c = 0; c < CT; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float e = to_f32(row[8 * c + (i & 1)]);
                        if (key < lim[mt][i >> 1] && l[mt][i >> 1] != 0.f && !(fabsf(e) < INFINITY)) o[mt][c][i] += e;
                    }
        }
    }
    if (x.pieces > 1) {
        auto slot_of = [&](int piece) { return A.part + int64_t(piece) * ((D + 2) * PF_ROWS); };
        float* part = slot_of(x.piece);
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) __stcg(part + ((mt * CT + c) * 4 + i) * PF_THREADS + threadIdx.x, o[mt][c][i]);
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
                if (t == 0) {
                    const int row = warp * 32 + mt * 16 + hf * 8 + g;
                    __stcg(part + D * PF_ROWS + row, m[mt][hf]);
                    __stcg(part + (D + 1) * PF_ROWS + row, l[mt][hf]);
                }
        }
        __threadfence();
        __syncwarp();
        int last = 0;
        if (lane == 0) last = pf_arrive(A.count + x.first * 4 + warp, A.call, uint32_t(x.pieces));
        if (!__shfl_sync(0xffffffffu, last, 0)) return;
        __threadfence();
        // all pieces of these 32 rows are there: join them in the order of the keys
        auto row_of = [&](int mt, int hf) { return warp * 32 + mt * 16 + hf * 8 + g; };
        float ref[2][2];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                m[mt][hf] = -INFINITY;
                for (int c = x.first; c < x.first + x.pieces; ++c) m[mt][hf] = fmaxf(m[mt][hf], __ldcg(slot_of(c) + D * PF_ROWS + row_of(mt, hf)));
                ref[mt][hf] = m[mt][hf] == -INFINITY ? 0.f : m[mt][hf];
                l[mt][hf] = 0.f;
            }
#pragma unroll
            for (int c = 0; c < CT; ++c) o[mt][c][0] = o[mt][c][1] = o[mt][c][2] = o[mt][c][3] = 0.f;
        }
        for (int piece = x.first; piece < x.first + x.pieces; ++piece) {
            const float* from = slot_of(piece);
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                float f[2];
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    f[hf] = ex2(__ldcg(from + D * PF_ROWS + row_of(mt, hf)) - ref[mt][hf]);
                    l[mt][hf] = __fmaf_rn(__ldcg(from + (D + 1) * PF_ROWS + row_of(mt, hf)), f[hf], l[mt][hf]);
                }
#pragma unroll
                for (int c = 0; c < CT; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        o[mt][c][i] = __fmaf_rn(__ldcg(from + ((mt * CT + c) * 4 + i) * PF_THREADS + threadIdx.x), f[i >> 1], o[mt][c][i]);
            }
        }
    }

    // ---------------- division by l; the rows go through the warp's part of the query tile, to leave in whole sectors ----------------
    __syncwarp();
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            const float sum = l[mt][hf], inv = sum > 0.f ? 1.f / sum : (sum == sum ? 0.f : sum);
            const int row = warp * 32 + mt * 16 + hf * 8 + g;
#pragma unroll
            for (int c = 0; c < CT; ++c)
                *reinterpret_cast<uint32_t*>(pf_smem + pf_at<D>(row, c) + 4 * t) = pack_f32<T>(o[mt][c][2 * hf] * inv, o[mt][c][2 * hf + 1] * inv);
            int head;
            const int tok = token(row, head);
            if (A.lse && t == 0 && tok >= 0)
                A.lse[int64_t(x.q0 + tok) * A.Hq + head] = sum == 0.f ? -INFINITY : m[mt][hf] * 0.693147180559945309f + logf(sum);
        }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < S::CHUNKS; ++i) {
        const int e = i * 32 + lane, row = warp * 32 + e / S::CHUNKS, chunk = e % S::CHUNKS;
        int head;
        const int tok = token(row, head);
        if (tok >= 0)
            *reinterpret_cast<uint4*>(static_cast<T*>(A.out) + (int64_t(x.q0 + tok) * A.Hq + head) * D + chunk * 8) =
                *reinterpret_cast<const uint4*>(pf_smem + pf_at<D>(row, chunk));
    }
}

}  // namespace kvb
