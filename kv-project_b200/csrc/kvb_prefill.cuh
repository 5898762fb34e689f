// kvb_prefill.cuh - causal attention of packed prompts on the 5th-generation tensor cores.
//
//   S = Q K^T,  x = scaling log2(e) S,  m = running row maximum of x,  P = 2^(x - m),  l = sum P,  O = P V,
//   out = O / l,  lse = ln 2 m + ln l, over the keys j <= i + (keys - queries) that a query sees.
//
// One pass over the keys with the running maximum and sum of a softmax.  The `rep` query heads of a KV head are
// packed into the tile's rows (row = token * rep + head in the group), so a tile of 128 rows is 128 / rep tokens
// of one KV head and a short chunk still fills it.  A work item is two such tiles, A and B, of one sequence and KV
// head; both read the same key and value tiles of 128 tokens.  While the softmax of one tile runs on the CUDA cores
// (a warpgroup of its own, thread = row) the tensor cores work for the other:
//   warp 8    schedules the items and issues the TMA loads (128-byte swizzle; Q once per item, K and V through a ring)
//   warp 9    allocates tensor memory and issues the MMAs: S = Q K^T (both operands from shared memory) and
//             O += P V with P read from tensor memory and V as the MN-major operand
//   warps 0-3, 4-7   the softmax of tile A, B: S from tensor memory, P (rounded to the inputs' type: it is the
//             MMA's operand) back over it, the division by l and the stores
// Tensor memory (512 columns): S / P of A and B (128 + 128), O of A and B (d + d).  O is rescaled only when a
// row's maximum grew by more than 2^8 (P then reaches 256 at most, well inside float16's range; the sums stay in
// float32), which is seldom after the first tiles.
//
// A tile's step is a chain (logits from the tensor cores, weights, the two products), the other tile's fills its gaps, and
// what the chain costs beside the products bounds the kernel.  So P is handed over in two parts, 96 columns and 32, and the
// first part's product runs while the second is computed; and the MMA warp runs converged (16384 tokens, 32 heads over 8,
// d 128: 2102 us without either).  All roles run with the 168 registers that ten warps leave a thread, and a step with 128
// logits, their weights and sums wants more: the last 32 logits are read twice, first for the maximum only (1915 us, 8
// packed prompts of 7208 tokens 139; 2068 and 162 with spills; weights computed ahead of the maximum, which has to be redone
// where it grew, 1983 and 150).  Registers moved between the roles (setmaxnreg, 224 and 56) took 1876 and 135, but one of
// some 45000 calls ended in an illegal access, none of 150000 without.
//
// Replayed graphs of ten calls on many items have ended in an illegal access too, with and without those registers and
// programmatic launches, seldom and never in the first replay; a kernel that checked its own addresses ended the same way,
// and reading shows every access in bounds and every copy, product and arrival waited for.  Until the cause is known the
// call refuses a stream that is being captured.
//
// Measured and left (some with those registers): two threads a row (1971), steps of 64 keys with two score buffers (1894), an
// MMA warp per tile (1929), an eighth to a half of the exponentials as polynomials (1838 to 1906), growth seen from the sum
// of the weights instead of the maximum (no difference).
//
// Masks: logits of keys past a row's limit become -inf by selection, so what lies there does not matter; values
// there would still meet a weight of zero in the MMA (0 * NaN), so in tiles that some row of the item does not see
// whole, value rows past the sequence become zeros in shared memory, and non-finite entries of the sequence's own
// later tokens too, which the rows that do see them get added back at the end.
//
// Work items are dealt in descending order of their key tiles, forth and back over the CTAs; items of more tiles than a
// CTA's fair share (few rows over long keys) come first, cut into equal pieces of at most that many: each piece leaves
// its O, m and l in the workspace, and the warp that completes the last piece of its 32 rows joins them in the order of
// the keys.  Every CTA finds its next item from the lengths (bisection on the tile count, sums of tile counts in closed
// form, a warp's lanes over the sequences), so no plan is built before the launch and no counter is kept.  Two chunks after
// prefixes (500 after 7000 and 1100 after 333, 16 heads over 4, d 64): 134 us without pieces.  Equal shares of
// consecutive work, cut anywhere, balance as well but cut almost every share's ends: packed prompts 167 to 189
// instead of 150 us.
//
// Every wait is bounded; after a timeout all roles stop, copies in flight are waited for and tensor memory is freed.
#pragma once
#include <cuda.h>

#include <climits>
#include <type_traits>

#include "kvb_common.cuh"
#include "kvb_pages_view.cuh"
#include "kvb_spectral.cuh"

namespace kvb {

constexpr int PF_KT = 128;                    // keys per tile
constexpr int PF_THREADS = 320;
constexpr int PF_TMEM_COLS = 512;
constexpr float PF_LAZY = 8.f;                // log2 of how far a maximum may grow before O is rescaled

struct PrefillParams {
    CUtensorMap tm_q;                         // (d, Hq, nq), box 64 x rep x (128 / rep)
    CUtensorMap tm_k, tm_v;                   // (d, Hkv, nk), box 64 x 1 x 128
    const void* v;                            // values again, for the non-finite entries that are added back
    int64_t v_row, v_head;
    const int32_t* cu_q;
    const int32_t* cu_k;
    int64_t nq, nk;
    int n, Hq, Hkv, rep, tt;                  // tt = 128 / rep tokens per tile
    float* part;                              // [2 grid pieces][2 tiles][d + 2][128]: O by column, m, l; null: no item is cut
    uint32_t* count;                          // [2 grid pieces][8 warps]
    float lam;                                // |scaling| log2(e), > 0
    int negate;                               // scaling < 0
    void* out;                                // (nq, Hq, d)
    float* lse;                               // (nq, Hq) or null
};

template <int D>
struct PfShape {
    static constexpr int HALVES = D / 64;
    static constexpr int TILE_BYTES = 128 * D * 2;
    static constexpr int STAGES = D == 128 ? 5 : 8;
    static constexpr int Q_BYTES = 2 * TILE_BYTES;
    static constexpr int SMEM = 1024 + Q_BYTES + STAGES * TILE_BYTES + 1024;
};

struct PfItem {
    int q0, ql, k0, kl;                       // the sequence's rows
    int t0;                                   // first token of tile A within it
    int head;                                 // KV head; < 0: no more work
    int j0;                                   // first key tile of this piece
    int n[2];                                 // key tiles of A and B in this piece
    int piece, first, pieces;                 // number of this piece and of the item's first; how many the item has
    int jm;                                   // first key tile that some row does not see whole
    uint32_t bad[4][4];                       // non-finite value rows of the tiles jm ..
};

struct PfShared {
    uint64_t q_full, q_empty;
    uint64_t kv_full[8], kv_empty[8];
    uint64_t s_full[2], p_most[2], p_full[2], o_full[2];        // p_most: the first 96 columns of P
    uint64_t item_full[2], item_empty[2];
    uint32_t tmem;
    int abort;
    uint32_t kv_issued, q_issued;
    PfItem item[2];
};
static_assert(sizeof(PfShared) <= 1024, "the barrier block");

// K-major and MN-major (128-byte swizzle) shared-memory matrix descriptors: 8-row (8-k) groups 1024 B apart; for the
// MN-major one `lead` bytes from one 64-element block of the contiguous dimension to the next.
__device__ __forceinline__ uint64_t pf_desc_mn(uint32_t saddr, uint32_t lead) {
    return uint64_t((saddr >> 4) & 0x3FFF) | (uint64_t(lead >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
           (uint64_t(2) << 61);
}

__host__ __device__ constexpr uint32_t pf_idesc(int N, int bf16, int b_mn) {
    return (1u << 4) | (uint32_t(bf16) << 7) | (uint32_t(bf16) << 10) | (uint32_t(b_mn) << 16) | (uint32_t(N >> 3) << 17) |
           (uint32_t(128 >> 4) << 24);
}

// The MMA warp runs converged, so that descriptors stay in uniform registers (issued from a divergent branch of one lane an
// MMA took 91 cycles, 64 is its time on the tensor core); `lead` is set in the one lane that issues.
__device__ __forceinline__ uint32_t pf_elect() {
    uint32_t lead;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(lead));
    return lead;
}
// D[tmem] (+)= A[smem] B[smem]
__device__ __forceinline__ void pf_mma_ss(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, int acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead)
        : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]
__device__ __forceinline__ void pf_mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, int acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void pf_commit(uint32_t lead, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
        "r"(lead)
        : "memory");
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

#define PF_R8(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7])
#define PF_W8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])

// 32 columns of this thread's tensor-memory lane: valid after pf_wait_ld()
__device__ __forceinline__ void pf_ld32(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : PF_R8(r, 0), PF_R8(r, 8), PF_R8(r, 16), PF_R8(r, 24)
        : "r"(addr));
}
__device__ __forceinline__ void pf_st32(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::PF_W8(r, 0),
        PF_W8(r, 8), PF_W8(r, 16), PF_W8(r, 24), "r"(addr)
        : "memory");
}
__device__ __forceinline__ void pf_st16(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::PF_W8(r, 0),
        PF_W8(r, 8), "r"(addr)
        : "memory");
}
__device__ __forceinline__ void pf_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pf_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <typename T>
__device__ __forceinline__ uint32_t pf_pack(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pf_pack<__half>(float lo, float hi) { return pack_half2(lo, hi); }
template <>
__device__ __forceinline__ uint32_t pf_pack<__nv_bfloat16>(float lo, float hi) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
}

// Two float32 operations in one instruction.
__device__ __forceinline__ uint64_t pf_two(float a, float b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float2 pf_split(uint64_t a) {
    float2 d;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(a));
    return d;
}
__device__ __forceinline__ uint64_t pf_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t pf_add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float pf_max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// P of 32 columns: 2^(v lam - ref), packed, and their sums added.
template <typename T>
__device__ __forceinline__ void pf_weights(const uint32_t* v, uint64_t lam, uint64_t nref, uint32_t* p, uint64_t (&sum)[2]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float2 y = pf_split(pf_fma2(pf_two(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), lam, nref));
        const float a = ex2(y.x), b = ex2(y.y);
        sum[i & 1] = pf_add2(sum[i & 1], pf_two(a, b));
        p[i] = pf_pack<T>(a, b);
    }
}

// Whether one of the two packed values is not finite: x * 0 is NaN for NaN and infinities only.
template <typename T>
__device__ __forceinline__ bool pf_not_finite(const uint4& w) {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const uint32_t zero = 0;
    const T2 z = *reinterpret_cast<const T2*>(&zero);
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
    T2 s = z;
#pragma unroll
    for (int i = 0; i < 4; ++i) s = __hfma2(*reinterpret_cast<const T2*>(&a[i]), z, s);
    return __hisnan(s.x) || __hisnan(s.y);
}

// ---------------------------------------------------------------------------------------------
// Work items: those of more tiles than the fair share, in pieces, then the others in descending order of key tiles.
// ---------------------------------------------------------------------------------------------
struct PfSeq {
    int q0, ql, k0, kl, pairs;
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
        q.pairs = (q.ql + 2 * A.tt - 1) / (2 * A.tt);
    }
    return q;
}

// How many of a sequence's tile pairs have t key tiles or more: pair p ends at the query min(2 tt (p + 1), ql), which
// sees kl - ql + that many keys.
__device__ __forceinline__ int pf_count(const PfSeq& q, int t, int tt) {
    if (t <= 0) return q.pairs;
    const int need = PF_KT * (t - 1) + 1;
    if (q.kl < need) return 0;
    const int first = max(need - q.kl + q.ql + 2 * tt - 1, 0) / (2 * tt) - 1;      // ceil(..) - 1
    return q.pairs - min(max(first, 0), q.pairs - 1);
}

__device__ __forceinline__ int pf_warp_sum(int v) { return __reduce_add_sync(0xffffffffu, v); }

// sum over i < n of floor((a i + b) / m), for a, b >= 0 (the Euclidean reduction of a and the divisor).  Intermediate
// values stay below 2^32: n is a count of tile pairs, whose rows have to fit the GPU's memory.
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

// Pieces of up to `keys` keys (a multiple of the tile) in the pairs before p, a pair counting one at least unless it sees
// no key.
__device__ __forceinline__ int pf_pieces(const PfSeq& q, int p, int tt, uint32_t keys) {
    const int full = min(p, q.pairs - 1), a = q.kl - q.ql, b = 2 * tt;         // pairs that end before the sequence does
    const int i0 = a < 0 ? min(-a / b, full) : 0;                              // those before see no key
    int c = full > i0 ? int(pf_floor_sum(full - i0, keys, b, uint32_t(a + b * (i0 + 1)) + keys - 1)) : 0;
    if (p == q.pairs && p > 0) c += int((uint32_t(q.kl) + keys - 1) / keys);
    return c;
}

// The tiles j0 .. j1 - 1 of a pair (out: its sequence and head).
__device__ __forceinline__ void pf_tiles_of(const PrefillParams& A, int pair, int j0, int j1, PfItem& out) {
    out.t0 = pair * 2 * A.tt;
    out.j0 = j0;
    for (int w = 0; w < 2; ++w) {
        const int last = min(out.t0 + (w + 1) * A.tt, out.ql);              // tokens before it
        const int keys = last > out.t0 + w * A.tt ? min(max(out.kl - out.ql + last, 0), out.kl) : 0;
        out.n[w] = max(min((keys + PF_KT - 1) / PF_KT, j1) - j0, 0);
    }
    out.jm = max(out.kl - out.ql + out.t0 + 1, 0) / PF_KT;
}

constexpr int PF_SHARE = 8;                   // items of fewer tiles are never cut

struct PfCuts {
    int share;                                // items of more tiles are cut into pieces of at most so many
    int items;                                // how many are,
    int pieces;                               // into how many pieces
};

// The fair share (not below eight tiles), and what it cuts; whole warp.  The share is that of a bound on the number of
// tiles, at most half a tile an item too high; so there are at most 2 ctas pieces, each having half a share or more.
// Item and piece counts fit 32 bits by far: 256 query rows an item.
__device__ __forceinline__ PfCuts pf_cuts(const PrefillParams& A, int ctas) {
    const int lane = threadIdx.x & 31;
    PfCuts c{INT_MAX, 0, 0};
    if (!A.part) return c;
    float tiles = 0.f;
    int most = 0;
    for (int s0 = 0; s0 < A.n; s0 += 32) {
        const PfSeq q = pf_seq(A, s0 + lane);
        if (q.pairs == 0) continue;
        // the pairs from the first that sees a key on end at a + b (i + 1) keys or before
        const int a = q.kl - q.ql, b = 2 * A.tt, i0 = a < 0 ? min(-a / b, q.pairs) : 0;
        const float k = float(q.pairs - i0);
        tiles += k * (float(a) + float(b) * (float(i0) + 0.5f * (k + 1.f))) * (1.f / PF_KT) + k;
        most = max(most, (q.kl + PF_KT - 1) / PF_KT);
    }
    tiles = warp_sum(tiles) * float(A.Hkv);
    most = __reduce_max_sync(0xffffffffu, most);
    const float share = fmaxf(float(PF_SHARE), tiles * 1.0001f / float(ctas) + 1.f);
    if (float(most) <= share) return c;
    c.share = int(share);
    for (int s0 = 0; s0 < A.n; s0 += 32) {
        const PfSeq q = pf_seq(A, s0 + lane);
        const int cut = q.pairs ? pf_count(q, c.share + 1, A.tt) : 0;
        const uint32_t keys = uint32_t(c.share) * PF_KT;
        c.items += cut * A.Hkv;
        if (cut) c.pieces += (pf_pieces(q, q.pairs, A.tt, keys) - pf_pieces(q, q.pairs - cut, A.tt, keys)) * A.Hkv;
    }
    c.items = __reduce_add_sync(0xffffffffu, c.items);
    c.pieces = __reduce_add_sync(0xffffffffu, c.pieces);
    return c;
}

// Piece `idx` of the cut items; whole warp.
__device__ __forceinline__ void pf_piece(const PrefillParams& A, const PfCuts& cuts, int idx, PfItem& out) {
    const int lane = threadIdx.x & 31;
    const uint32_t keys = uint32_t(cuts.share) * PF_KT;
    int r = idx;
    for (int s0 = 0; s0 < A.n; s0 += 32) {
        const PfSeq q = pf_seq(A, s0 + lane);
        const int cut = q.pairs ? pf_count(q, cuts.share + 1, A.tt) : 0;
        const int before = cut ? pf_pieces(q, q.pairs - cut, A.tt, keys) : 0;
        const int per = cut ? pf_pieces(q, q.pairs, A.tt, keys) - before : 0;                  // pieces of one head
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
        c.pairs = __shfl_sync(0xffffffffu, q.pairs, src);
        r -= __shfl_sync(0xffffffffu, x - per * A.Hkv, src);
        const int one = __shfl_sync(0xffffffffu, per, src), skipped = __shfl_sync(0xffffffffu, before, src);
        const int head = r / one;
        r -= head * one;
        // the largest pair whose pieces begin at or before r, by 32-way search
        int lo = c.pairs - __shfl_sync(0xffffffffu, cut, src), len = c.pairs - lo, at = 0;
        while (true) {
            const int step = (len + 31) / 32, p = lo + lane * step;
            const int v = p < lo + len ? pf_pieces(c, p, A.tt, keys) - skipped : 0;
            const int k = 31 - __clz(int(__ballot_sync(0xffffffffu, p < lo + len && v <= r) | 1u));
            at = __shfl_sync(0xffffffffu, v, k);
            lo += k * step;
            len = min(step, c.pairs - lo);
            if (step == 1) break;
        }
        out.q0 = c.q0, out.ql = c.ql, out.k0 = c.k0, out.kl = c.kl;
        out.head = head;
        const int e = c.kl - c.ql + min(2 * A.tt * (lo + 1), c.ql), tiles = (e + PF_KT - 1) / PF_KT, k = r - at;
        out.pieces = (tiles + cuts.share - 1) / cuts.share;
        out.piece = idx;
        out.first = idx - k;
        pf_tiles_of(A, lo, int(int64_t(tiles) * k / out.pieces), int(int64_t(tiles) * (k + 1) / out.pieces), out);
        return;
    }
}

// Item `idx`; `t` the last item's key tiles (a bound for the search), or < 0 at first.  Whole warp; false when there
// are no more.
__device__ __forceinline__ bool pf_item(const PrefillParams& A, const PfCuts& cuts, int idx, int& t, PfItem& out) {
    const int lane = threadIdx.x & 31;
    if (idx < cuts.pieces) {
        pf_piece(A, cuts, idx, out);
        return true;
    }
    idx += cuts.items - cuts.pieces;              // place among all items by their tiles
    const PfSeq mine = pf_seq(A, lane);
    auto total = [&](int tiles) {                 // items of `tiles` key tiles or more
        int c = mine.pairs ? pf_count(mine, tiles, A.tt) : 0;
        for (int s0 = 32; s0 < A.n; s0 += 32) {
            const PfSeq q = pf_seq(A, s0 + lane);
            if (q.pairs) c += pf_count(q, tiles, A.tt);
        }
        return pf_warp_sum(c) * A.Hkv;
    };
    int hi = t;
    if (t < 0) {
        int most = (mine.kl + PF_KT - 1) / PF_KT;
        for (int s0 = 32; s0 < A.n; s0 += 32) most = max(most, (pf_seq(A, s0 + lane).kl + PF_KT - 1) / PF_KT);
        hi = min(__reduce_max_sync(0xffffffffu, most), cuts.share);
        if (idx >= total(0)) return false;
    }
    int lo = 0, above = 0;                        // the largest t with total(t) > idx, and total(t + 1)
    if (const int c = total(hi); c > idx) {
        lo = hi;
        above = total(hi + 1);
    } else {
        above = c;
        --hi;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2, m = total(mid);
            if (m > idx) lo = mid;
            else {
                hi = mid - 1;
                above = m;
            }
        }
        if (lo == 0 && total(0) <= idx) return false;
    }
    t = lo;
    int r = idx - above;                          // rank among the items of t tiles
    for (int s0 = 0; s0 < A.n; s0 += 32) {
        const PfSeq q = s0 == 0 ? mine : pf_seq(A, s0 + lane);
        const int before = q.pairs ? pf_count(q, t + 1, A.tt) : 0, c = (q.pairs ? pf_count(q, t, A.tt) : 0) - before;
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
        pf_tiles_of(A, __shfl_sync(0xffffffffu, q.pairs - before - c, src) + step, 0, INT_MAX, out);
        return true;
    }
    return false;
}

template <typename T, int D>
__global__ void __launch_bounds__(PF_THREADS, 1) prefill_kernel(const __grid_constant__ PrefillParams A) {
    using S = PfShape<D>;
    constexpr int BF16 = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    extern __shared__ uint8_t pf_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pf_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sq = base;                                          // [tile][half][128 rows][64 ch]
    uint8_t* skv = base + S::Q_BYTES;                            // [stage][half][128 tokens][64 ch]: K, V, K, V, ...
    PfShared& sh = *reinterpret_cast<PfShared*>(skv + S::STAGES * S::TILE_BYTES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        mbar_init(&sh.q_full, 1);
        mbar_init(&sh.q_empty, 1);
        for (int i = 0; i < S::STAGES; ++i) {
            mbar_init(&sh.kv_full[i], 1);
            mbar_init(&sh.kv_empty[i], 1);
        }
        for (int w = 0; w < 2; ++w) {
            mbar_init(&sh.s_full[w], 1);
            mbar_init(&sh.p_most[w], 4);
            mbar_init(&sh.p_full[w], 4);
            mbar_init(&sh.o_full[w], 1);
            mbar_init(&sh.item_full[w], 1);
            mbar_init(&sh.item_empty[w], 9);
        }
        sh.abort = 0;
        sh.kv_issued = sh.q_issued = 0;
        fence_mbar_init();
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                     "r"(PF_TMEM_COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    volatile int* abort = &sh.abort;
    // a wait that gave up stops every role
    auto wait = [&](uint64_t* bar, uint32_t count) {
        if (mbar_try_wait(bar, count & 1)) return true;
        if (*abort) return false;
        if (mbar_wait(bar, count & 1)) return true;
        *abort = 1;
        return false;
    };

    if (warp == 8) {
        // ---------------- schedule and loads ----------------
        uint32_t it = 0, items = 0;
        int t = -1;
        bool ok = true;
        const PfCuts cuts = pf_cuts(A, gridDim.x);
        for (int64_t round = 0; ok; ++round) {
            const int idx = int(round * gridDim.x + (round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x));
            PfItem x;
            const bool more = pf_item(A, cuts, idx, t, x);
            PfItem& slot = sh.item[round & 1];
            if (round >= 2) ok = __all_sync(0xffffffffu, wait(&sh.item_empty[round & 1], uint32_t(round / 2 - 1)));
            if (!ok) break;
            if (lane == 0) {
                slot = x;
                if (!more) slot.head = -1;
                for (int i = 0; i < 16; ++i) slot.bad[i / 4][i % 4] = 0;
                mbar_arrive(&sh.item_full[round & 1]);
            }
            if (!more) break;
            const int nt = max(x.n[0], x.n[1]);
            if (lane == 0 && nt > 0) {
                ok = items == 0 || wait(&sh.q_empty, items - 1);
                if (ok) {
                    const uint32_t bytes = uint32_t(A.tt * A.rep) * D * 2;
                    mbar_arrive_expect_tx(&sh.q_full, 2 * bytes);
                    for (int w = 0; w < 2; ++w)
                        for (int h = 0; h < S::HALVES; ++h)
                            tma_load_3d(sq + w * S::TILE_BYTES + h * (128 * 128), &A.tm_q, h * 64, x.head * A.rep,
                                        x.q0 + x.t0 + w * A.tt, &sh.q_full);
                    sh.q_issued = ++items;
                }
                for (int j = 0; ok && j < 2 * nt; ++j, ++it) {
                    const int st = it % S::STAGES;
                    if (it >= S::STAGES && !wait(&sh.kv_empty[st], it / S::STAGES - 1)) { ok = false; break; }
                    mbar_arrive_expect_tx(&sh.kv_full[st], S::TILE_BYTES);
                    for (int h = 0; h < S::HALVES; ++h)
                        tma_load_3d(skv + st * S::TILE_BYTES + h * (128 * 128), j & 1 ? &A.tm_v : &A.tm_k, h * 64, x.head,
                                    x.k0 + (x.j0 + (j >> 1)) * PF_KT, &sh.kv_full[st]);
                    sh.kv_issued = it + 1;
                }
            }
            ok = __shfl_sync(0xffffffffu, int(ok), 0);
        }
        // the MMAs' last arrivals are in before the CTA may leave
        for (uint32_t k = it > uint32_t(S::STAGES) ? it - S::STAGES : 0; ok && lane == 0 && k < it; ++k)
            ok = wait(&sh.kv_empty[k % S::STAGES], k / S::STAGES);
        if (ok && lane == 0 && items > 0) wait(&sh.q_empty, items - 1);
    } else if (warp == 9) {
        // ---------------- MMA issue ----------------
        constexpr uint32_t IDESC_S = pf_idesc(PF_KT, BF16, 0), IDESC_O = pf_idesc(D, BF16, 1);
        const uint32_t lead = pf_elect(), tm = __shfl_sync(0xffffffffu, tmem, 0);
        const uint64_t q_desc = umma_desc_sw128(smem_u32(sq)), k_desc = umma_desc_sw128(smem_u32(skv)),
                       v_desc = pf_desc_mn(smem_u32(skv), 128 * 128);
        auto all = [&](bool b) { return __all_sync(0xffffffffu, b) != 0; };
        uint32_t items = 0, pv[2] = {0, 0};
        uint32_t st = 0, ph = 0;                                 // stage and phase of the next load to be used
        auto next = [&]() {
            if (++st == S::STAGES) { st = 0; ph ^= 1; }
        };
        // descriptor addresses count 16 bytes
        auto scores = [&](int w, uint32_t kst) {                 // S_w = Q_w K^T
            const uint64_t a = q_desc + uint32_t(w * (S::TILE_BYTES >> 4)), b = k_desc + kst * uint32_t(S::TILE_BYTES >> 4);
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                const uint32_t off = ((k >> 2) * (128 * 128) + (k & 3) * 32) >> 4;
                pf_mma_ss(lead, tm + uint32_t(w * PF_KT), a + off, b + off, IDESC_S, k != 0);
            }
            pf_commit(lead, &sh.s_full[w]);
        };
        bool ok = true;
        for (int64_t round = 0; ok; ++round) {
            if (!all(wait(&sh.item_full[round & 1], uint32_t(round / 2)))) break;
            const PfItem& x = sh.item[round & 1];
            const int n0 = __shfl_sync(0xffffffffu, x.n[0], 0), n1 = __shfl_sync(0xffffffffu, x.n[1], 0);
            const int head = __shfl_sync(0xffffffffu, x.head, 0);
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.item_empty[round & 1]);
            if (head < 0) break;
            const int nt = max(n0, n1);
            if (nt == 0) continue;
            ok = all(wait(&sh.q_full, items) && wait(&sh.kv_full[st], ph));
            ++items;
            if (!ok) break;
            tc_fence_after();
            for (int w = 0; w < 2; ++w)
                if ((w ? n1 : n0) > 0) scores(w, st);
            pf_commit(lead, &sh.kv_empty[st]);
            if (nt == 1) pf_commit(lead, &sh.q_empty);
            next();
            for (int j = 0; ok && j < nt; ++j) {
                const uint32_t vst = st;                         // V(j), then K(j + 1)
                const uint32_t vph = ph;
                next();
                const uint32_t kst = st;
                const bool more = j + 1 < nt;
                ok = all(lane & 1 && more ? wait(&sh.kv_full[kst], ph) : wait(&sh.kv_full[vst], vph));
                if (more) next();
                for (int w = 0; ok && w < 2; ++w) {
                    const int n = w ? n1 : n0;
                    if (j >= n) continue;
                    const uint64_t v = v_desc + vst * uint32_t(S::TILE_BYTES >> 4);
                    auto values = [&](int k) {                   // O_w += P_w V, 16 tokens
                        pf_mma_ts(lead, tm + 256 + uint32_t(w * D), tm + uint32_t(w * PF_KT + k * 8), v + uint32_t(k * (2048 >> 4)), IDESC_O,
                                  j != 0 || k != 0);
                    };
                    ok = all(wait(&sh.p_most[w], pv[w]));
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int k = 0; k < 6; ++k) values(k);
                    ok = all(wait(&sh.p_full[w], pv[w]++));
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int k = 6; k < PF_KT / 16; ++k) values(k);
                    pf_commit(lead, &sh.o_full[w]);
                    if (j + 1 < n) scores(w, kst);
                }
                if (!ok) break;
                pf_commit(lead, &sh.kv_empty[vst]);
                if (more) pf_commit(lead, &sh.kv_empty[kst]);
                if (j + 2 == nt) pf_commit(lead, &sh.q_empty);   // the last scores are issued
            }
        }
        // after a timeout the MMAs already issued finish before tensor memory is released
        if (*abort)
            for (int w = 0; w < 2; ++w)
                if (pv[w] > 0) mbar_wait(&sh.o_full[w], (pv[w] - 1) & 1, 10000000ull);
    } else {
        // ---------------- softmax: warpgroup w, thread = row ----------------
        const int w = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = tmem + (uint32_t((warp & 3) * 32) << 16);
        const uint32_t s_col = lanes + uint32_t(w * PF_KT), o_col = lanes + 256 + uint32_t(w * D);
        uint32_t steps = 0, kv = 0;                              // this tile's MMA rounds; loads of the items so far
        auto all = [&](bool b) { return __all_sync(0xffffffffu, b) != 0; };
        for (int64_t round = 0;; ++round) {
            if (!all(wait(&sh.item_full[round & 1], uint32_t(round / 2)))) break;
            PfItem& x = sh.item[round & 1];
            const int head = x.head;
            if (head < 0) break;
            const int n = x.n[w], nt = max(x.n[0], x.n[1]), kl = x.kl;
            const int j0 = x.j0, jm = x.jm - j0;                 // key tiles are counted from the piece's first
            const int tok = x.t0 + w * A.tt + row / A.rep;       // token of the sequence
            const bool valid = row < A.tt * A.rep && tok < x.ql;
            const int limit = valid ? min(max(kl - x.ql + tok + 1, 0), kl) : INT_MAX;    // rows of no token mask nothing
            const int jmask = __reduce_min_sync(0xffffffffu, limit) / PF_KT - j0;        // first tile that a row of the warp does not see whole
            float m = -INFINITY, l = 0.f;
            bool ok = true;
            for (int j = 0; j < n; ++j, ++steps) {
                if (!(ok = all(wait(&sh.s_full[w], steps)))) break;
                tc_fence_after();
                // The logits take 96 registers: of the last 32 only the maximum is kept, they are read again below.
                uint32_t r[PF_KT - 32], p[32];
                float* v = reinterpret_cast<float*>(r);
                const int lim = limit - (j0 + j) * PF_KT;
                const bool masked = j >= jmask;
                auto logits = [&](uint32_t* x, int c0, int n) {  // the sign of the scaling, and the mask
                    if (A.negate) {
#pragma unroll
                        for (int i = 0; i < n; ++i) x[i] ^= 0x80000000u;
                    }
                    if (masked) {
#pragma unroll
                        for (int i = 0; i < n; ++i) x[i] = c0 + i < lim ? x[i] : 0xff800000u;
                    }
                };
                pf_ld32(s_col + PF_KT - 32, p);
#pragma unroll
                for (int c = 0; c < PF_KT - 32; c += 32) pf_ld32(s_col + c, r + c);
                pf_wait_ld();
                logits(p, PF_KT - 32, 32);
                float last[2] = {__uint_as_float(p[0]), __uint_as_float(p[1])};
#pragma unroll
                for (int i = 2; i < 32; i += 2) last[i / 2 & 1] = pf_max3_nan(last[i / 2 & 1], __uint_as_float(p[i]), __uint_as_float(p[i + 1]));
                logits(r, 0, PF_KT - 32);
                uint64_t sum[2] = {0, 0};
                auto weights = [&](const uint32_t* x, uint32_t* to) {                // of 32 logits
                    const float ref = m == -INFINITY ? 0.f : m;
                    pf_weights<T>(x, pf_two(A.lam, A.lam), pf_two(-ref, -ref), to, sum);
                };
                auto maximum = [&]() {
                    float mx[4] = {last[0], last[1], v[0], v[1]};
#pragma unroll
                    for (int i = 2; i < PF_KT - 34; i += 8)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (i + 4 + k < PF_KT - 32) mx[k] = pf_max3_nan(mx[k], v[i + k], v[i + 4 + k]);
                            else if (i + k < PF_KT - 32) mx[k] = pf_max3_nan(mx[k], v[i + k], v[i + k]);
                    return pf_max3_nan(pf_max3_nan(mx[0], mx[1], mx[2]), mx[3], mx[3]) * A.lam;
                };
                // the reference so far serves unless a row's maximum grew by 2^8, has not begun, or is not finite
                const float top = maximum();
                if (__any_sync(0xffffffffu, valid && !(top <= m + PF_LAZY && m > -INFINITY))) {
                    // a row that has seen nothing takes its first maximum as it is; O is zero until then.  NaN and +inf
                    // make the row NaN, as they do in the formula.
                    const bool odd = !(top < INFINITY), grow = valid && (top > m + PF_LAZY || odd) && m > -INFINITY;
                    const float to = odd ? NAN : top;
                    if (m == -INFINITY) m = to;
                    if (__any_sync(0xffffffffu, grow)) {
                        // O holds the sums of the tiles before: wait for them, and scale the rows that grew
                        const float f = grow ? ex2(m - to) : 1.f;
                        m = grow ? to : m;
                        l *= f;
                        if (j > 0) {
                            if (!(ok = all(wait(&sh.o_full[w], steps - 1)))) break;
                            tc_fence_after();
#pragma unroll 1
                            for (int c = 0; c < D; c += 32) {
                                pf_ld32(o_col + c, p);
                                pf_wait_ld();
#pragma unroll
                                for (int i = 0; i < 32; ++i) p[i] = __float_as_uint(__uint_as_float(p[i]) * f);
                                pf_st32(o_col + c, p);
                            }
                        }
                    }
                }
                weights(r, p);
                weights(r + 32, p + 16);
                pf_st32(s_col, p);
                if (j >= jm) {
                    // value rows that some row of the item does not see: see the head of this file
                    const uint32_t vj = kv + 2 * j + 1;
                    if (!(ok = all(wait(&sh.kv_full[vj % S::STAGES], vj / S::STAGES)))) break;
                    uint8_t* vt = skv + (vj % S::STAGES) * S::TILE_BYTES + row * 128;
                    const bool past = (j0 + j) * PF_KT + row >= kl;
                    bool bad = false;
                    if (!past) {
#pragma unroll
                        for (int c = 0; c < D / 8; ++c)
                            bad |= pf_not_finite<T>(*reinterpret_cast<const uint4*>(vt + (c >> 3) * (128 * 128) + ((c & 7) ^ (row & 7)) * 16));
                    }
                    const uint32_t mask = __ballot_sync(0xffffffffu, bad);
                    if (mask && lane == 0) atomicOr(&x.bad[j - jm][warp & 3], mask);
                    __threadfence_block();
                    if (past) {
#pragma unroll
                        for (int c = 0; c < D / 8; ++c) *reinterpret_cast<uint4*>(vt + (c >> 3) * (128 * 128) + c % 8 * 16) = uint4{0, 0, 0, 0};
                    } else if (bad) {
                        for (int c = 0; c < D; ++c) {
                            T* e = reinterpret_cast<T*>(vt + (c >> 6) * (128 * 128) + (((c >> 3) & 7) ^ (row & 7)) * 16) + (c & 7);
                            if (!(fabsf(to_f32(*e)) < INFINITY)) *e = from_f32<T>(0.f);
                        }
                    }
                    fence_proxy_async_smem();
                }
                weights(r + 64, p);
                pf_st16(s_col + 32, p);
                pf_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_most[w]);
                pf_ld32(s_col + PF_KT - 32, r);
                pf_wait_ld();
                logits(r, PF_KT - 32, 32);
                weights(r, p + 16);
                pf_st16(s_col + 48, p + 16);
                const float2 s0 = pf_split(sum[0]), s1 = pf_split(sum[1]);
                l += (s0.x + s0.y) + (s1.x + s1.y);
                pf_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_full[w]);
            }
            if (!ok) break;
            if (n > 0) {
                if (!all(wait(&sh.o_full[w], steps - 1))) break;
                tc_fence_after();
            }
            // records of non-finite values, complete: the last MMA waited for all four warps' P, made after them
            bool any_bad = false;
            if (jm < nt)
                for (int i = 0; i < 16; ++i) any_bad |= reinterpret_cast<volatile uint32_t*>(x.bad)[i] != 0;
            const int64_t out_row = int64_t(x.q0) + tok;
            const int hq = head * A.rep + row % A.rep;
            T* dst = static_cast<T*>(A.out) + (out_row * A.Hq + hq) * D;
            auto store = [&](const uint32_t (&o)[32], int c, float sum) {
                const float inv = sum > 0.f ? 1.f / sum : (sum == sum ? 0.f : sum);
                if (!valid) return;
#pragma unroll
                for (int i = 0; i < 2; ++i) {                    // whole 32-byte sectors: a lane has a row of its own
                    uint32_t h[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        h[k] = pf_pack<T>(__uint_as_float(o[16 * i + 2 * k]) * inv, __uint_as_float(o[16 * i + 2 * k + 1]) * inv);
                    asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::PF_W8(h, 0), "l"(dst + c + 16 * i) : "memory");
                }
            };
            auto store_lse = [&](float top, float sum) {
                if (valid && A.lse)
                    A.lse[out_row * A.Hq + hq] = sum == 0.f ? -INFINITY : top * 0.693147180559945309f + logf(sum);
            };
            const bool whole = x.pieces == 1, used = __any_sync(0xffffffffu, valid);
            auto slot_of = [&](int piece) {                      // this tile's part: O by column, then m and l
                return A.part + (int64_t(piece) * 2 + w) * ((D + 2) * 128) + row;
            };
            float* part = whole ? nullptr : slot_of(x.piece);
#pragma unroll 1
            for (int c = 0; c < (used ? D : 0); c += 32) {
                uint32_t o[32];
                __syncwarp();                                    // after the stores of some lanes
                if (n > 0) {
                    pf_ld32(o_col + c, o);
                    pf_wait_ld();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0;
                }
                if (any_bad && valid && l != 0.f) {
                    const T* vp = static_cast<const T*>(A.v) + int64_t(x.k0) * A.v_row + head * A.v_head + c;
                    for (int b = 0; b < 4 * PF_KT; ++b) {
                        const int key = (j0 + jm) * PF_KT + b;
                        if (key < limit && (x.bad[b >> 7][(b >> 5) & 3] >> (b & 31) & 1)) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                const float e = to_f32(vp[key * A.v_row + i]);
                                if (!(fabsf(e) < INFINITY)) o[i] = __float_as_uint(__uint_as_float(o[i]) + e);
                            }
                        }
                    }
                }
                if (whole) {
                    store(o, c, l);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) __stcg(part + (c + i) * 128, __uint_as_float(o[i]));
                }
            }
            if (whole) {
                store_lse(m, l);
            } else if (used) {
                __stcg(part + D * 128, m);
                __stcg(part + (D + 1) * 128, l);
                __threadfence();
                __syncwarp();
                uint32_t* count = A.count + x.first * 8 + warp;
                uint32_t before = 0;
                if (lane == 0) before = atomicAdd(count, 1u);
                before = __shfl_sync(0xffffffffu, before, 0);
                if (before + 1 > uint32_t(x.pieces)) {
                    if (lane == 0) raise_status(KVB_DEV_WORKSPACE);
                } else if (before + 1 == uint32_t(x.pieces)) {
                    // all pieces of these 32 rows are there: join them in the order of the keys
                    if (lane == 0) *count = 0;
                    __threadfence();
                    float top = -INFINITY;
                    for (int c = x.first; c < x.first + x.pieces; ++c) top = fmaxf(top, __ldcg(slot_of(c) + D * 128));
                    const float ref = top == -INFINITY ? 0.f : top;
                    float sum = 0.f;
                    for (int c = x.first; c < x.first + x.pieces; ++c)
                        sum = __fmaf_rn(__ldcg(slot_of(c) + (D + 1) * 128), ex2(__ldcg(slot_of(c) + D * 128) - ref), sum);
#pragma unroll 1
                    for (int ch = 0; ch < D; ch += 32) {
                        float acc[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) acc[i] = 0.f;
                        for (int c = x.first; c < x.first + x.pieces; ++c) {
                            const float* q = slot_of(c);
                            const float f = ex2(__ldcg(q + D * 128) - ref);
#pragma unroll
                            for (int i = 0; i < 32; ++i) acc[i] = __fmaf_rn(__ldcg(q + (ch + i) * 128), f, acc[i]);
                        }
                        uint32_t o[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(acc[i]);
                        store(o, ch, sum);
                    }
                    store_lse(top, sum);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.item_empty[round & 1]);
            kv += 2 * nt;
        }
    }

    __syncthreads();
    if (threadIdx.x == 0 && *abort) {
        raise_status(KVB_DEV_TIMEOUT);
        const uint32_t n = sh.kv_issued;
        for (uint32_t k = n > uint32_t(S::STAGES) ? n - S::STAGES : 0; k < n; ++k)
            mbar_wait(&sh.kv_full[k % S::STAGES], (k / S::STAGES) & 1, 10000000ull);
        if (sh.q_issued > 0) mbar_wait(&sh.q_full, (sh.q_issued - 1) & 1, 10000000ull);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(PF_TMEM_COLS));
}

}  // namespace kvb
