// kvb_rows_tc.cuh - what the attention kernels on the 5th-generation tensor cores share (kvb_cross_tc.cuh, kvb_shared_tc.cuh):
// groups of 256 query rows over units of 64 keys.
//
//   S = Q K^T,  x = scaling log2(e) S,  m = running row maximum of x,  P = 2^(x - m),  l = sum P,  O = P V,  out = O / l.
//
// One persistent CTA per SM takes an equal run of units (PdPlan), so that any mixture of lengths is balanced; items that a
// run's end cuts leave partial sums in the workspace, which a second kernel joins in the order of the keys.
//
// Two tiles of 128 rows, each with a warpgroup for its softmax (a thread a row) and a warp that issues O += P V; S of both in
// turn comes from another warp, so that one tile's softmax runs beside the other's products.  An item of more than 128 rows is two tiles
// of rows over the same keys; one of 128 or fewer is the same rows twice, the first tile over the even units and the second
// over the odd ones, joined at its end through shared memory: a single tile would leave the tensor cores idle during its softmax.
//
// Tensor memory: two S of 64 columns for each tile, O (128 columns each); P in 16 bits takes the columns of its S, from where it
// is the A operand of P V.  While a tile's softmax works on one S, the next is computed into the other columns, once the P V
// that reads the weights there is done (by barrier: the instruction set orders products of one accumulator only).  O is
// rescaled only when a row's maximum grew by more than 2^8.
//
// Every aligned instruction (tensor memory loads, stores, allocation; elect) is executed by whole warps: decisions before
// them are votes or the same in all lanes, and loops over lanes' own conditions end in __syncwarp.  Waits are bounded; after one that ran
// out a role ends (and then what waits for it), products and copies in flight are waited for (bounded), and tensor memory is
// freed.
#pragma once
#include <cuda.h>

#include <type_traits>

#include "kvb_paged_decode.cuh"

namespace kvb {

constexpr int CM_ROWS = 128;                  // of a tile
constexpr int CM_KEYS = 64;                   // of a unit
constexpr int CM_SOFTMAX = 8;                 // warps; then one that issues S, one per tile that issues O, and those that bring keys and values
constexpr int CM_FIXED = 6;                   // what an item costs beside its units, in units
constexpr int CM_TMEM = 512;
constexpr int CM_FMA = 1;                     // pairs of keys of four whose weights take the FMA pipe

template <int D>
struct CmShape {
    static constexpr int HALVES = D / 64;
    static constexpr int QHALF = CM_ROWS * 128, HALF = CM_KEYS * 128;           // bytes of 64 channels of a tile's queries, of a unit's keys
    static constexpr int QTILE = HALVES * QHALF, TILE = HALVES * HALF;
    static constexpr int XROWS = 32 * 32 + 3 * 32;               // floats a warp passes on at a time: 32 channels of its rows, maxima and sums
    static constexpr int XBYTES = 4 * XROWS * 4;
};

// Shared-memory matrix descriptors, 128-byte swizzle.  K-major: 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t cm_desc_k(uint32_t saddr) {
    return uint64_t((saddr >> 4) & 0x3FFF) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// MN-major: 64 channels a row, 8-key groups 1024 bytes apart, the other 64 channels `lead` bytes further
__device__ __forceinline__ uint64_t cm_desc_mn(uint32_t saddr, uint32_t lead) {
    return uint64_t((saddr >> 4) & 0x3FFF) | (uint64_t((lead >> 4) & 0x3FFF) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
           (uint64_t(2) << 61);
}
__host__ __device__ constexpr uint32_t cm_idesc(int N, int bf16, int b_mn) {
    return (1u << 4) | (uint32_t(bf16) << 7) | (uint32_t(bf16) << 10) | (uint32_t(b_mn) << 16) | (uint32_t(N >> 3) << 17) |
           (uint32_t(128 >> 4) << 24);
}
// Issued by one lane of a converged warp, the same every time.  (With the lane's own predicate a product takes 64 cycles to
// issue, from a branch of one lane more; elected, 64 x 64 x 16 and smaller ones go at their own rate.)
__device__ __forceinline__ void cm_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, int acc) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void cm_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, int acc) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void cm_commit(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void cm_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void cm_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of the thread's lane, waited for in the same statement: nothing reads the registers before
__device__ __forceinline__ void cm_ld32(uint32_t taddr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
// The 64 columns of S of the thread's lane, waited for in the same statement: nothing reads the registers before
__device__ __forceinline__ void cm_ld64(uint32_t taddr, float (&v)[64]) {
    uint32_t r[64];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
        "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
        "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
          "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
          "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
          "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]),
          "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]),
          "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}
// 32 columns of the thread's lane; cm_wait_st() before anyone else reads them
__device__ __forceinline__ void cm_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void cm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// two float32 values at once
__device__ __forceinline__ float2 cm_fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 cm_mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 cm_add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// a whole sector
__device__ __forceinline__ void cm_store32(void* to, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                 "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// the greatest of three, NaN if one is
__device__ __forceinline__ float cm_max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// 2^x of two values up to 2^22 on the FMA pipe: x = n + r, |r| <= 1/2, by rounding to integers (adding 1.5 2^23), a minimax
// polynomial of 2^r with value 1 at 0, n added to the exponent.  -127 and less give 0.  Relative error 2.8e-6 (of the fourth
// degree; with one of the third, 1.0e-4, the sums and so the log-sum-exp lost digits that float32 has).
__device__ __forceinline__ float2 cm_ex2(float2 x) {
    x.x = fmaxf(x.x, -127.f);
    x.y = fmaxf(x.y, -127.f);
    const float2 t = cm_add2(x, float2{12582912.f, 12582912.f});
    const float2 r = cm_fma2(cm_add2(t, float2{-12582912.f, -12582912.f}), float2{-1.f, -1.f}, x);
    float2 p = cm_fma2(float2{0.009582576341927052f, 0.009582576341927052f}, r, float2{0.05590682849287987f, 0.05590682849287987f});
    p = cm_fma2(p, r, float2{0.24024106562137604f, 0.24024106562137604f});
    p = cm_fma2(p, r, float2{0.6931241154670715f, 0.6931241154670715f});
    p = cm_fma2(p, r, float2{1.f, 1.f});
    return float2{__int_as_float(__float_as_int(p.x) + (__float_as_int(t.x) << 23)), __int_as_float(__float_as_int(p.y) + (__float_as_int(t.y) << 23))};
}

struct CmBars {
    uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4], q_full[2], drained[3], x_full[4], x_empty[4];
    uint64_t s_full[2][2], p_ready[2][2], pv_done[2][2];         // of a tile, by the half of its columns

    // `loads`: arrivals that fill a stage of keys or values
    __device__ void init(uint32_t loads) {
        for (int i = 0; i < 4; ++i) {
            mbar_init(&k_full[i], loads);
            mbar_init(&v_full[i], loads);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_empty[i], 2);
            mbar_init(&x_full[i], 1);
            mbar_init(&x_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 4);
            for (int k = 0; k < 2; ++k) {
                mbar_init(&s_full[i][k], 1);
                mbar_init(&p_ready[i][k], 4);
                mbar_init(&pv_done[i][k], 1);
            }
        }
        for (int i = 0; i < 3; ++i) mbar_init(&drained[i], 1);
    }
};

// a whole warp's wait, the same answer in all lanes
__device__ __forceinline__ bool cm_wait(uint64_t* bar, uint32_t count) { return __all_sync(0xffffffffu, mbar_wait(bar, count & 1)); }

// Units and places before each of n sequences, pre[0 .. n] and shares[0 .. n], from units_of(i, u, p): inclusive scans by the
// whole block, a block of threads at a time.  False when the sums pass 32 bits.
template <int WARPS, typename F>
__device__ __forceinline__ bool cm_scan(int n, int* pre, int* shares, int (*warp_sum)[WARPS], F units_of) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int before_u = 0, before_p = 0;
    if (threadIdx.x == 0) pre[0] = shares[0] = 0;
    for (int i0 = 0; i0 < n; i0 += 32 * WARPS) {
        const int i = i0 + threadIdx.x;
        int u = 0, p = 0;
        if (i < n) units_of(i, u, p);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int a = __shfl_up_sync(0xffffffffu, u, o), b = __shfl_up_sync(0xffffffffu, p, o);
            if (lane >= o) u += a, p += b;
        }
        __syncthreads();
        if (lane == 31) warp_sum[0][warp] = u, warp_sum[1][warp] = p;
        __syncthreads();
        int sum_u = 0, sum_p = 0;
        for (int w = 0; w < WARPS; ++w) {
            if (w == warp) u += sum_u, p += sum_p;
            sum_u += warp_sum[0][w], sum_p += warp_sum[1][w];
        }
        if (i < n) pre[i + 1] = before_u + u, shares[i + 1] = before_p + p;
        before_u += sum_u, before_p += sum_p;
    }
    __syncthreads();
    bool fits = true;                                            // a sum that passed 32 bits shows as one that falls
    for (int i = threadIdx.x; i < n; i += 32 * WARPS) fits &= shares[i + 1] >= shares[i] && pre[i + 1] >= pre[i];
    return __syncthreads_and(fits);
}

// The work of pre and shares in equal runs for `ctas` CTAs at most.
template <int FIXED>
__device__ __forceinline__ void cm_deal(PdPlan<true, FIXED>& W, int n, const int* pre, const int* shares, int ctas) {
    const int work = shares[n];
    W.pre = pre;
    W.shares = shares;
    W.n = n;
    W.hg = 0;
    W.ctas = max(1, min(ctas, work / PD_LEAST));
    W.quota = work / W.ctas;
    W.extra = work - W.quota * W.ctas;
}

// What the issuing warps know of a piece of an item: the units that pass, those with keys, the keys from its first unit on,
// whether the tiles share its units.
struct CmStep {
    int advance, tiles, left;
    bool split;
};
// the same in all lanes, known to the compiler as such
__device__ __forceinline__ CmStep cm_uniform(const CmStep& x) {
    return CmStep{__shfl_sync(0xffffffffu, x.advance, 0), __shfl_sync(0xffffffffu, x.tiles, 0), __shfl_sync(0xffffffffu, x.left, 0),
                  __shfl_sync(0xffffffffu, int(x.split), 0) != 0};
}
// units of tile t among `tiles`, and the number of its j-th
__device__ __forceinline__ int cm_units(bool split, int tiles, int t) { return split ? (tiles + 1 - t) / 2 : tiles; }
__device__ __forceinline__ int cm_unit(bool split, int t, int j) { return split ? 2 * j + t : j; }

// The warp that issues S = Q K^T: both tiles' in turn, unit by unit.  step_at(cur): the piece at unit cur.
template <int D, int BF16, int STAGES, typename F>
__device__ __forceinline__ void cm_issue_scores(CmBars& B, uint32_t tmem, uint32_t sq, uint32_t sk, int u0, int u1, F step_at) {
    using S = CmShape<D>;
    constexpr uint32_t IS = cm_idesc(CM_KEYS, BF16, 0);
    const uint64_t dq = cm_desc_k(sq), dk = cm_desc_k(sk);
    uint32_t it = 0, sn[2] = {0, 0}, items[2] = {0, 0};          // units of the block; S and items of the tiles
    bool ok = true;
    for (int cur = u0; cur < u1 && ok;) {
        const CmStep x = cm_uniform(step_at(cur));
        if (x.tiles > 0) ok = cm_wait(&B.q_full[0], items[0]++);
        if (ok && cm_units(x.split, x.tiles, 1) > 0) ok = cm_wait(&B.q_full[1], items[1]++);
        for (int u = 0; u < x.tiles && ok; ++u, ++it) {
            const uint32_t st = it % STAGES;
            const uint64_t k = dk + uint64_t(st * (S::TILE >> 4));
            ok = cm_wait(&B.k_full[st], it / STAGES);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if (!ok || (x.split && (u & 1) != t)) continue;
                const uint32_t half = sn[t] & 1;
                // the product two before, which reads the weights in these columns, is done
                if (sn[t] >= 2 && !(ok = cm_wait(&B.pv_done[t][half], (sn[t] >> 1) - 1))) continue;
                cm_after();
#pragma unroll
                for (int c = 0; c < D / 16; ++c)                 // descriptors count 16 bytes
                    cm_mma_ss(tmem + t * 128 + CM_KEYS * half, dq + uint64_t(t * (S::QTILE >> 4) + (c >> 2) * (S::QHALF >> 4) + (c & 3) * 2),
                              k + uint64_t((c >> 2) * (S::HALF >> 4) + (c & 3) * 2), IS, c > 0);
                cm_commit(&B.s_full[t][half]);
                ++sn[t];
            }
            if (ok) cm_commit(&B.k_empty[st]);
        }
        cur += x.advance;
    }
    if (!ok) {                                                   // products in flight end before tensor memory is freed
        cm_commit(&B.drained[0]);
        mbar_wait(&B.drained[0], 0, 10000000ull);
    }
    __syncwarp();
}

// The warp that issues O += P V of tile t (P of type bfloat16 or float16, as V is).
template <int D, int BF16, int STAGES, typename F>
__device__ __forceinline__ void cm_issue_values(CmBars& B, uint32_t tmem, uint32_t sv, int t, int u0, int u1, F step_at) {
    using S = CmShape<D>;
    constexpr uint32_t IO = cm_idesc(D, BF16, 1);
    const uint32_t ts = tmem + t * 128, to = tmem + 256 + t * 128, lane = threadIdx.x & 31;
    const uint64_t dv = cm_desc_mn(sv, S::HALF);
    uint32_t it = 0, sn = 0;
    bool ok = true;
    for (int cur = u0; cur < u1 && ok;) {
        const CmStep x = cm_uniform(step_at(cur));
        int first = 1;
        for (int u = 0; u < x.tiles && ok; ++u, ++it) {
            const uint32_t st = it % STAGES, half = sn & 1, p = ts + CM_KEYS * half;
            const uint64_t v = dv + uint64_t(st * (S::TILE >> 4));
            if (!(ok = cm_wait(&B.v_full[st], it / STAGES))) break;
            if (x.split && (u & 1) != t) {                       // the other tile's: the stage is free for this one
                if (lane == 0) mbar_arrive(&B.v_empty[st]);
                __syncwarp();
                continue;
            }
            if (!(ok = cm_wait(&B.p_ready[t][half], sn >> 1))) break;
            cm_after();
            const int steps = min((x.left - u * CM_KEYS + 15) / 16, CM_KEYS / 16);
#pragma unroll
            for (int c = 0; c < CM_KEYS / 16; ++c)
                if (c < steps) cm_mma_ts(to, p + 8 * c, v + uint64_t(c * (2048 >> 4)), IO, !first || c > 0);
            cm_commit(&B.pv_done[t][half]);
            cm_commit(&B.v_empty[st]);
            first = 0;
            ++sn;
        }
        cur += x.advance;
    }
    if (!ok) {
        cm_commit(&B.drained[1 + t]);
        mbar_wait(&B.drained[1 + t], 0, 10000000ull);
    }
    __syncwarp();
}

// O of the thread's row times f.
template <int D>
__device__ __forceinline__ void cm_rescale(uint32_t to, float f) {
#pragma unroll 1
    for (int c = 0; c < D / 32; ++c) {
        float v[32];
        cm_ld32(to + 32 * c, v);
        uint32_t w[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(v[i] * f);
        cm_st32(to + 32 * c, w);
    }
}

// A cut item's partial in the workspace, two a CTA (of its first item, of its last): O (256 rows, D), then the rows' maxima, sums
// and, where the values have a reference of their own (WREF), that.
template <int D>
constexpr int CM_PART = 2 * CM_ROWS * (D + 3);

// What the joining kernel is told of an item that a CTA's run begins and its end cuts: rows, parts (slot0, then slots 2 c of the
// CTAs up to c1), and I, which it hands to the function that stores the rows.
template <typename I>
struct CmCut {
    int rows, slot0, c0, c1;
    I item;
};

// Of CTA `cta`, by one thread: item_of(piece, item) gives the rows.
template <int FIXED, typename I, typename F>
__device__ __forceinline__ void cm_note_cut(const PdPlan<true, FIXED>& W, int cta, CmCut<I>* cuts, F item_of) {
    CmCut<I> x{};
    const int u = cta + 1 < W.ctas ? W.units_before(W.share(cta + 1)) : 0;
    if (u > 0 && u < W.pre[W.n]) {
        const PdPiece p = pd_piece(W, u, u + 1);
        if (p.a > 0 && u - p.a >= W.units_before(W.share(cta))) {
            x.rows = item_of(p, x.item);
            x.c0 = W.holder(p.v0 + FIXED);
            x.c1 = W.holder(p.v0 + FIXED + p.units - 1);
            // the partial of c0 is its first one, unless the item begins inside its run
            x.slot0 = 2 * x.c0 + (W.share(x.c0) < p.v0 ? 1 : 0);
        }
    }
    cuts[cta] = x;
}

// Joining, in a kernel of its own after the first (a row's parts may be a hundred, and joined by the block that finishes an item
// they were most of its time): a warp takes a row of a cut item (two of 64 channels), the parts in the order of the keys.
constexpr int CJ_WARPS = 8;                   // a thread for each CTA of the first kernel at least
constexpr int CJ_CH = 4;                      // channels of a lane

template <int D, bool WREF, typename I, typename F>
__device__ __forceinline__ void cm_join(const CmCut<I>* cuts, int ctas, const float* part, F finish) {
    __shared__ CmCut<I> cut[32 * CJ_WARPS];
    __shared__ int before[32 * CJ_WARPS + 1], warp_sum[CJ_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, id = threadIdx.x;
    chain_kernels();
    CmCut<I> mine{};
    if (id < ctas) mine = cuts[id];
    cut[id] = mine;
    constexpr int LANES = D / CJ_CH, PER = 32 / LANES;           // of a row; rows of a warp
    int x = (mine.rows + PER - 1) / PER;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) warp_sum[warp] = x;
    __syncthreads();
    for (int w = 0; w < warp; ++w) x += warp_sum[w];
    before[id + 1] = x;
    if (id == 0) before[0] = 0;
    __syncthreads();
    for (int task = blockIdx.x * CJ_WARPS + warp; task < before[32 * CJ_WARPS]; task += gridDim.x * CJ_WARPS) {
        int lo = 0;
#pragma unroll
        for (int step = 16 * CJ_WARPS; step > 0; step >>= 1)
            if (before[lo + step] <= task) lo += step;
        const CmCut<I>& c = cut[lo];
        const int row = (task - before[lo]) * PER + lane / LANES, ch = lane % LANES * CJ_CH;
        if (row >= c.rows) continue;
        constexpr int B = 4;                                     // parts whose loads are in flight together
        float top = -INFINITY, topw = -INFINITY, sum = 0.f, acc[CJ_CH];
#pragma unroll
        for (int i = 0; i < CJ_CH; ++i) acc[i] = 0.f;
#pragma unroll 1
        for (int k0 = c.c0; k0 <= c.c1; k0 += B) {
            float m[B], l[B], w[B];
            float4 o[B];
#pragma unroll
            for (int k = 0; k < B; ++k) {
                const float* from = part + int64_t(k0 + k == c.c0 ? c.slot0 : 2 * (k0 + k)) * CM_PART<D>;
                const bool ok = k0 + k <= c.c1;
                const float* st = from + 2 * CM_ROWS * D + row;
                m[k] = ok ? __ldcg(st) : -INFINITY;
                l[k] = ok ? __ldcg(st + 2 * CM_ROWS) : 0.f;
                w[k] = !WREF ? m[k] : ok ? __ldcg(st + 4 * CM_ROWS) : -INFINITY;
                o[k] = ok ? __ldcg(reinterpret_cast<const float4*>(from + row * D + ch)) : float4{0.f, 0.f, 0.f, 0.f};
            }
            float most = top, mostw = topw;
#pragma unroll
            for (int k = 0; k < B; ++k) most = fmaxf(most, m[k]), mostw = fmaxf(mostw, w[k]);
            const float ref = most == -INFINITY ? 0.f : most, refw = mostw == -INFINITY ? 0.f : mostw;
            sum *= ex2(top - ref);
            const float old = ex2(topw - refw);
#pragma unroll
            for (int i = 0; i < CJ_CH; ++i) acc[i] *= old;
#pragma unroll
            for (int k = 0; k < B; ++k) {
                if (k0 + k > c.c1) break;
                sum = __fmaf_rn(l[k], ex2(m[k] - ref), sum);
                const float f = ex2(w[k] - refw);
                acc[0] = __fmaf_rn(o[k].x, f, acc[0]);
                acc[1] = __fmaf_rn(o[k].y, f, acc[1]);
                acc[2] = __fmaf_rn(o[k].z, f, acc[2]);
                acc[3] = __fmaf_rn(o[k].w, f, acc[3]);
            }
            top = most, topw = mostw;
        }
        finish(c.item, row, ch, acc, top, sum, topw);
    }
}

// 32 channels of a row of 32-bit values
__device__ __forceinline__ void cm_put(float* to, const float (&v)[32]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = __float_as_uint(v[8 * i + k]);
        cm_store32(to + 8 * i, w);
    }
}

__device__ __forceinline__ float cm_inverse(float sum) { return sum > 0.f ? 1.f / sum : (sum == sum ? 0.f : sum); }

}  // namespace kvb
