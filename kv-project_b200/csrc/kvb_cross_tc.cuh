// kvb_cross_tc.cuh - attention of packed queries to keys of another length (an encoder's states), many queries per sequence,
// on the 5th-generation tensor cores.
//
//   S = Q K^T,  x = scaling log2(e) S,  m = running row maximum of x,  P = 2^(x - m),  l = sum P,  O = P V,  out = O / l,
// over all keys of the sequence.
//
// One persistent CTA per SM.  A work item is a group of 256 query rows (row = token * rep + head in the group: the rep query
// heads of a KV head and the sequence's queries packed together) of one (sequence, KV head), a unit of work its product with
// 64 keys; every CTA takes an equal run of units, found from the offsets inside the kernel, so that any mixture of lengths is
// balanced.  Items that a run's end cuts leave partial sums in the workspace, and the last warp to arrive joins them in the
// order of the keys.
//
// The 256 rows are two tiles of 128, each with a warpgroup for its softmax (a thread a row) and a warp that issues O += P V;
// S of both in turn comes from another, so that one tile's softmax runs beside the other's products; both read the same keys and values, which one warp
// copies with TMA through rings.  Tensor memory: two S of 64 columns for each tile, O (128 columns each); P is rounded to the
// inputs' type and takes the columns of its S, from where it is the A operand of P V.  While a tile's softmax works on one S,
// the next is computed into the other columns, once the P V that reads the weights there is done (by barrier: the instruction
// set orders products of one accumulator only).  O is rescaled only when a row's maximum grew by more than 2^8.
//
// Every aligned instruction (tensor memory loads, stores, allocation) is executed by whole warps: decisions before them are
// votes, and loops over lanes' own conditions end in __syncwarp.  Waits are bounded; after one that ran out nothing is issued any
// more, products and copies in flight are waited for (bounded), and tensor memory is freed.
//
// Values past a sequence's end belong to the next one: their weight is zero, but zero times NaN is not, so the rows of the
// last 16 that lie past the end are zeroed in shared memory, and steps of 16 keys behind them left out.
#pragma once
#include <cuda.h>

#include <type_traits>

#include "kvb_cross.cuh"

namespace kvb {

constexpr int CM_ROWS = 128;                  // of a tile
constexpr int CM_KEYS = 64;                   // of a unit
constexpr int CM_SOFTMAX = 8;                 // warps
constexpr int CM_WARPS = CM_SOFTMAX + 4;      // and one that issues S, one per tile that issues O, and the copying warp
constexpr int CM_FIXED = 6;                   // what an item costs beside its units, in units
constexpr int CM_TMEM = 512;
constexpr int CM_FMA = 1;                     // pairs of keys of four whose weights take the FMA pipe

template <int D>
struct CmShape {
    static constexpr int HALVES = D / 64;
    static constexpr int QHALF = CM_ROWS * 128, HALF = CM_KEYS * 128;           // bytes of 64 channels of a tile's queries, of a unit's keys
    static constexpr int QTILE = HALVES * QHALF, TILE = HALVES * HALF;
    static constexpr int STAGES = 4;                            // of keys and of values
    static constexpr int SMEM = 1024 + 2 * QTILE + 2 * STAGES * TILE;
    static constexpr int PART = 2 * (D + 2) * CM_ROWS;          // floats: O by column and row, maximum, sum of the two tiles
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
// polynomial of 2^r with value 1 at 0, n added to the exponent.  -127 and less give 0.  Relative error 1.01e-4 (third degree,
// beside bfloat16's 2^-8) or 2.8e-6 (fourth, beside float16's 2^-11).
template <typename T>
__device__ __forceinline__ float2 cm_ex2(float2 x) {
    x.x = fmaxf(x.x, -127.f);
    x.y = fmaxf(x.y, -127.f);
    const float2 t = cm_add2(x, float2{12582912.f, 12582912.f});
    const float2 r = cm_fma2(cm_add2(t, float2{-12582912.f, -12582912.f}), float2{-1.f, -1.f}, x);
    float2 p;
    if constexpr (std::is_same<T, __half>::value) {
        p = cm_fma2(float2{0.009582576341927052f, 0.009582576341927052f}, r, float2{0.05590682849287987f, 0.05590682849287987f});
        p = cm_fma2(p, r, float2{0.24024106562137604f, 0.24024106562137604f});
        p = cm_fma2(p, r, float2{0.6931241154670715f, 0.6931241154670715f});
    } else {
        p = cm_fma2(float2{0.055009059607982635f, 0.055009059607982635f}, r, float2{0.2422109693288803f, 0.2422109693288803f});
        p = cm_fma2(p, r, float2{0.6932829022407532f, 0.6932829022407532f});
    }
    p = cm_fma2(p, r, float2{1.f, 1.f});
    return float2{__int_as_float(__float_as_int(p.x) + (__float_as_int(t.x) << 23)), __int_as_float(__float_as_int(p.y) + (__float_as_int(t.y) << 23))};
}

struct CmBars {
    uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4], q_full[2], drained[3];
    uint64_t s_full[2][2], p_ready[2][2], pv_done[2][2];         // of a tile, by the half of its columns
};

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
    uint8_t* const sv = sk + S::STAGES * S::TILE;
    // the warp's number from a shuffle: the compiler then knows it, and what follows from it, to be the same in all lanes
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 4; ++i) {
            mbar_init(&B.k_full[i], 1);
            mbar_init(&B.v_full[i], 1);
            mbar_init(&B.k_empty[i], 1);
            mbar_init(&B.v_empty[i], 2);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&B.q_full[i], 4);
            for (int k = 0; k < 2; ++k) {
                mbar_init(&B.s_full[i][k], 1);
                mbar_init(&B.p_ready[i][k], 4);
                mbar_init(&B.pv_done[i][k], 1);
            }
        }
        for (int i = 0; i < 3; ++i) mbar_init(&B.drained[i], 1);
        fence_mbar_init();
        pre[0] = shares[0] = 0;
    }
    chain_kernels();
    auto seq_at = [&](int i) { return cr_seq(A.cu_q, A.cu_k, A.nq, A.nk, i); };
    // units and places before each sequence: inclusive scans, a block of threads at a time
    int before_u = 0, before_p = 0;
    for (int i0 = 0; i0 < A.n; i0 += 32 * CM_WARPS) {
        const int i = i0 + threadIdx.x;
        int u = 0, p = 0;
        if (i < A.n) {
            const CrSeq x = seq_at(i);
            const int hg = int((int64_t(x.ql) * A.rep + 2 * CM_ROWS - 1) / (2 * CM_ROWS)) * A.Hkv;
            u = max(1, (x.kl + CM_KEYS - 1) / CM_KEYS) * hg;     // without keys one empty unit: its rows are written
            p = u + CM_FIXED * hg;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int a = __shfl_up_sync(0xffffffffu, u, o), b = __shfl_up_sync(0xffffffffu, p, o);
            if (lane >= o) u += a, p += b;
        }
        __syncthreads();
        if (lane == 31) warp_sum[0][warp] = u, warp_sum[1][warp] = p;
        __syncthreads();
        int sum_u = 0, sum_p = 0;
        for (int w = 0; w < CM_WARPS; ++w) {
            if (w == warp) u += sum_u, p += sum_p;
            sum_u += warp_sum[0][w], sum_p += warp_sum[1][w];
        }
        if (i < A.n) pre[i + 1] = before_u + u, shares[i + 1] = before_p + p;
        before_u += sum_u, before_p += sum_p;
    }
    __syncthreads();
    bool fits = true;                                            // offsets that do not ascend may hold more work than 32 bits do
    for (int i = threadIdx.x; i < A.n; i += 32 * CM_WARPS) fits &= shares[i + 1] >= shares[i] && pre[i + 1] >= pre[i];
    if (!__syncthreads_and(fits)) {
        if (threadIdx.x == 0) raise_status(KVB_DEV_BOUNDS);
        return;
    }
    const int work = shares[A.n];
    if (work == 0) return;
    PdPlan<PD_SEGMENTS, CM_FIXED> W;
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

    if (warp == CM_SOFTMAX) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(CM_TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    cm_before();
    __syncthreads();
    cm_after();
    const uint32_t tmem = s_tmem;
    // a whole warp's wait, the same answer in all lanes; after one that ran out a role ends, and so does what waits for it
    auto wait = [&](uint64_t* bar, uint32_t count) { return bool(__all_sync(0xffffffffu, mbar_wait(bar, count & 1))); };
    // the piece that begins at unit `cur`
    struct Item {
        PdPiece p;
        CrSeq s;
        int h, row0, nrows, tiles;                               // KV head, first row, rows, key tiles
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

    if (warp < CM_SOFTMAX) {
        // ---------------- softmax of tile t: thread = row ----------------
        const int t = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
        const uint32_t lanes = uint32_t(quarter * 32) << 16, ts = tmem + lanes + t * 128, to = tmem + lanes + 256 + t * 128;
        auto load_q = [&](const Item& x) {                       // the warp's 32 rows of the tile, swizzled; zeros past the last
            constexpr int CHUNKS = D / 8, PER = 32 / CHUNKS;     // 16-byte chunks of a row, rows at a time
            const int c = lane % CHUNKS;
            uint4 v[32 / PER];
#pragma unroll
            for (int i = 0; i < 32 / PER; ++i) {
                const int row = t * CM_ROWS + quarter * 32 + i * PER + lane / CHUNKS, at = x.row0 + row, tok = pd_div(at, A.by_rep);
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
        auto rescale = [&](float f) {                            // O of the row times f
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                float v[32];
                cm_ld32(to + 32 * c, v);
                uint32_t w[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(v[i] * f);
                cm_st32(to + 32 * c, w);
            }
        };
        auto has_work = [&](const Item& x) { return x.tiles > 0 && x.nrows > t * CM_ROWS; };
        Item x{};
        if (u0 < u1) {
            x = item_at(u0);
            if (has_work(x)) load_q(x);
        }
        uint32_t sn = 0, it = 0;                                 // S of this tile so far; key tiles of the block
        int first = 1;
        bool ok = true;
        for (int cur = u0; cur < u1 && ok;) {
            const bool mine = x.nrows > t * CM_ROWS;
            float m = -INFINITY, l = 0.f;
            if (mine) {
                for (int j = 0; j < x.tiles; ++j, ++sn) {
                    const uint32_t half = sn & 1, cols = ts + CM_KEYS * half;
                    if (!(ok = wait(&B.s_full[t][half], sn >> 1))) break;
                    cm_after();
                    const int left = x.s.kl - (x.p.a + j) * CM_KEYS;             // keys of the sequence from this unit on
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
                        if (j > 0) {                             // once the product before is done
                            if (!(ok = wait(&B.pv_done[t][half ^ 1], (sn - 1) >> 1))) break;
                            cm_after();
                            rescale(f);
                        }
                    }
                    const float ref = m == -INFINITY ? 0.f : m;
                    const float2 lam2{A.lam, A.lam}, ref2{-ref, -ref};
                    float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
                    uint32_t w[CM_KEYS / 2];
                    // of four pairs of keys CM_FMA on the FMA pipe: with all on the special-function unit, which the two
                    // warpgroups share, it is what bounds the step
                    auto weights = [&](auto plain) {
#pragma unroll
                        for (int i = 0; i < CM_KEYS / 2; ++i) {
                            float2 e = cm_fma2(float2{v[2 * i], v[2 * i + 1]}, lam2, ref2);
                            if (plain && i % 4 < CM_FMA) {
                                e = cm_ex2<T>(e);
                            } else {
                                e.x = ex2(e.x);
                                e.y = ex2(e.y);
                            }
                            sum[i & 1] = cm_add2(sum[i & 1], e);
                            w[i] = pack_f32<T>(e.x, e.y);
                        }
                    };
                    // NaN and infinities, masked keys and rows that have seen nothing want the exact limits
                    if (__all_sync(0xffffffffu, fabsf(y) < INFINITY) && left >= CM_KEYS) weights(std::true_type{});
                    else weights(std::false_type{});
                    cm_st32(cols, w);
                    const float2 both = cm_add2(sum[0], sum[1]);
                    l += both.x + both.y;
                    if (left < CM_KEYS) {                        // value rows past the end, up to the last step's 16
                        const uint32_t st = (it + j) % S::STAGES;
                        if (!(ok = wait(&B.v_full[st], (it + j) / S::STAGES))) break;
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
            }
            if (!ok) break;
            it += x.tiles;
            const Item done = x;
            const int next = cur + x.p.b - x.p.a;
            if (next < u1) {                                     // all products with this item's queries are done
                x = item_at(next);
                if (has_work(x)) load_q(x);
            }
            if (mine) {
                if (done.tiles > 0 && !(ok = wait(&B.pv_done[t][(sn - 1) & 1], (sn - 1) >> 1))) break;     // nothing is written
                cm_after();
                const bool whole = done.p.a == 0 && done.p.b == done.p.units;
                const bool row_ok = t * CM_ROWS + r < done.nrows;
                const int at = done.row0 + t * CM_ROWS + r, tok = pd_div(at, A.by_rep);
                const int64_t row = (int64_t(done.s.q0) + tok) * A.Hq + done.h * A.rep + at - tok * A.rep;
                auto store = [&](int c, const float (&v)[32], float inv) {       // 32 channels of the row
                    if (!row_ok) return;
                    T* to = static_cast<T*>(A.out) + row * D + 32 * c;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t w[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) w[k] = pack_f32<T>(v[16 * i + 2 * k] * inv, v[16 * i + 2 * k + 1] * inv);
                        cm_store32(to + 16 * i, w);
                    }
                };
                auto finish = [&](float top, float sum) {
                    if (A.lse && row_ok) A.lse[row] = sum == 0.f ? -INFINITY : top * 0.693147180559945309f + logf(sum);
                };
                auto inverse = [](float sum) { return sum > 0.f ? 1.f / sum : (sum == sum ? 0.f : sum); };
                if (done.tiles == 0) {
                    float v[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = 0.f;
                    for (int c = 0; c < D / 32; ++c) store(c, v, 0.f);
                    finish(0.f, 0.f);
                } else if (whole) {
                    const float inv = inverse(l);
#pragma unroll 1
                    for (int c = 0; c < D / 32; ++c) {
                        float v[32];
                        cm_ld32(to + 32 * c, v);
                        store(c, v, inv);
                        __syncwarp();
                    }
                    finish(m, l);
                } else {
                    auto part_of = [&](int slot) { return A.part + int64_t(slot) * S::PART + t * (D + 2) * CM_ROWS + r; };
                    float* part = part_of(2 * cta + (first ? 0 : 1));
#pragma unroll 1
                    for (int c = 0; c < D / 32; ++c) {
                        float v[32];
                        cm_ld32(to + 32 * c, v);
#pragma unroll
                        for (int i = 0; i < 32; ++i) __stcg(part + (32 * c + i) * CM_ROWS, v[i]);
                    }
                    __stcg(part + D * CM_ROWS, m);
                    __stcg(part + (D + 1) * CM_ROWS, l);
                    // the CTAs c0 .. c1 hold the item's units: the last warp to arrive joins its 32 rows
                    const int c0 = W.holder(done.p.v0 + CM_FIXED), c1 = W.holder(done.p.v0 + CM_FIXED + done.p.units - 1);
                    uint32_t* count = A.count + c0 * CM_SOFTMAX + warp;
                    uint32_t seen = 0;
                    __syncwarp();
                    if (lane == 0) seen = atomic_add_acq_rel(count, 1u);
                    seen = __shfl_sync(0xffffffffu, seen, 0);
                    if (seen > uint32_t(c1 - c0)) {
                        if (lane == 0) raise_status(KVB_DEV_WORKSPACE);
                    } else if (seen == uint32_t(c1 - c0)) {
                        if (lane == 0) *count = 0;
                        // the partial of c is its first one, unless the item begins inside c's run
                        const int slot0 = 2 * c0 + (W.share(c0) < done.p.v0 ? 1 : 0);
                        auto from = [&](int c) { return part_of(c == c0 ? slot0 : 2 * c); };
                        float top = -INFINITY, all = 0.f;
                        for (int c = c0; c <= c1; ++c) top = fmaxf(top, __ldcg(from(c) + D * CM_ROWS));
                        const float ref = top == -INFINITY ? 0.f : top;
                        for (int c = c0; c <= c1; ++c) all = __fmaf_rn(__ldcg(from(c) + (D + 1) * CM_ROWS), ex2(__ldcg(from(c) + D * CM_ROWS) - ref), all);
                        const float inv = inverse(all);
#pragma unroll 1
                        for (int c32 = 0; c32 < D / 32; ++c32) {
                            float v[32];
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = 0.f;
#pragma unroll 1
                            for (int c = c0; c <= c1; ++c) {
                                const float* o = from(c);
                                const float f = ex2(__ldcg(o + D * CM_ROWS) - ref);
#pragma unroll
                                for (int i = 0; i < 32; ++i) v[i] = __fmaf_rn(__ldcg(o + (32 * c32 + i) * CM_ROWS), f, v[i]);
                            }
                            store(c32, v, inv);
                        }
                        finish(top, all);
                    }
                }
                __syncwarp();
                cm_before();                                     // O is read: the next product into it comes after the next P
            }
            cur = next;
            first = 0;
        }
    } else if (warp < CM_SOFTMAX + 3) {
        // ---------------- products: S = Q K^T of both tiles in turn from one warp, O += P V of each from another ----------------
        const int role = warp - CM_SOFTMAX;
        constexpr uint32_t IS = cm_idesc(CM_KEYS, BF16, 0), IO = cm_idesc(D, BF16, 1);
        uint32_t it = 0, sn[2] = {0, 0}, items[2] = {0, 0};      // units of the block; S and items of the tiles
        bool ok = true;
        for (int cur = u0; cur < u1 && ok;) {
            const Item x = item_at(cur);
            const int tiles = __shfl_sync(0xffffffffu, x.tiles, 0), left = __shfl_sync(0xffffffffu, x.s.kl - x.p.a * CM_KEYS, 0);
            const bool both = __shfl_sync(0xffffffffu, x.nrows, 0) > CM_ROWS;
            if (role == 0) {
                const uint64_t dq = cm_desc_k(smem_u32(sq)), dk = cm_desc_k(smem_u32(sk));
                if (tiles > 0) ok = wait(&B.q_full[0], items[0]++) && (!both || wait(&B.q_full[1], items[1]++));
                for (int j = 0; j < tiles && ok; ++j, ++it) {
                    const uint32_t st = it % S::STAGES;
                    const uint64_t k = dk + uint64_t(st * (S::TILE >> 4));
                    ok = wait(&B.k_full[st], it / S::STAGES);
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (!ok || (t == 1 && !both)) break;
                        const uint32_t half = sn[t] & 1;
                        // the product two before, which reads the weights in these columns, is done
                        if (sn[t] >= 2 && !(ok = wait(&B.pv_done[t][half], (sn[t] >> 1) - 1))) break;
                        cm_after();
#pragma unroll
                        for (int c = 0; c < D / 16; ++c)         // descriptors count 16 bytes
                            cm_mma_ss(tmem + t * 128 + CM_KEYS * half, dq + uint64_t(t * (S::QTILE >> 4) + (c >> 2) * (S::QHALF >> 4) + (c & 3) * 2),
                                      k + uint64_t((c >> 2) * (S::HALF >> 4) + (c & 3) * 2), IS, c > 0);
                        cm_commit(&B.s_full[t][half]);
                        ++sn[t];
                    }
                    if (ok) cm_commit(&B.k_empty[st]);
                }
            } else {
                const int t = role - 1;
                const uint32_t ts = tmem + t * 128, to = tmem + 256 + t * 128;
                const uint64_t dv = cm_desc_mn(smem_u32(sv), S::HALF);
                for (int j = 0; j < tiles && ok; ++j, ++it) {
                    const uint32_t st = it % S::STAGES, half = sn[0] & 1, p = ts + CM_KEYS * half;
                    const uint64_t v = dv + uint64_t(st * (S::TILE >> 4));
                    if (!(ok = wait(&B.v_full[st], it / S::STAGES))) break;
                    if (t == 1 && !both) {                       // nothing to multiply: the stage is free for this tile
                        if (lane == 0) mbar_arrive(&B.v_empty[st]);
                        __syncwarp();
                        continue;
                    }
                    if (!(ok = wait(&B.p_ready[t][half], sn[0] >> 1))) break;
                    cm_after();
                    const int steps = min((left - j * CM_KEYS + 15) / 16, CM_KEYS / 16);
#pragma unroll
                    for (int c = 0; c < CM_KEYS / 16; ++c)
                        if (c < steps) cm_mma_ts(to, p + 8 * c, v + uint64_t(c * (2048 >> 4)), IO, j > 0 || c > 0);
                    cm_commit(&B.pv_done[t][half]);
                    cm_commit(&B.v_empty[st]);
                    ++sn[0];
                }
            }
            cur += __shfl_sync(0xffffffffu, x.p.b - x.p.a, 0);
        }
        if (!ok) {                                               // products in flight end before tensor memory is freed
            cm_commit(&B.drained[role]);
            mbar_wait(&B.drained[role], 0, 10000000ull);
        }
        __syncwarp();
    } else {
        // ---------------- copies ----------------
        uint32_t it = 0;
        bool ok = true;
        for (int cur = u0; cur < u1 && ok;) {
            const Item x = item_at(cur);
            for (int j = 0; j < x.tiles && ok; ++j, ++it) {
                const uint32_t st = it % S::STAGES, use = it / S::STAGES;
                const int row = x.s.k0 + (x.p.a + j) * CM_KEYS;
                if (it >= S::STAGES && !(ok = wait(&B.k_empty[st], use - 1))) break;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&B.k_full[st], S::TILE);
                    for (int c = 0; c < S::HALVES; ++c)
                        tma_load_3d(sk + st * S::TILE + c * S::HALF, &A.tm_k, 64 * c, x.h * A.k_heads, row, &B.k_full[st]);
                }
                __syncwarp();
                if (it >= S::STAGES && !(ok = wait(&B.v_empty[st], use - 1))) {
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
        for (uint32_t k = it > S::STAGES ? it - S::STAGES : 0; k < it; ++k) {
            mbar_wait(&B.k_full[k % S::STAGES], (k / S::STAGES) & 1, 10000000ull);
            mbar_wait(&B.v_full[k % S::STAGES], (k / S::STAGES) & 1, 10000000ull);
        }
        __syncwarp();
    }
    cm_before();
    __syncthreads();
    cm_after();
    if (warp == CM_SOFTMAX) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(CM_TMEM));
}

}  // namespace kvb
