// kvb_pages.cuh - the 8-bit paged KV cache: what fills it, reads it back and moves its pages.
//
// A page holds `page` consecutive tokens of one sequence for every KV head: codes (Hkv, page, d) uint8 for
// keys and for values, and one float32 scale per (page, head) and side.  A stored value is
// (code - 128) * scale; codes lie in [1, 255], so 128 is zero and -127 .. 127 are symmetric.
//
//   write    s = max |x| / 127 over the page's rows so far (non-finite x left out; 0 where that maximum is
//            below 2^-100), code = clamp(rint(x * (1 / s)), -127, 127) + 128, NaN -> 128.  Rows that are
//            already in the page keep it as long as it suffices: s = max(s_old, s_new rows); where it grows
//            they are recoded from their codes, code' = rint((code - 128) * (s_old / s)) + 128.  Each
//            operation is one float32 rounding, so the codes are a function of the writes alone.
//   extend   pages for sequences that grow; a fresh page is the lowest id whose reference count is zero
//   fork     a sequence becomes a copy of another: full pages are shared (reference counts), the last
//            partial page is copied, because it will be written
//   free     drops a sequence's references
//   compact  live pages with id >= n_live move, in ascending order, into the holes below, in ascending
//            order, so that the pool's first n_live pages are the live ones
//   copy     whole pages, codes and scales
//
// All of it moves bytes: the floor is the bytes read and written at the measured copy bandwidth, and for
// small calls the launches.
#pragma once

#include <type_traits>

#include "kvb_pages_view.cuh"

namespace kvb {

// The sequence whose packed rows hold virtual page slot x: sequence i owns the slots from
// cu[i] / page + 2 i on, which are enough for every page that its rows touch (cu[i + 1] - cu[i] rows touch at
// most that difference / page + 2 pages).  Whole warp; 32-way search, so one round trip for n <= 32.
__device__ __forceinline__ int touch_sequence(const int32_t* cu, int n, int page, int64_t x, int64_t& slot0) {
    const int lane = threadIdx.x & 31;
    int lo = 0, len = n;
    while (true) {
        const int step = (len + 31) / 32;
        const int i = lo + lane * step;
        const bool le = i < lo + len && int64_t(cu[i] >> page_shift(page)) + 2 * int64_t(i) <= x;
        const int k = 31 - __clz(int(__ballot_sync(0xffffffffu, le) | 1u));
        lo += k * step;
        len = min(step, n - lo);
        if (step == 1) break;
    }
    slot0 = int64_t(cu[lo] >> page_shift(page)) + 2 * int64_t(lo);
    return lo;
}

// One page's part of a packed write or read.
struct Touch {
    int slot, block;      // the page is table[slot][block]; slot < 0: nothing to do
    int row0, rows;       // rows of the page
    int64_t token0;       // first packed row
};

__device__ __forceinline__ Touch find_touch(const PagesView& P, const int32_t* slots, const int32_t* start,
                                            const int32_t* cu, int n, int64_t rows, int64_t x) {
    Touch t{-1, 0, 0, 0, 0};
    int64_t slot0;
    const int i = touch_sequence(cu, n, P.page, x, slot0);
    const int a = cu[i], b = cu[i + 1], st = start[i], slot = slots[i];
    if (st < 0 || b <= a) return t;
    const int64_t block = (st >> page_shift(P.page)) + (x - slot0);
    const int64_t lo = imax64(st, block * P.page), hi = imin64(int64_t(st) + (b - a), (block + 1) * P.page);
    if (lo >= hi) return t;
    if (a < 0 || b > rows || slot < 0 || slot >= P.n_slots || block >= P.max_blocks) {
        raise_status(KVB_DEV_BOUNDS);
        return t;
    }
    t.slot = slot;
    t.block = int(block);
    t.row0 = int(lo - block * P.page);
    t.rows = int(hi - lo);
    t.token0 = a + (lo - st);
    return t;
}

// The page of a touch, or -1 (with the status bit).
__device__ __forceinline__ int64_t touch_page(const PagesView& P, const Touch& t) {
    const int id = P.table[int64_t(t.slot) * P.max_blocks + t.block];
    if (id >= 0 && id < P.n_pages) return id;
    raise_status(KVB_DEV_BOUNDS);
    return -1;
}

// max over the block of non-negative floats
__device__ __forceinline__ float block_max(float v, float* sh) {
    v = warp_max(v);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    float m = 0.f;
    for (int w = 0; w < int(blockDim.x >> 5); ++w) m = fmaxf(m, sh[w]);
    return m;
}

__device__ __forceinline__ uint8_t code8(float x, float inv) {
    const float c = x * inv;
    return uint8_t(int(c != c ? 0.f : fminf(fmaxf(rintf(c), -127.f), 127.f)) + 128);
}

struct PageRowsParams {
    PagesView P;
    const int32_t* slots;
    const int32_t* start;
    const int32_t* cu;
    int n;
    int64_t rows;
    const void* x[2];              // k, v
    int64_t row_stride[2], head_stride[2];
    void* out[2];                  // read: dense (rows, Hkv, d)
    int whole;                     // read: out is 32-byte aligned, a thread stores whole sectors
};

// scale of a page that has `old` and takes rows of magnitude up to a
__device__ __forceinline__ float page_scale(float old, float a) { return fmaxf(old, a < 0x1p-100f ? 0.f : __fdiv_rn(a, 127.f)); }

// Recode the rows before the first new one for a scale that grew; whole block, 16 codes a thread and round.
__device__ __forceinline__ void recode_rows(uint8_t* codes, int n, float ratio) {
    for (int e = threadIdx.x * 16; e < n; e += blockDim.x * 16) {
        uint4 w = *reinterpret_cast<uint4*>(codes + e);
        uint8_t* c = reinterpret_cast<uint8_t*>(&w);
#pragma unroll
        for (int i = 0; i < 16; ++i) c[i] = uint8_t(int(rintf(float(int(c[i]) - 128) * ratio)) + 128);
        *reinterpret_cast<uint4*>(codes + e) = w;
    }
}

// Any type, strides and alignment, the rows read twice.  grid (touch slots, Hkv, 2)
template <typename T>
__global__ void page_write_any_kernel(const __grid_constant__ PageRowsParams A) {
    chain_kernels();
    __shared__ float sh[32];
    const PagesView& P = A.P;
    const int h = blockIdx.y, side = blockIdx.z;
    const Touch t = find_touch(P, A.slots, A.start, A.cu, A.n, A.rows, blockIdx.x);
    if (t.slot < 0) return;
    const int64_t page = touch_page(P, t);
    if (page < 0) return;
    if (P.refs[page] > 1) {                    // a page that several sequences hold is not written
        if (threadIdx.x == 0) raise_status(KVB_DEV_BOUNDS);
        return;
    }
    const T* x = static_cast<const T*>(A.x[side]) + t.token0 * A.row_stride[side] + h * A.head_stride[side];
    uint8_t* codes = (side ? P.vc : P.kc) + (page * P.Hkv + h) * int64_t(P.page) * P.d;
    float* scale = (side ? P.vs : P.ks) + page * P.Hkv + h;
    const float old = t.row0 > 0 ? *scale : 0.f;
    const int total = t.rows * P.d;
    float a = 0.f;
    for (int e = threadIdx.x; e < total; e += blockDim.x) {
        const float v = to_f32(x[(e / P.d) * A.row_stride[side] + e % P.d]);
        a = fmaxf(a, fabsf(v) < INFINITY ? fabsf(v) : 0.f);
    }
    const float s = page_scale(old, block_max(a, sh));
    if (s > old && old > 0.f) recode_rows(codes, t.row0 * P.d, __fdiv_rn(old, s));
    const float inv = s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
    for (int e = threadIdx.x; e < total; e += blockDim.x)
        codes[t.row0 * P.d + e] = code8(to_f32(x[(e / P.d) * A.row_stride[side] + e % P.d]), inv);
    if (threadIdx.x == 0) *scale = s;          // every thread has read the old one before block_max's barrier
}

constexpr int PW_THREADS = 128;

template <typename T>
__device__ __forceinline__ float2 pair_f32(uint32_t w);
template <>
__device__ __forceinline__ float2 pair_f32<__half>(uint32_t w) { return unpack_half2(w); }
template <>
__device__ __forceinline__ float2 pair_f32<__nv_bfloat16>(uint32_t w) {
    return float2{__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
}

// 16-bit rows on 16-byte strides: a thread holds 8 values of up to ROUNDS rounds in registers, so the rows are read
// once.  The maximum is taken on the magnitudes' bits, two a word (they order like the values), which also shows whether
// a value is not finite; without one, rint(x inv) + 128 is the low byte of x inv + (1.5 2^23 + 128), as |x inv| <= 127 up to
// the roundings of s and 1 / s.  Bound by the bytes; many small blocks keep enough loads in flight (blocks of 256: 42.6 us
// below), and rows read with the streaming hint leave the codes in the L2 (38.0 without).  16384 tokens, 8 heads,
// d 128 (67 MB read, 34 MB written), and read back: 36.7 us, 5.5 TB/s.
template <typename T, int ROUNDS>
__global__ void __launch_bounds__(PW_THREADS) page_write_kernel(const __grid_constant__ PageRowsParams A) {
    chain_kernels();
    __shared__ uint32_t sh[PW_THREADS / 32];
    const PagesView& P = A.P;
    const int h = blockIdx.y, side = blockIdx.z;
    const Touch t = find_touch(P, A.slots, A.start, A.cu, A.n, A.rows, blockIdx.x);
    if (t.slot < 0) return;
    // threads of a row, rows of a round
    const int shift = P.d == 128 ? 4 : 3, r0 = threadIdx.x >> shift, step = PW_THREADS >> shift;
    const int c = (threadIdx.x & ((1 << shift) - 1)) * 8;
    const T* x = static_cast<const T*>(A.x[side]) + t.token0 * A.row_stride[side] + h * A.head_stride[side] + c;
    uint4 raw[ROUNDS];
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        const int r = r0 + i * step;
        raw[i] = r < t.rows ? __ldcs(reinterpret_cast<const uint4*>(x + r * A.row_stride[side])) : uint4{0, 0, 0, 0};
    }
    const int64_t page = touch_page(P, t);
    if (page < 0) return;
    if (P.refs[page] > 1) {                    // a page that several sequences hold is not written
        if (threadIdx.x == 0) raise_status(KVB_DEV_BOUNDS);
        return;
    }
    uint8_t* codes = (side ? P.vc : P.kc) + (page * P.Hkv + h) * int64_t(P.page) * P.d;
    float* scale = (side ? P.vs : P.ks) + page * P.Hkv + h;
    const float old = t.row0 > 0 ? *scale : 0.f;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        top = __vmaxu2(top, raw[i].x & 0x7fff7fffu);
        top = __vmaxu2(top, raw[i].y & 0x7fff7fffu);
        top = __vmaxu2(top, raw[i].z & 0x7fff7fffu);
        top = __vmaxu2(top, raw[i].w & 0x7fff7fffu);
    }
    auto block_top = [&](uint32_t v) {
        v = __reduce_max_sync(0xffffffffu, max(v & 0xffffu, v >> 16));
        if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
        __syncthreads();
        uint32_t m = sh[0];
#pragma unroll
        for (int w = 1; w < PW_THREADS / 32; ++w) m = max(m, sh[w]);
        return m;
    };
    constexpr uint32_t INF_BITS = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    uint32_t m = block_top(top);
    const bool finite = m < INF_BITS;
    if (!finite) {                             // the largest of the finite ones
        top = 0;
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i) {
            const uint32_t ws[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t lo = ws[k] & 0x7fffu, hi = (ws[k] >> 16) & 0x7fffu;
                top = max(top, max(lo < INF_BITS ? lo : 0u, hi < INF_BITS ? hi : 0u));
            }
        }
        __syncthreads();
        m = block_top(top);
    }
    const float s = page_scale(old, pair_f32<T>(m).x);
    if (s > old && old > 0.f) recode_rows(codes, t.row0 * P.d, __fdiv_rn(old, s));
    const float inv = s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        const int r = r0 + i * step;
        if (r >= t.rows) break;
        const uint32_t ws[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        uint32_t out[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float2 a = pair_f32<T>(ws[2 * k]), b = pair_f32<T>(ws[2 * k + 1]);
            if (finite) {
                constexpr float MAGIC = 12582912.f + 128.f;
                const uint32_t u0 = __float_as_uint(__fadd_rn(__fmul_rn(a.x, inv), MAGIC)), u1 = __float_as_uint(__fadd_rn(__fmul_rn(a.y, inv), MAGIC));
                const uint32_t u2 = __float_as_uint(__fadd_rn(__fmul_rn(b.x, inv), MAGIC)), u3 = __float_as_uint(__fadd_rn(__fmul_rn(b.y, inv), MAGIC));
                out[k] = __byte_perm(__byte_perm(u0, u1, 0x0040), __byte_perm(u2, u3, 0x0040), 0x5410);
            } else {
                out[k] = code8(a.x, inv) | uint32_t(code8(a.y, inv)) << 8 | uint32_t(code8(b.x, inv)) << 16 | uint32_t(code8(b.y, inv)) << 24;
            }
        }
        *reinterpret_cast<uint2*>(codes + (t.row0 + r) * P.d + c) = uint2{out[0], out[1]};
    }
    if (threadIdx.x == 0) *scale = s;          // every thread has read the old one before block_top's barrier
}

// The codes of a touched page (both sides, all heads) in shares of 8192, one to a block: a thread takes 16 codes in each of
// 4 rounds, its loads in flight together.  A byte b becomes the float32 pattern 0x4b000000 | b = 2^23 + b, less 2^23 +
// 128: exact.  Bound by the bytes; a block per head and side took 47 us where pages are small (16 x 64, 20600 rows of 4
// heads), 14 with stores of 16 bytes, these 11.  grid (touch slots, ceil(2 Hkv page d / 8192))
constexpr int PR_SHARE = 8192;

template <typename T>
__global__ void __launch_bounds__(PW_THREADS) page_read_kernel(const __grid_constant__ PageRowsParams A) {
    chain_kernels();
    const PagesView& P = A.P;
    const Touch t = find_touch(P, A.slots, A.start, A.cu, A.n, A.rows, blockIdx.x);
    if (t.slot < 0) return;
    const int64_t page = touch_page(P, t);
    if (page < 0) return;
    const int log_d = P.d == 128 ? 7 : 6, log_block = log_d + 31 - __clz(P.page);
    constexpr int ROUNDS = PR_SHARE / (16 * PW_THREADS);
    uint4 w[ROUNDS];
    float s[ROUNDS];
    T* to[ROUNDS];
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        const int e = blockIdx.y * PR_SHARE + (i * PW_THREADS + threadIdx.x) * 16, hs = e >> log_block;
        const int side = hs >= P.Hkv, h = hs - side * P.Hkv, in = e & ((1 << log_block) - 1), r = (in >> log_d) - t.row0;
        to[i] = nullptr;
        if (hs >= 2 * P.Hkv || r < 0 || r >= t.rows) continue;
        const int64_t ph = page * P.Hkv + h;
        w[i] = *reinterpret_cast<const uint4*>((side ? P.vc : P.kc) + (ph << log_block) + in);
        s[i] = (side ? P.vs : P.ks)[ph];
        to[i] = static_cast<T*>(A.out[side]) + ((t.token0 + r) * P.Hkv + h) * P.d + (in & (P.d - 1));
    }
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        if (!to[i]) continue;
        const uint32_t ws[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
        float f[16];
#pragma unroll
        for (int k = 0; k < 16; ++k)
            f[k] = (__uint_as_float(__byte_perm(ws[k >> 2], 0x4b000000u, 0x7440 | (k & 3))) - 8388736.f) * s[i];
        alignas(16) T o[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) o[k] = from_f32<T>(f[k]);
        const uint32_t* u = reinterpret_cast<const uint32_t*>(o);
        constexpr int WORDS = sizeof(T) * 4;
        if (A.whole) {
#pragma unroll
            for (int k = 0; k < WORDS; k += 8)
                asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(u[k]), "r"(u[k + 1]), "r"(u[k + 2]), "r"(u[k + 3]),
                             "r"(u[k + 4]), "r"(u[k + 5]), "r"(u[k + 6]), "r"(u[k + 7]), "l"(reinterpret_cast<uint32_t*>(to[i]) + k)
                             : "memory");
        } else {
#pragma unroll
            for (int k = 0; k < WORDS; k += 4) reinterpret_cast<uint4*>(to[i])[k / 4] = uint4{u[k], u[k + 1], u[k + 2], u[k + 3]};
        }
    }
}

// ------------------------------------------------------------------------------------------------
// Page tables.  One block of 1024 threads plans (which pages are free, who gets which), blocks of the
// following launch move the data.
// ------------------------------------------------------------------------------------------------
constexpr int PG_THREADS = 1024;               // at most; a block of 32 threads per 1024 pages where that is less (page_block)
// pages whose state the planning block holds in registers
__device__ __forceinline__ int page_tile() { return int(blockDim.x) * 32; }

// Exclusive scan of one int per thread of the block; total in `sum`.
__device__ __forceinline__ int block_scan(int v, int* sh, int& sum) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) sh[w] = x;
    __syncthreads();
    int t = lane < int(blockDim.x >> 5) ? sh[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, t, o);
        if (lane >= o) t += y;
    }
    sum = __shfl_sync(0xffffffffu, t, 31);
    const int before = w ? __shfl_sync(0xffffffffu, t, w - 1) : 0;
    return before + x - v;
}

// Bit mask over the 32 pages tile0 + 1024 warp + 32 lane + 0..31: set where the page is free.  The loads are
// coalesced (each covers 32 consecutive pages of the warp's 1024) and all in flight together.
__device__ __forceinline__ uint32_t free_mask(const int32_t* refs, int64_t n_pages, int64_t tile0) {
    const int lane = threadIdx.x & 31;
    const int64_t base = tile0 + (threadIdx.x >> 5) * 1024;
    int r[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const int64_t p = base + i * 32 + lane;
        r[i] = p < n_pages ? refs[p] : -1;
    }
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const uint32_t m = __ballot_sync(0xffffffffu, r[i] == 0);
        if (lane == i) mine = m;
    }
    return mine;
}

// The `total` lowest free pages, in ascending order, to give(rank, page), every thread a rank (a lane's 32 pages may all
// be free and then hold consecutive ranks: they are listed in shared memory first, PG_LIST at a time).  False, and
// nothing given, when the pool has fewer.  Whole block; ends with a barrier.
constexpr int PG_LIST = 4096;

template <typename F>
__device__ __forceinline__ bool take_free(const PagesView& P, int total, int* sh, int* list, F give) {
    if (total == 0) return true;
    int found = 0, sum = 0, at = 0;
    uint32_t mask = 0;
    int64_t tile = -1;                         // whose mask and ranks are held
    for (int64_t t0 = 0; t0 < P.n_pages && found < total; t0 += page_tile()) {
        mask = free_mask(P.refs, P.n_pages, t0);
        at = block_scan(__popc(mask), sh, sum);
        tile = t0;
        found += sum;
    }
    if (found < total) return false;
    int before = 0;
    for (int64_t t0 = 0; t0 < P.n_pages && before < total; t0 += page_tile()) {
        if (tile != t0) {                      // a pool of one tile is read once
            mask = free_mask(P.refs, P.n_pages, t0);
            at = block_scan(__popc(mask), sh, sum);
            tile = t0;
        }
        const int64_t base = t0 + (threadIdx.x >> 5) * 1024 + (threadIdx.x & 31) * 32;
        const int take = min(sum, total - before);
        for (int w0 = 0; w0 < take; w0 += PG_LIST) {
            int rank = at - w0;
            for (uint32_t m = mask; m && rank < min(take - w0, PG_LIST); m &= m - 1, ++rank)
                if (rank >= 0) list[rank] = int(base + __ffs(m) - 1);
            __syncthreads();
            for (int r = threadIdx.x; r < min(take - w0, PG_LIST); r += blockDim.x) give(before + w0 + r, list[r]);
            __syncthreads();
        }
        before += sum;
    }
    return true;
}

// largest i with off[i] <= r (off ascending, off[0] = 0)
__device__ __forceinline__ int owner_of(const int* off, int n, int r) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (off[mid] <= r) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Whether a length is one that its row of the table can hold: the pool works on the caller's lengths.
__device__ __forceinline__ bool fits_row(const PagesView& P, int64_t len) { return len >= 0 && len <= int64_t(P.max_blocks) * P.page; }

// One block.  start[i] = the tokens that sequence slots[i] had, or -1 where the call was refused (a slot out of
// range, a length that does not fit, a row too short, not enough free pages): then nothing is changed.
__global__ void __launch_bounds__(PG_THREADS) page_extend_kernel(PagesView P, const int32_t* slots, const int32_t* add, int n,
                                                                 int32_t* start) {
    chain_kernels();
    extern __shared__ int off[];               // off[i]: pages of the sequences before i
    __shared__ int sh[32], list[PG_LIST];
    __shared__ int bad;
    __shared__ unsigned long long want;        // all pages that are needed: the sums below may pass 32 bits
    if (threadIdx.x == 0) bad = 0, want = 0;
    __syncthreads();
    int total = 0;
    for (int i0 = 0; i0 < n; i0 += blockDim.x) {
        const int i = i0 + threadIdx.x;
        int need = 0;
        if (i < n) {
            const int s = slots[i], a = add[i];
            const int have = s >= 0 && s < P.n_slots ? P.lens[s] : 0;
            if (s < 0 || s >= P.n_slots || a < 0 || !fits_row(P, have) || !fits_row(P, int64_t(have) + a)) bad = 1;
            else need = blocks_of(have + a, P.page) - blocks_of(have, P.page);
        }
        // in two halves, whose sums fit a warp's reduction (64-bit additions of all threads: 0.8 us more)
        const unsigned lo = __reduce_add_sync(0xffffffffu, unsigned(need) & 0xffffu), hi = __reduce_add_sync(0xffffffffu, unsigned(need) >> 16);
        if ((threadIdx.x & 31) == 0 && (lo | hi)) atomicAdd(&want, lo + (static_cast<unsigned long long>(hi) << 16));
        int sum;
        const int at = block_scan(need, sh, sum);
        if (i < n) off[i] = total + at;
        total += sum;
    }
    __syncthreads();
    if (bad) {
        if (threadIdx.x == 0) raise_status(KVB_DEV_BOUNDS);
    } else if (want > static_cast<unsigned long long>(P.n_pages) || !take_free(P, total, sh, list, [&](int rank, int id) {
                   const int i = owner_of(off, n, rank);
                   const int s = slots[i];
                   P.table[int64_t(s) * P.max_blocks + blocks_of(P.lens[s], P.page) + rank - off[i]] = id;
                   P.refs[id] = 1;
               })) {
        if (threadIdx.x == 0) { raise_status(KVB_DEV_POOL); bad = 1; }
    }
    __syncthreads();                           // the lengths were read by every thread's give()
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        start[i] = bad ? -1 : P.lens[slots[i]];
        if (!bad) P.lens[slots[i]] += add[i];
    }
}

// One block per sequence.
__global__ void page_free_kernel(PagesView P, const int32_t* slots) {
    chain_kernels();
    __shared__ int len;
    const int s = slots[blockIdx.x];
    if (s < 0 || s >= P.n_slots) {
        if (threadIdx.x == 0) raise_status(KVB_DEV_BOUNDS);
        return;
    }
    if (threadIdx.x == 0) len = atomicExch(&P.lens[s], 0);          // a slot named twice is freed once
    __syncthreads();
    int32_t* row = P.table + int64_t(s) * P.max_blocks;
    for (int b = threadIdx.x; b < min(blocks_of(len, P.page), P.max_blocks); b += blockDim.x) {
        const int id = row[b];
        if (id >= 0 && id < P.n_pages) atomicSub(&P.refs[id], 1);
        row[b] = -1;
    }
}

constexpr int PG_COPY_THREADS = 256;

// Part `part` of `parts` of one page's codes (and, part 0, its scales); whole block of PG_COPY_THREADS, 4 loads in flight.
__device__ __forceinline__ void copy_page(const PagesView& P, int64_t from, int64_t to, int part, int parts) {
    const int side16 = P.Hkv * P.page * P.d / 16, all16 = 2 * side16;        // 16-byte words: keys, then values
    const uint4* k0 = reinterpret_cast<const uint4*>(P.kc) + from * side16;
    const uint4* v0 = reinterpret_cast<const uint4*>(P.vc) + from * side16 - side16;
    uint4* k1 = reinterpret_cast<uint4*>(P.kc) + to * side16;
    uint4* v1 = reinterpret_cast<uint4*>(P.vc) + to * side16 - side16;
    const int per = (all16 + parts - 1) / parts, end = min(all16, per * (part + 1));
    for (int i0 = per * part + threadIdx.x; i0 < end; i0 += 4 * PG_COPY_THREADS) {
        uint4 w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = i0 + k * PG_COPY_THREADS;
            if (i < end) w[k] = __ldcg((i < side16 ? k0 : v0) + i);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = i0 + k * PG_COPY_THREADS;
            if (i < end) __stcg((i < side16 ? k1 : v1) + i, w[k]);
        }
    }
    if (part == 0)
        for (int h = threadIdx.x; h < P.Hkv; h += PG_COPY_THREADS) {
            P.ks[to * P.Hkv + h] = P.ks[from * P.Hkv + h];
            P.vs[to * P.Hkv + h] = P.vs[from * P.Hkv + h];
        }
}

// grid (pages, parts)
__global__ void page_copy_kernel(PagesView P, const int32_t* src, const int32_t* dst) {
    chain_kernels();
    const int a = src[blockIdx.x], b = dst[blockIdx.x];
    if (a < 0 || b < 0 || a >= P.n_pages || b >= P.n_pages) {
        if (threadIdx.x == 0) raise_status(KVB_DEV_BOUNDS);
        return;
    }
    if (a != b) copy_page(P, a, b, blockIdx.y, gridDim.y);
}

// Workspace of a fork: [ok, pad, ...] then per fork: length, fresh page (or -1); then the source rows.
struct ForkWork {
    int32_t* head;      // [0]: 1 when the call goes ahead
    int32_t* len;       // (n)
    int32_t* fresh;     // (n)
    int32_t* rows;      // (n, max_blocks)
};

// One block: lengths and fresh pages of all forks, from the state before any of them.
__global__ void __launch_bounds__(PG_THREADS) fork_plan_kernel(PagesView P, const int32_t* src, const int32_t* dst, int n,
                                                               ForkWork W) {
    chain_kernels();
    extern __shared__ int off[];
    __shared__ int sh[32], list[PG_LIST];
    __shared__ int bad;
    if (threadIdx.x == 0) bad = 0;
    __syncthreads();
    int total = 0;
    for (int i0 = 0; i0 < n; i0 += blockDim.x) {
        const int i = i0 + threadIdx.x;
        int part = 0;
        if (i < n) {
            const int s = src[i], t = dst[i];
            if (s < 0 || s >= P.n_slots || t < 0 || t >= P.n_slots || !fits_row(P, P.lens[s]) || !fits_row(P, P.lens[t])) bad = 1;
            else {
                const int len = P.lens[s];
                W.len[i] = len;
                part = s != t && (len & (P.page - 1)) != 0;
            }
            W.fresh[i] = -1;
        }
        int sum;
        const int at = block_scan(part, sh, sum);
        if (i < n) off[i] = total + at;
        total += sum;
    }
    if (threadIdx.x == 0) off[n] = total;
    __syncthreads();
    // rank r belongs to the last i with off[i] <= r: that i has a partial page, those sharing its offset before it none
    if (bad) {
        if (threadIdx.x == 0) raise_status(KVB_DEV_BOUNDS);
    } else if (!take_free(P, total, sh, list, [&](int rank, int id) { W.fresh[owner_of(off, n, rank)] = id; })) {
        if (threadIdx.x == 0) { raise_status(KVB_DEV_POOL); bad = 1; }
    }
    __syncthreads();
    if (threadIdx.x == 0) W.head[0] = !bad;
}

// grid (forks, 1 + parts): part 0 snapshots the source's row, the others copy its partial page
__global__ void fork_copy_kernel(PagesView P, const int32_t* src, ForkWork W) {
    chain_kernels();
    if (!W.head[0]) return;
    const int i = blockIdx.x;
    const int32_t* row = P.table + int64_t(src[i]) * P.max_blocks;
    const int nb = blocks_of(W.len[i], P.page), fresh = W.fresh[i];
    if (blockIdx.y == 0) {
        for (int b = threadIdx.x; b < nb; b += blockDim.x)
            W.rows[int64_t(i) * P.max_blocks + b] = b == nb - 1 && fresh >= 0 ? fresh : row[b];
    } else if (fresh >= 0) {
        const int from = row[nb - 1];
        if (from >= 0 && from < P.n_pages) copy_page(P, from, fresh, blockIdx.y - 1, gridDim.y - 1);
    }
}

// grid (forks): references and rows
__global__ void fork_commit_kernel(PagesView P, const int32_t* src, const int32_t* dst, ForkWork W) {
    chain_kernels();
    if (!W.head[0]) return;
    const int i = blockIdx.x, t = dst[i];
    if (src[i] == t) return;
    __shared__ int old;
    if (threadIdx.x == 0) old = P.lens[t];
    __syncthreads();
    int32_t* row = P.table + int64_t(t) * P.max_blocks;
    const int nb = blocks_of(W.len[i], P.page), ob = blocks_of(old, P.page);
    for (int b = threadIdx.x; b < max(nb, ob); b += blockDim.x) {
        if (b < ob && row[b] >= 0 && row[b] < P.n_pages) atomicSub(&P.refs[row[b]], 1);
        const int id = b < nb ? W.rows[int64_t(i) * P.max_blocks + b] : -1;
        if (id >= 0 && id < P.n_pages) atomicAdd(&P.refs[id], 1);
        row[b] = id;
    }
    if (threadIdx.x == 0) P.lens[t] = W.len[i];
}

// Workspace of a compaction: [n_live, moves], then move r: from[r] -> to[r], and new_id (by old page)
struct CompactWork {
    int32_t* head;
    int32_t* from;
    int32_t* to;
    int32_t* new_id;
};

// One block.  A pool of one tile is read once.
__global__ void __launch_bounds__(PG_THREADS) compact_plan_kernel(PagesView P, CompactWork W) {
    chain_kernels();
    __shared__ int sh[32], hole_list[PG_LIST], mover_list[PG_LIST];
    int live = 0, sum;
    uint32_t m = 0;
    for (int64_t t0 = 0; t0 < P.n_pages; t0 += page_tile()) {
        m = free_mask(P.refs, P.n_pages, t0);
        block_scan(__popc(m), sh, sum);
        live += int(imin64(page_tile(), P.n_pages - t0)) - sum;
    }
    // holes and movers in ascending order: as many of the one as of the other.  Where they fit they are listed in shared
    // memory and written out together.
    int holes = 0, movers = 0;
    const bool one = P.n_pages <= page_tile();
    for (int64_t t0 = 0; t0 < P.n_pages; t0 += page_tile()) {
        if (!one) m = free_mask(P.refs, P.n_pages, t0);
        const int64_t base = t0 + (threadIdx.x >> 5) * 1024 + (threadIdx.x & 31) * 32;
        const int64_t below = imin64(imax64(live - base, 0), 32), valid = imin64(imax64(P.n_pages - base, 0), 32);
        const uint32_t lo = below == 32 ? 0xffffffffu : (1u << below) - 1, in = valid == 32 ? 0xffffffffu : (1u << valid) - 1;
        uint32_t hole = m & lo, mover = ~m & in & ~lo;
        int both;                                                // two counts of at most 2^15 in one scan
        const int at = block_scan(__popc(hole) | __popc(mover) << 16, sh, both);
        const int nh = both & 0xffff, nm = int(uint32_t(both) >> 16);
        int rh = at & 0xffff, rm = int(uint32_t(at) >> 16);
        for (; hole; hole &= hole - 1, ++rh) {
            const int id = int(base + __ffs(hole) - 1);
            if (rh < PG_LIST) hole_list[rh] = id;
            else W.to[holes + rh] = id;
        }
        for (; mover; mover &= mover - 1, ++rm) {
            const int id = int(base + __ffs(mover) - 1);
            if (rm < PG_LIST) mover_list[rm] = id;
            else W.from[movers + rm] = id;
        }
        __syncthreads();
        for (int r = threadIdx.x; r < min(nh, PG_LIST); r += blockDim.x) W.to[holes + r] = hole_list[r];
        for (int r = threadIdx.x; r < min(nm, PG_LIST); r += blockDim.x) W.from[movers + r] = mover_list[r];
        if (one)
            for (int r = threadIdx.x; r < min(nm, PG_LIST); r += blockDim.x) W.new_id[mover_list[r]] = hole_list[r];
        holes += nh;
        movers += nm;
        __syncthreads();
    }
    for (int r = (one ? PG_LIST : 0) + threadIdx.x; r < movers; r += blockDim.x) W.new_id[W.from[r]] = W.to[r];
    if (threadIdx.x == 0) {
        W.head[0] = live;
        W.head[1] = movers;
    }
}

// The moves of one pool, eighths of pages to many blocks: freeing, compacting (375 pages of 131 KB) and extending takes 38.5
// us with 16 blocks an SM and 4 loads of a thread in flight, 43.8 with quarters, 4 blocks and 8 loads.  With `commit` also the reference counts and the table (once, where pools share them).
__global__ void compact_move_kernel(PagesView P, CompactWork W, int32_t* n_live, int commit) {
    chain_kernels();
    const int live = W.head[0], moves = W.head[1];
    constexpr int PARTS = 8;
    for (int w = blockIdx.x; w < moves * PARTS; w += gridDim.x) {
        const int r = w / PARTS;
        copy_page(P, W.from[r], W.to[r], w % PARTS, PARTS);
        if (commit && w % PARTS == 0 && threadIdx.x == 0) {
            P.refs[W.to[r]] = P.refs[W.from[r]];
            P.refs[W.from[r]] = 0;
        }
    }
    if (!commit) return;
    if (blockIdx.x == 0 && threadIdx.x == 0) *n_live = live;
    const int64_t entries = int64_t(P.n_slots) * P.max_blocks;
    for (int64_t e = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; e < entries; e += int64_t(gridDim.x) * blockDim.x) {
        const int id = P.table[e];
        if (id >= live && id < P.n_pages) P.table[e] = W.new_id[id];
    }
}

}  // namespace kvb
