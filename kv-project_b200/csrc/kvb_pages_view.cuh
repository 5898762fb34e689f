// kvb_pages_view.cuh - the 8-bit paged cache as kernels see it, and the rounding to 16-bit types.
#pragma once

#include "kvb_common.cuh"

namespace kvb {

// kvb_pages of include/kvb.h
struct PagesView {
    uint8_t* kc;
    uint8_t* vc;
    float* ks;
    float* vs;
    int32_t* table;
    int32_t* lens;
    int32_t* refs;
    int64_t n_pages;
    int Hkv, d, page, n_slots, max_blocks;
};

// pages are 16, 32, 64 or 128 tokens: a shift instead of the 20 and more instructions of a division
__device__ __forceinline__ int page_shift(int page) { return 31 - __clz(page); }
__device__ __forceinline__ int blocks_of(int n, int page) { return (n + page - 1) >> page_shift(page); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// two values of a 16-bit type in a word, the first in its low half
template <typename T>
__device__ __forceinline__ uint32_t pack_f32(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack_f32<__half>(float lo, float hi) { return pack_half2(lo, hi); }
template <>
__device__ __forceinline__ uint32_t pack_f32<__nv_bfloat16>(float lo, float hi) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
}

}  // namespace kvb
