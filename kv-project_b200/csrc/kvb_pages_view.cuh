// kvb_pages_view.cuh - the 8-bit paged cache as kernels see it, and the rounding to an output type.
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

__device__ __forceinline__ int blocks_of(int n, int page) { return (n + page - 1) / page; }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

}  // namespace kvb
