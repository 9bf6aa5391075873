// Shared pieces of the 8-bit KV cache kernels: e4m3 codes with one power-of-two scale per (block of slots, plane, head).
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace tidal {

// A scale byte b stands for 2^(b-127): the exponent field of that float (b = 0 gives +0, so the block reads as zeros).
__device__ __forceinline__ float scale_value(uint32_t byte) { return __uint_as_float(byte << 23); }

// Smallest biased exponent b >= 1 with amax <= 448 * 2^(b-127).  448 = 1.75 * 2^8: the exponent of amax less 8, one more
// when its mantissa lies above 1.75.  amax finite and >= 0.
__device__ __forceinline__ int scale_byte(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int b = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return b < 1 ? 1 : b;
}

// Two floats to e4m3 (nearest, ties to even; |x| > 448 and infinities saturate, NaN stays NaN), the first in the low byte.
__device__ __forceinline__ uint32_t pack_e4m3(float lo, float hi) {
    return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
// ... and back, exactly: every e4m3 value is an fp16 value.
__device__ __forceinline__ float2 unpack_e4m3(uint32_t pair) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)pair, __NV_E4M3);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Where slot `slot` of sequence b lives: its page (-1 when out of range) and, in *entry, its place in the page.
struct SlotMap {
    const int32_t* page_table;
    int64_t pt_stride, num_pages;
    int32_t page_size;
    __device__ __forceinline__ int64_t page_of(int b, int slot, int* entry) const {
        if (slot < 0) return -1;
        const int pg = page_size == 1 ? slot : slot / page_size;
        *entry = slot - pg * page_size;
        const int64_t page = page_table ? (int64_t)page_table[(size_t)b * pt_stride + pg] : (int64_t)b * pt_stride + pg;
        return page < 0 || page >= num_pages ? -1 : page;
    }
};

}  // namespace tidal
