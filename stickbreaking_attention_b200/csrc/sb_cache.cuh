// What the kernels of the 8-bit paged cache share: argument checks, the layout of a page, e4m3 codes.
#pragma once

#include <cuda_fp8.h>

#include "sb_common.cuh"

namespace sb {

inline int cache_row(int head_dim) { return head_dim <= 32 ? 32 : head_dim <= 64 ? 64 : 128; }
inline bool page_size_ok(int n) { return n == 16 || n == 32 || n == 64 || n == 128; }

// e4m3: the largest value, and the smallest exponent of a scale (2^-118 and its reciprocal are normal float32 numbers, so are the
// largest, 2^120 for values up to 2^128, and its own)
constexpr int kScaleMinExp = -118;

// The smallest power of two s with a <= 448 s, at least 2^-118, for a finite a >= 0: 448 = 1.75 * 2^8.
__device__ inline float scale_for(float a) {
    const uint32_t bits = __float_as_uint(a);
    int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = max(e, kScaleMinExp);
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// the code of a float32 number that is at most 448 in magnitude; NaN code for infinities and NaN
__device__ inline uint8_t to_e4m3(float x) {
    const uint8_t c = (uint8_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
    return fabsf(x) <= 3.4028234664e38f ? c : (uint8_t)0x7f;
}
__device__ inline float from_e4m3(uint8_t c) { return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3))); }

int launch_cache_blocks(const SbBlocksParams& p, cudaStream_t st);
int launch_cache_append(const SbCacheParams& p, cudaStream_t st);
size_t cached_workspace(const SbCacheParams& p);
size_t cached_tc_workspace(const SbCacheParams& p);
int launch_cached_tc(const SbCacheParams& p, cudaStream_t st);
int launch_cached_fwd(const SbCacheParams& p, cudaStream_t st);

}  // namespace sb
