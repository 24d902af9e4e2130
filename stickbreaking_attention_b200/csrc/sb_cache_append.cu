// New keys and values into the pages of the 8-bit cache.
//
// Scales are powers of two: x / s and the step from an old scale to a larger one are exact, and the only rounding is e4m3's own, so that results
// do not depend on how often a page was written (but for values that fall below e4m3's normal range on the larger scale).  Bound by memory:
// every new value is read once and one byte written.  A block takes one piece (the new tokens of one page) of one head, keys or values, 8 values a
// thread and load, and keeps them in registers between the two uses, the largest magnitude and the codes; a second pass over global memory, with
// single values, took 279 us where this one takes 36 (32 heads, 8400 tokens, head dim 128, bfloat16: 31 us at the copy's bandwidth).
#include "sb_cache.cuh"

namespace sb {

namespace {

constexpr int kThreads = 256;
constexpr float kMaxFloat = 3.4028234664e38f;

__device__ inline float finite_abs(float x) {
    const float a = fabsf(x);
    return a <= kMaxFloat ? a : 0.f;
}

template <typename T>
struct alignas(16) Eight {
    T x[8];
};

// Largest magnitude of eight values, infinity included, NaN not
__device__ inline float top_of(const Eight<float>& v) {
    float a = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) a = fmaxf(a, fabsf(v.x[e]));
    return a;
}
__device__ inline float top_of(const Eight<__half>& v) {
    const __half2* w = (const __half2*)v.x;
    const __half2 a = __hmax2(__hmax2(__habs2(w[0]), __habs2(w[1])), __hmax2(__habs2(w[2]), __habs2(w[3])));
    return fmaxf(__low2float(a), __high2float(a));
}
__device__ inline float top_of(const Eight<__nv_bfloat16>& v) {
    const __nv_bfloat162* w = (const __nv_bfloat162*)v.x;
    const __nv_bfloat162 a = __hmax2(__hmax2(__habs2(w[0]), __habs2(w[1])), __hmax2(__habs2(w[2]), __habs2(w[3])));
    return fmaxf(__low2float(a), __high2float(a));
}

// C: chunks of eight values a thread has at most.  `whole`: rows may be read eight values at a time.
template <typename T, int C>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ SbCacheParams p, const int whole) {
    __shared__ float warp_max[kThreads / 32];
    pdl_wait();
    pdl_launch_dependents();
    const int head = blockIdx.x % p.kv_heads, piece = blockIdx.x / p.kv_heads;
    const bool values = blockIdx.y != 0;
    const int4 pc = ((const int4*)p.pieces)[piece];
    const int page = pc.x, row0 = pc.y, old = pc.z, n = pc.w, P = p.page_tokens, D = p.head_dim, row = p.row;
    if (page < 0) return;
    if (page >= p.pages || old < 0 || n < 1 || old > P - n || row0 < 0 || row0 > p.tokens - n) {
        if (threadIdx.x == 0) atomicOr(p.status, SBATTN_ST_BAD_PAGES);
        return;
    }
    const SbMat& m = values ? p.v : p.k;
    const T* src = (const T*)m.ptr + head * m.stride_h + (int64_t)row0 * m.stride_t;
    uint8_t* codes = (uint8_t*)(values ? p.v_codes : p.k_codes) + (int64_t)page * (values ? p.v_stride : p.k_stride) + (int64_t)head * P * row;
    float* scale = (values ? p.v_scale : p.k_scale) + (int64_t)page * (values ? p.v_scale_stride : p.k_scale_stride) + head;
    const float had = old > 0 ? *scale : 0.f;
    const int shift = row == 128 ? 4 : row == 64 ? 3 : 2, chunks = n << shift;  // rows of 1 << shift chunks; at most C * kThreads
    Eight<T> x[C];
    float a = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = c * kThreads + threadIdx.x;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[c].x[e] = T(0.f);
        if (i < chunks) {
            const int d = (i & ((1 << shift) - 1)) * 8;
            const T* from = src + (int64_t)(i >> shift) * m.stride_t + d;
            if (whole) {
                if (d < D) x[c] = *(const Eight<T>*)from;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (d + e < D) x[c].x[e] = from[e];
            }
        }
    }
    const auto block_max = [&]() {
        a = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(a)));
        if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = a;
        __syncthreads();  // every thread has read the old scale, too
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) a = fmaxf(a, warp_max[w]);
    };
#pragma unroll
    for (int c = 0; c < C; ++c) a = fmaxf(a, top_of(x[c]));
    block_max();
    const bool infinite = a > kMaxFloat;  // rare: infinities do not count, and are stored as NaN
    if (infinite) {
        a = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) a = fmaxf(a, finite_abs(to_f32(x[c].x[e])));
        __syncthreads();
        block_max();
    }
    float s = scale_for(a);
    if (old > 0) {
        if (had >= s) {
            s = had;
        } else {  // the tokens that are there on the new scale
            const float shrink = had / s;
            for (int i = threadIdx.x; i < old * row; i += kThreads) {
                const uint8_t c = codes[i];
                if ((c & 0x7f) != 0x7f) codes[i] = to_e4m3(from_e4m3(c) * shrink);
            }
        }
    }
    const float inverse = 1.f / s;  // exact
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = c * kThreads + threadIdx.x;
        if (i >= chunks) break;
        uint32_t w[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = to_f32(x[c].x[4 * h + e]) * inverse;
            w[h] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3) |
                   (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3) << 16;
            if (infinite)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (!(fabsf(y[e]) <= kMaxFloat)) w[h] = (w[h] & ~(0xffu << (8 * e))) | (0x7fu << (8 * e));
        }
        *(uint2*)(codes + (int64_t)old * row + (int64_t)i * 8) = make_uint2(w[0], w[1]);
    }
    if (threadIdx.x == 0) *scale = s;
}

template <typename T, int C>
int launch_c(const SbCacheParams& p, bool whole, cudaStream_t st) {
    return launch_kernel(append_kernel<T, C>, dim3((unsigned)(p.n_pieces * p.kv_heads), 2), dim3(kThreads), 0, st, p, whole ? 1 : 0);
}
template <typename T>
int launch(const SbCacheParams& p, cudaStream_t st) {
    const auto aligned = [](const SbMat& m) { return (((uintptr_t)m.ptr | (uintptr_t)(m.stride_h * sizeof(T)) | (uintptr_t)(m.stride_t * sizeof(T))) & 15) == 0; };
    const bool whole = p.head_dim % 8 == 0 && aligned(p.k) && aligned(p.v);
    const int c = (p.page_tokens * p.row + 8 * kThreads - 1) / (8 * kThreads);  // a page's chunks
    return c <= 1 ? launch_c<T, 1>(p, whole, st) : c == 2 ? launch_c<T, 2>(p, whole, st) : c <= 4 ? launch_c<T, 4>(p, whole, st) : launch_c<T, 8>(p, whole, st);
}

}  // namespace

int launch_cache_append(const SbCacheParams& p, cudaStream_t st) {
    if (p.dtype == SBATTN_F32) return launch<float>(p, st);
    if (p.dtype == SBATTN_F16) return launch<__half>(p, st);
    return launch<__nv_bfloat16>(p, st);
}

}  // namespace sb
