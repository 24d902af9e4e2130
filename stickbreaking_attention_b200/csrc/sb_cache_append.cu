// New keys and values into the pages of the 8-bit cache.
#include "sb_cache.cuh"

namespace sb {

namespace {

constexpr int kThreads = 256;

__device__ inline float finite_abs(float x) {
    const float a = fabsf(x);
    return a <= 3.4028234664e38f ? a : 0.f;
}

// One block: one piece (the new tokens of one page), one head, keys or values.  Two passes over the new values (the second one finds them in the
// L1): their largest magnitude, which settles the scale, and the codes.
template <typename T>
__global__ void __launch_bounds__(kThreads) append_kernel(const SbCacheParams p) {
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
    float a = 0.f;
    for (int i = threadIdx.x; i < n * row; i += kThreads) {
        const int t = i / row, d = i % row;
        if (d < D) a = fmaxf(a, finite_abs(to_f32(src[(int64_t)t * m.stride_t + d])));
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, off));
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = a;
    __syncthreads();
    for (int w = 0; w < kThreads / 32; ++w) a = fmaxf(a, warp_max[w]);
    float s = scale_for(a);
    if (old > 0) {
        const float had = *scale;
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
    for (int i = threadIdx.x; i < n * row; i += kThreads) {
        const int t = i / row, d = i % row;
        codes[(int64_t)old * row + i] = d < D ? to_e4m3(to_f32(src[(int64_t)t * m.stride_t + d]) / s) : (uint8_t)0;
    }
    __syncthreads();  // every thread has read the old scale
    if (threadIdx.x == 0) *scale = s;
}

template <typename T>
int launch(const SbCacheParams& p, cudaStream_t st) {
    return launch_kernel(append_kernel<T>, dim3((unsigned)(p.n_pieces * p.kv_heads), 2), dim3(kThreads), 0, st, p);
}

}  // namespace

int launch_cache_append(const SbCacheParams& p, cudaStream_t st) {
    if (p.dtype == SBATTN_F32) return launch<float>(p, st);
    if (p.dtype == SBATTN_F16) return launch<__half>(p, st);
    return launch<__nv_bfloat16>(p, st);
}

}  // namespace sb
