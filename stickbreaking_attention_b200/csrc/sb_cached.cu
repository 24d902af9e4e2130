// Stick-breaking attention of new tokens over the 8-bit paged cache.
#include "sb_cache.cuh"

namespace sb {

namespace {

constexpr int kWarps = 4;

// One warp per query row and head, 32 keys at a time from the right: a lane forms the score of one key, the suffix sums of log(1 - beta) go
// over the lanes, and the weighted sum of the values is shared out by columns of D.
template <typename T>
__global__ void __launch_bounds__(32 * kWarps) cached_kernel(const SbCacheParams p) {
    __shared__ float qs[kWarps][kMaxHeadDim], ws[kWarps][32];
    __shared__ const uint8_t* vs[kWarps][32];
    pdl_wait();
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = blockIdx.y, t = blockIdx.x * kWarps + warp;
    if (p.ends && blockIdx.x == 0 && blockIdx.y == 0)
        for (int s = threadIdx.x; s < p.requests; s += 32 * kWarps)
            if (p.ends[s] < (s > 0 ? p.ends[s - 1] : 0) || p.ends[s] > p.tokens) atomicOr(p.status, SBATTN_ST_BAD_SEQLENS);
    if (t >= p.tokens) return;
    const int D = p.head_dim, P = p.page_tokens, g = h / (p.heads / p.kv_heads);
    int r = t, n = 1, i = 0;
    if (p.ends) {
        int lo = 0, hi = p.requests;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (p.ends[mid] > t) hi = mid; else lo = mid + 1;
        }
        r = lo;
        if (r < p.requests) {
            const int first = r > 0 ? p.ends[r - 1] : 0;
            n = p.ends[r] - first;
            i = t - first;
        }
    }
    T* rem = (T*)p.rem.ptr + h * p.rem.stride_h + t * p.rem.stride_t;
    const int len = r < p.requests ? p.lengths[r] : 0;
    if (r >= p.requests || (!p.ends && len == 0)) {
        if (lane == 0) *rem = from_f32<T>(0.f);
        return;
    }
    if (i < 0 || len < n || len > (int64_t)p.width * P) {
        if (lane == 0) {
            *rem = from_f32<T>(0.f);
            atomicOr(p.status, SBATTN_ST_BAD_SEQLENS);
        }
        return;
    }
    const T* q = (const T*)p.q.ptr + h * p.q.stride_h + t * p.q.stride_t;
    for (int d = lane; d < D; d += 32) qs[warp][d] = to_f32(q[d]);
    const int keys = len - n + i + (p.attend_current ? 1 : 0);
    float acc[4] = {0.f, 0.f, 0.f, 0.f}, right = 0.f;
    for (int hi = keys; hi > 0; hi -= 32) {
        const int j = hi - 1 - lane;
        float x = 0.f, soft = 0.f, weight = 0.f;
        const uint8_t* vp = nullptr;
        __syncwarp();
        if (j >= 0) {
            int page = p.tables[r * p.table_stride + j / P];
            if (page < 0 || page >= p.pages) {
                atomicOr(p.status, SBATTN_ST_BAD_PAGES);
                page = 0;
            }
            const int64_t at = ((int64_t)g * P + j % P) * p.row;
            const uint8_t* kp = (const uint8_t*)p.k_codes + page * p.k_stride + at;
            vp = (const uint8_t*)p.v_codes + page * p.v_stride + at;
            for (int d = 0; d < D; ++d) x = fmaf(qs[warp][d], from_e4m3(kp[d]), x);
            x *= p.k_scale[page * p.k_scale_stride + g] * p.inv_temp;
            soft = fmaxf(x, 0.f) + log1pf(expf(-fabsf(x)));
            if (x != x) soft = x;
            weight = p.v_scale[page * p.v_scale_stride + g];
        }
        float sum = soft;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const float y = __shfl_up_sync(0xffffffffu, sum, off);
            if (lane >= off) sum += y;
        }
        const float before = __shfl_up_sync(0xffffffffu, sum, 1);  // the keys to the right of this one
        weight *= expf(-(right + (lane > 0 ? before : 0.f))) / (1.f + expf(-x));
        ws[warp][lane] = weight;
        vs[warp][lane] = vp;
        right += __shfl_sync(0xffffffffu, sum, 31);
        __syncwarp();
        for (int l = 0; l < 32 && l < hi; ++l) {
            const float w = ws[warp][l];
            for (int c = 0; c < 4; ++c)
                if (lane + 32 * c < D) acc[c] = fmaf(w, from_e4m3(vs[warp][l][lane + 32 * c]), acc[c]);
        }
    }
    const T left = from_f32<T>(expf(-right));
    T* o = (T*)p.o.ptr + h * p.o.stride_h + t * p.o.stride_t;
    const T* v = p.v.ptr ? (const T*)p.v.ptr + g * p.v.stride_h + t * p.v.stride_t : nullptr;
    for (int c = 0; c < 4; ++c)
        if (const int d = lane + 32 * c; d < D) o[d] = from_f32<T>(v ? fmaf(to_f32(left), to_f32(v[d]), acc[c]) : acc[c]);
    if (lane == 0) *rem = left;
}

template <typename T>
int launch(const SbCacheParams& p, cudaStream_t st) {
    const dim3 grid((unsigned)((p.tokens + kWarps - 1) / kWarps), (unsigned)p.heads);
    return launch_kernel(cached_kernel<T>, grid, dim3(32 * kWarps), 0, st, p);
}

}  // namespace

size_t cached_workspace(const SbCacheParams&) { return 0; }

int launch_cached_fwd(const SbCacheParams& p, cudaStream_t st) {
    if (p.dtype == SBATTN_F32) return launch<float>(p, st);
    if (p.dtype == SBATTN_F16) return launch<__half>(p, st);
    return launch<__nv_bfloat16>(p, st);
}

}  // namespace sb
