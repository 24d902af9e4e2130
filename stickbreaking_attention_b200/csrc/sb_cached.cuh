// What the kernels of attention over the 8-bit paged cache share: the line of work over all requests, key/value heads and tiles of queries, cut
// into equal shares wherever the cuts fall, and the joining of what the cuts have parted.
#pragma once

#include "sb_cache.cuh"

namespace sb {

namespace cached {

struct Job {
    int r, g, tile;      // request, key/value head, tile of columns
    int first, n, len;   // rows of q of the request, tokens
    int raw, take;       // first unit of this share's part of the job, and units
    int pos, end, steps; // steps of keys, counted from the right: [pos, end) of steps
    int cols, keys;      // columns of the tile, keys that its last column sees
    bool starts, ends;   // with its first unit in this share, with its last one
};

// What the host knows of a launch besides the parameters
struct Plan {
    int shared, shift;   // queries' heads per key/value head, and its logarithm if it is a power of two, else -1
    int quads, pairs;    // q may be read four values at a time; o written, and v read, two at a time
    int octets;          // q, o and v eight at a time
    int shares;          // of the work, at most: warps or blocks of the grid
    float* slots;        // [shares][2] partial results: of a job that goes on from the share before, and of one that starts here and goes on
    int4* seams;         // [shares][2]: of the job that a share's first unit goes on with, if it started in the share before: (first row of q or -1, rows,
                         // head, tile), (last share, 0, 0, 0)
};

// floats of a partial result: [column][d], then the sums
__host__ __device__ constexpr int slot_floats(int cols, int dp) { return cols * dp + cols; }

// four codes to two pairs of float16
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127

__device__ __forceinline__ float ex2(float x) {  // 2^x, 2 units of the last place, subnormal results too
    float y;
    asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// a / b of non-negative numbers, in 32 bits where they fit
__device__ __forceinline__ long long quotient(long long a, long long b) {
    return (a | b) >> 32 ? a / b : (long long)((unsigned)a / (unsigned)b);
}

// The line of work: every request's tiles of COLS queries, per key/value head, in steps of STEP keys.  What a job costs besides its steps (its queries, its
// results) counts as COST units ahead of them, so that shares with more jobs have fewer steps.
template <typename T, int DP, int COLS, int STEP, int COST>
struct Jobs {
    const SbCacheParams& p;
    const Plan& pl;
    const int* starts;  // units per head before each request
    int see;

    static __device__ __forceinline__ long long units_of(const Plan& pl, int len, int n, int see) {  // per key/value head
        const int tiles = (n * pl.shared + COLS - 1) / COLS, keys = len - 1 + see;
        return (long long)tiles * (max(1, (keys + STEP - 1) / STEP) + COST);
    }
    // the seam of the job of unit u, which is raw units into it, for the join kernel: this share's if the job started in the share before
    __device__ __forceinline__ void mark(const Job& j, long long u, long long units, long long shares, long long self) const {
        const long long first = u - j.raw, last = first + j.steps + COST;
        if (first < quotient(units * (self - 1), shares)) return;
        pl.seams[2 * self] = make_int4(j.first, j.n, j.g, j.tile);
        pl.seams[2 * self + 1] = make_int4((int)quotient(last * shares - 1, units), 0, 0, 0);  // the share of unit last - 1
    }
    // the last request whose units start at or before u
    __device__ __forceinline__ int find(long long u) const {
        int lo = 0, hi = p.requests;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if ((long long)starts[mid] * p.kv_heads <= u) lo = mid; else hi = mid;
        }
        return lo;
    }
    // the job of unit u, up to unit `stop`; r: a request at or before it
    __device__ __forceinline__ Job open(long long u, long long stop, int r) const {
        Job j;
        while ((long long)starts[r + 1] * p.kv_heads <= u) ++r;
        j.r = r;
        request(r, j.first, j.n, j.len);
        const int tiles = (j.n * pl.shared + COLS - 1) / COLS;
        j.steps = max(1, (j.len - 1 + see + STEP - 1) / STEP);
        const unsigned long long in = (unsigned long long)(u - (long long)starts[r] * p.kv_heads);
        const unsigned cost = (unsigned)j.steps + COST;
        unsigned long long job;
        if (in >> 32) {
            job = in / cost;
            j.raw = (int)(in % cost);
        } else {
            job = (unsigned)in / cost;
            j.raw = (int)((unsigned)in % cost);
        }
        j.g = (int)(job / (unsigned)tiles);
        j.tile = (int)(job % (unsigned)tiles);
        j.take = (int)min((long long)cost - j.raw, stop - u);
        j.pos = max(0, j.raw - COST);
        j.end = max(0, j.raw + j.take - COST);
        j.starts = j.raw == 0;
        j.ends = j.raw + j.take == (int)cost;
        j.cols = min(COLS, j.n * pl.shared - j.tile * COLS);
        j.keys = j.len - j.n + token(j.tile * COLS + j.cols - 1) + see;
        return j;
    }
    __device__ __forceinline__ void request(int r, int& first, int& n, int& len) const {
        len = p.lengths[r];
        if (p.ends) {
            first = r > 0 ? p.ends[r - 1] : 0;
            n = p.ends[r] - first;
        } else {
            first = r;
            n = len > 0 ? 1 : 0;
        }
    }
    // first step, counted from the right, that holds a key which the tile sees
    __device__ __forceinline__ int first_pos(const Job& j) const { return max(j.pos, j.steps - max(1, (j.keys + STEP - 1) / STEP)); }
    // keys that column c of the tile sees
    __device__ __forceinline__ int sees(const Job& j, int c) const { return j.len - j.n + token(j.tile * COLS + c) + see; }
    __device__ __forceinline__ int token(int col) const { return pl.shift >= 0 ? col >> pl.shift : col / pl.shared; }  // of a request, by column

    __device__ __forceinline__ int row_of(const Job& j, int c, int& head) const {
        const int col = j.tile * COLS + c, row = token(col);
        head = j.g * pl.shared + col - row * pl.shared;
        return j.first + row;
    }
    // N results of one column from d0 on, and with `writes_rem` what is left of the stick
    template <int N>
    __device__ __forceinline__ void store(const Job& j, int c, int d0, const float (&x)[N], float sum, bool writes_rem) const {
        int h;
        const int t = row_of(j, c, h);
        const T left = from_f32<T>(ex2(-sum));
        T* o = (T*)p.o.ptr + h * p.o.stride_h + t * p.o.stride_t + d0;
        const T* v = p.v.ptr ? (const T*)p.v.ptr + j.g * p.v.stride_h + t * p.v.stride_t + d0 : nullptr;
        struct alignas(2 * sizeof(T)) Two {
            T a, b;
        };
        struct alignas(sizeof(T) == 2 ? 16 : 32) Eight {
            T a[8];
        };
        if (N % 8 == 0 && sizeof(T) == 2 && pl.octets) {
#pragma unroll
            for (int i = 0; i + 7 < N; i += 8)
                if (d0 + i < p.head_dim) {
                    const float l = to_f32(left);
                    Eight w, y;
                    if (v) w = *(const Eight*)(v + i);
#pragma unroll
                    for (int e = 0; e < 8; ++e) y.a[e] = from_f32<T>(v ? fmaf(l, to_f32(w.a[e]), x[i + e]) : x[i + e]);
                    *(Eight*)(o + i) = y;
                }
        } else if (N > 1 && pl.pairs) {
            Two w[N / 2 + 1];
            if (v)
#pragma unroll
                for (int i = 0; i + 1 < N; i += 2)
                    if (d0 + i < p.head_dim) w[i / 2] = *(const Two*)(v + i);
#pragma unroll
            for (int i = 0; i + 1 < N; i += 2)
                if (d0 + i < p.head_dim) {
                    const float l = to_f32(left);
                    *(Two*)(o + i) = v ? Two{from_f32<T>(fmaf(l, to_f32(w[i / 2].a), x[i])), from_f32<T>(fmaf(l, to_f32(w[i / 2].b), x[i + 1]))}
                                       : Two{from_f32<T>(x[i]), from_f32<T>(x[i + 1])};
                }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (d0 + i < p.head_dim) o[i] = from_f32<T>(v ? fmaf(to_f32(left), to_f32(v[i]), x[i]) : x[i]);
        }
        if (writes_rem) ((T*)p.rem.ptr)[h * p.rem.stride_h + t * p.rem.stride_t] = left;
    }
};


// Where every request's units start (starts[R + 1], per key/value head): a prefix sum over the requests, by every block for itself.  Returns the
// sum; requests that do not fit together are reported and get no units.
template <typename J, int kThreads>
__device__ __forceinline__ long long scan_requests(const SbCacheParams& p, const Plan& pl, int* starts, int see) {
    constexpr int kWarps = kThreads / 32;
    __shared__ long long warp_sums[kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, R = p.requests, P = p.page_tokens;
    long long carry = 0;
    bool bad = false;
    for (int base = 0; base < R; base += kThreads) {
        const int r = base + threadIdx.x;
        long long mine = 0;
        if (r < R) {
            const int len = p.lengths[r];
            int first = r, last = r + (len > 0 ? 1 : 0);
            if (p.ends) {
                first = r > 0 ? p.ends[r - 1] : 0;
                last = p.ends[r];
            }
            const long long n = (long long)last - first;
            if (first < 0 || n < 0 || last > p.tokens || len < n || len > (long long)p.width * P) bad = true;
            else if (n > 0) mine = J::units_of(pl, len, (int)n, see);
        }
        long long x = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, off);
            if (lane >= off) x += y;
        }
        if (lane == 31) warp_sums[warp] = x;
        __syncthreads();
        long long before = carry;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += warp_sums[w];
            carry += warp_sums[w];
        }
        if (r < R) starts[r] = (int)min(before + x - mine, 0x7fffffffll);
        __syncthreads();
    }
    if (threadIdx.x == 0) starts[R] = (int)min(carry, 0x7fffffffll);
    if (carry > 0x7fffffffll) bad = true, carry = 0;
    if (bad) atomicOr(p.status, SBATTN_ST_BAD_SEQLENS);
    __syncthreads();
    return carry;
}

// rem of the rows that belong to no request
template <typename T>
__device__ __forceinline__ void clear_rem(const SbCacheParams& p, int kThreads) {
    const int R = p.requests;
    if (p.ends) {
        const int first = R > 0 ? max(0, p.ends[R - 1]) : 0;
        const long long rows = (long long)max(0, p.tokens - first) * p.heads;
        for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < rows; i += (long long)gridDim.x * kThreads)
            ((T*)p.rem.ptr)[(i % p.heads) * p.rem.stride_h + (first + i / p.heads) * p.rem.stride_t] = from_f32<T>(0.f);
    } else {
        for (int t = blockIdx.x * kThreads + threadIdx.x; t < p.tokens; t += gridDim.x * kThreads)
            if (t >= R || p.lengths[t] <= 0)
                for (int h = 0; h < p.heads; ++h) ((T*)p.rem.ptr)[h * p.rem.stride_h + t * p.rem.stride_t] = from_f32<T>(0.f);
    }
}

// One column of `count` partial results, from the right, joined by one warp: lane l has the values lane * N ... of x.  slot(a): the a-th one.
// The loads do not wait for one another.
template <int DP, int COLS, int N, typename F>
__device__ __forceinline__ void join_parts(int count, int c, int lane, F slot, float (&x)[N], float& sum) {
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = 0.f;
    const auto fetch = [&](int first, float (&y)[8][N]) {  // eight parts from `first` on
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (first + k >= count) break;
            const float* from = slot(first + k) + c * DP + lane * N;
            if constexpr (N == 4) *(float4*)y[k] = *(const float4*)from;
            else if constexpr (N == 2) *(float2*)y[k] = *(const float2*)from;
            else y[k][0] = from[0];
        }
    };
    for (int base = 0; base < count; base += 32) {
        alignas(16) float y[8][N];
        float s = base + lane < count ? slot(base + lane)[COLS * DP + c] : 0.f;
        fetch(base, y);
        const int n = min(32, count - base);
#pragma unroll 1
        for (int off = 1; off < n; off <<= 1) {
            const float z = __shfl_up_sync(0xffffffffu, s, off);
            if (lane >= off) s += z;
        }
        float right = __shfl_up_sync(0xffffffffu, s, 1);
        if (lane == 0) right = 0.f;
        const float weight = ex2(-(sum + right));
        for (int a = 0; a < n; a += 8) {
            if (a > 0) fetch(base + a, y);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (a + k >= n) break;
                const float w = __shfl_sync(0xffffffffu, weight, a + k);
#pragma unroll
                for (int i = 0; i < N; ++i) x[i] = fmaf(w, y[k][i], x[i]);
            }
        }
        sum += __shfl_sync(0xffffffffu, s, n - 1);
    }
}

// Jobs that several shares have parts of.  One block per seam between two shares: its warps take the columns, and where there are few of them, parts
// of the line of partial results, which meet in shared memory.
template <typename T, int DP, int COLS>
__global__ void __launch_bounds__(256) cached_join_kernel(const __grid_constant__ SbCacheParams p, const __grid_constant__ Plan pl) {
    constexpr int N = DP / 32;
    __shared__ float xs[8][DP], sums[8];
    pdl_wait();
    pdl_launch_dependents();
    const int b = blockIdx.x + 1, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int4 seam = pl.seams[2 * b], seam1 = pl.seams[2 * b + 1];
    if (seam.x < 0) return;
    const Jobs<T, DP, COLS, 1, 0> k{p, pl, nullptr, p.attend_current ? 1 : 0};
    Job j;
    j.first = seam.x;
    j.n = seam.y;
    j.g = seam.z;
    j.tile = seam.w;
    j.cols = min(COLS, j.n * pl.shared - j.tile * COLS);
    const int count = seam1.x - b + 2, splits = j.cols <= 1 ? 8 : j.cols <= 2 ? 4 : j.cols <= 4 ? 2 : 1;
    const int part = warp % splits, a0 = count * part / splits, a1 = count * (part + 1) / splits;
    float x[N], sum = 0.f;
    if (splits == 1) {
        for (int c = 32 * blockIdx.y + warp; c < min(j.cols, 32 * (int)blockIdx.y + 32); c += 8) {
            join_parts<DP, COLS>(count, c, lane, [&](int a) { return pl.slots + ((size_t)(b - 1 + a) * 2 + (a == 0 ? 1 : 0)) * slot_floats(COLS, DP); }, x, sum);
            k.store(j, c, lane * N, x, sum, lane == 0);
        }
        return;
    }
    const int c = warp / splits;
    if (blockIdx.y > 0) return;
    if (c < j.cols)
        join_parts<DP, COLS>(a1 - a0, c, lane, [&](int a) { return pl.slots + ((size_t)(b - 1 + a0 + a) * 2 + (a0 + a == 0 ? 1 : 0)) * slot_floats(COLS, DP); }, x, sum);
#pragma unroll
    for (int i = 0; i < N; ++i) xs[warp][lane * N + i] = x[i];
    if (lane == 0) sums[warp] = sum;
    __syncthreads();
    if (part != 0) return;
    for (int s = 1; s < splits; ++s) {
        const float weight = ex2(-sum);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = fmaf(weight, xs[warp + s][lane * N + i], x[i]);
        sum += sums[warp + s];
    }
    if (c < j.cols) k.store(j, c, lane * N, x, sum, lane == 0);
}

// flags of what may be read and written together, and the parts of the workspace
inline Plan make_plan(const SbCacheParams& p, int shares) {
    Plan pl;
    pl.shared = p.heads / p.kv_heads;
    pl.shift = -1;
    for (int i = 0; i < 17; ++i)
        if (pl.shared == 1 << i) pl.shift = i;
    const int64_t size = p.dtype == SBATTN_F32 ? 4 : 2;
    const auto even = [&](const SbMat& m, int n) { return (((uintptr_t)m.ptr | (uintptr_t)(m.stride_h * size) | (uintptr_t)(m.stride_t * size)) & (n * size - 1)) == 0; };
    pl.quads = p.head_dim % 4 == 0 && even(p.q, 4);
    pl.pairs = p.head_dim % 2 == 0 && even(p.o, 2) && even(p.v, 2);
    pl.octets = p.head_dim % 8 == 0 && even(p.q, 8) && even(p.o, 8) && even(p.v, 8);
    pl.shares = shares;
    char* w = (char*)p.workspace;
    pl.seams = (int4*)w;
    pl.slots = (float*)(w + align_up(32 * (size_t)shares, 256));
    return pl;
}
inline size_t plan_bytes(int64_t shares, int cols, int dp) { return align_up(32 * (size_t)shares, 256) + (size_t)shares * 2 * slot_floats(cols, dp) * sizeof(float); }

template <typename T, int DP, int COLS>
int launch_join(const SbCacheParams& p, const Plan& pl, cudaStream_t st) {
    if (pl.shares < 2) return 0;
    return launch_kernel(cached_join_kernel<T, DP, COLS>, dim3((unsigned)pl.shares - 1, (COLS + 31) / 32), dim3(256), 0, st, p, pl);
}

}  // namespace cached

}  // namespace sb
