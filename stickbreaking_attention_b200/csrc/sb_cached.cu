// Stick-breaking attention of new tokens over the 8-bit paged cache.
//
// With x_ij = q_i . k_j * inv_temp * log2(e), beta = 1 / (1 + 2^-x) and soft(x) = log2(1 + 2^x) = -log2(1 - beta), a query's weights are
// A_ij = beta_ij 2^-(sum of soft over the keys to the right of j that it sees), and two ranges of keys, each treated as if nothing were to its
// right, join by o = o_right + 2^-S_right o_left, S = S_right + S_left: no maximum and no renormalisation.  So the keys of all
// requests and heads are one line of work, cut into equal shares for all warps of the GPU wherever the cuts fall; a second kernel joins what
// the cuts have parted.
//
// What bounds it is the cache's bytes (2 row bytes per key and head, once), as long as few queries share a key.  A warp goes through its share 32
// keys at a time, from the right:
//   * TMA loads of whole rows into a ring of its own, stages ahead; no barrier between warps;
//   * codes become float16, exactly, on the way from shared memory to the operands of warp-level matrix instructions.  K is the left operand (16 keys)
//     and the queries that share the keys (heads of a group, new tokens) are the 8 columns of the right one, V the left operand
//     of the second product, d by keys.  Eight columns are what tcgen05's 128 rows would be filled with: the data path of 8-bit codes through the
//     registers is needed either way, and the tensor pipe is idle most of the time;
//   * a lane forms one key's weight for every column in float32: soft and its sums over the lanes by shuffles, the carry compensated;
//   * the weights of 32 keys, with the scale of the values' page, are scaled by a power of two to at most 2^15 per column and split into two float16 terms
//     (22 bits: what is lost is below float32's own rounding of the sums), the two products are added to float32 accumulators.
// float32 queries are two float16 terms, too; 16-bit ones are scaled by a power of two per row and exact (bfloat16: elements above 2^-31 of the row's largest).
//
// Measured (a copy's bandwidth is 6 551 GB/s): 32 requests of 1000 ... 12 000 tokens, 32 heads, head dim 128, 1.32 GB of codes 222-240 us, 5 500-5 950 GB/s; one request
// of 65 536 tokens, 8 heads 40 us, of which the steps take 18 (a bandwidth of 7 300 GB/s; what the loads cannot use is the start, lengths, tables, queries, and the
// joins); 64 requests of 100 ... 4000 tokens, 8 heads of four queries each 46 us, 2 900 GB/s: four times the weights per key, and the steps' latency with three
// warps a scheduler. Twelve warps with two stages each against eight with three: 239 / 284 us on the first (fewer spills, less to hide a step's latency with).
#include "sb_cached.cuh"
#include "sb_sm100.cuh"

#include <cstddef>
#include <type_traits>

namespace sb {

namespace {

using namespace sm100;
using namespace cached;

constexpr int kCols = 8;       // queries that share a key's product
constexpr int kJobCost = 3;    // steps that a job costs besides its own (64 requests, 512 jobs: 61 us with 0, 53 with 1, 49 with 2, 47 with 4; 16 requests of
                               // a few new tokens: 29.3, 27.4, 27.3, 29.7)
constexpr int kColStride = 40; // floats from column to column in the exchange buffer: 4-byte stores and 8-byte loads without bank conflicts

__host__ __device__ constexpr int warps(int dp) { return dp == 128 ? 12 : 8; }
__host__ __device__ constexpr int blocks_per_sm(int dp) { return dp == 128 ? 1 : 2; }
__host__ __device__ constexpr int stages(int dp) { return dp == 32 ? 4 : dp == 64 ? 3 : 2; }
__host__ __device__ constexpr int stage_bytes(int dp) { return 2 * 32 * dp; }

template <int ST>
struct alignas(16) WarpScratch {
    float x[kCols * kColStride];  // scores, then the two terms of the weights
    float2 carry[kCols];          // sum of soft to the right of the present keys, and what rounding it has lost
    float factor[kCols];          // power of two that the weights were divided by
    float temp[kCols];            // inv_temp log2(e) by what the query was multiplied with
    int limit[kCols];             // keys that the column sees
    float scale[ST][4];           // per stage: keys' scale of the lower and upper 16 keys, values' scale
    uint64_t full[ST];
    Job job[2];                   // the present one and the next one: here, not in registers
};

template <int DP>
struct Layout {
    static constexpr size_t ring = (size_t)warps(DP) * stages(DP) * stage_bytes(DP);
    static constexpr size_t scratch = ring;
    static constexpr size_t starts = scratch + warps(DP) * sizeof(WarpScratch<stages(DP)>);
    static_assert(ring % 1024 == 0 && sizeof(WarpScratch<stages(DP)>) % 16 == 0 && offsetof(WarpScratch<stages(DP)>, scale) % 16 == 0, "16-byte accesses");
    static_assert(1024 + starts + 4 * (SBATTN_MAX_REQUESTS + 1) + 256 <= 232448, "shared memory of a block");
    static size_t bytes(int requests) { return 1024 + starts + sizeof(int) * ((size_t)requests + 1); }  // 1024: the ring is aligned by hand
};

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// log2(1 + e) for 0 <= e <= 1, to 3e-7 of itself however small e is: with s = e / (2 + e) it is 2 / ln 2 artanh(s) = s Q(s^2), Q fitted on
// [0, 1/9] by least squares of the relative error, reweighted until even (4e-9)
__device__ __forceinline__ float log2_1p(float e) {
    const float s = e * rcp(2.f + e), z = s * s;
    return s * fmaf(fmaf(fmaf(fmaf(0.40652743f, z, 0.40338624f), z, 0.57743740f), z, 0.96179163f), z, 2.88539004f);
}

// Places of rows in a stage.  Rows of 128 and 64 bytes are swizzled by TMA; which keys the lanes of a phase read is chosen so
// that eight (16-byte loads) or sixteen of them (8-byte) meet all banks once.
template <int DP> __device__ __forceinline__ int chunk_at(int key, int chunk) {
    return DP == 128 ? key * 128 + ((chunk ^ (key & 7)) << 4) : key * 64 + ((chunk ^ ((key >> 1) & 3)) << 4);
}
template <int DP> __device__ __forceinline__ int key_of_row(int r) { return DP == 128 ? (r >> 1) | ((r & 1) << 2) : r; }
template <int DP> __device__ __forceinline__ int key_of(int c, int i) {  // i-th of the four keys (of 16) of the lanes with lane % 4 = c
    if (DP == 128) return 2 * c + (i & 1) + 8 * (i >> 1);
    if (DP == 64) return (c & 1) + ((c >> 1) << 2) + 2 * (i & 1) + 8 * (i >> 1);
    return c + 4 * i;
}
template <int DP> __device__ __forceinline__ int place_of(int key) {  // 16 * half + 4 c + i of a key (of 32)
    const int k = key & 15;
    if (DP == 128) return (key & 16) + 4 * ((k & 7) >> 1) + (k & 1) + 2 * (k >> 3);
    if (DP == 64) return (key & 16) + 4 * ((k & 1) + ((k >> 1) & 2)) + ((k >> 1) & 1) + 2 * (k >> 3);
    return (key & 16) + 4 * (k & 3) + (k >> 2);
}

template <typename T, int DP>
__global__ void __launch_bounds__(32 * warps(DP), blocks_per_sm(DP))
cached_kernel(const __grid_constant__ SbCacheParams p, const __grid_constant__ Plan pl, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using K = Jobs<T, DP, kCols, 32, kJobCost>;
    constexpr bool kSplitQ = sizeof(T) == 4;
    constexpr int ST = stages(DP), KW = DP / 16, VW = DP / 32, M = DP / 16, kWarps = warps(DP), kThreads = 32 * kWarps;
    extern __shared__ uint8_t raw[];
    uint8_t* const sm = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    __shared__ uint32_t gave_up;
    __shared__ volatile long long all_units;  // here, not in registers
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rr = lane >> 2, cc = lane & 3;
    uint8_t* const ring = sm + (size_t)warp * ST * stage_bytes(DP);
    WarpScratch<ST>& ws = ((WarpScratch<ST>*)(sm + Layout<DP>::scratch))[warp];
    int* const starts = (int*)(sm + Layout<DP>::starts);
    const int see = p.attend_current ? 1 : 0, P = p.page_tokens;
    if (lane == 0)
        for (int s = 0; s < ST; ++s) mbar_init(&ws.full[s], 1);
    if (threadIdx.x == 0) gave_up = 0;
    fence_barrier_init();
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&kmap);
        tma_prefetch_desc(&vmap);
    }
    pdl_wait();
    pdl_launch_dependents();

    const long long carry = scan_requests<K, kThreads>(p, pl, starts, see);
    // one share of the units per warp, neighbouring ones on different SMs
    const auto self = [&]() { return (int)(warp * gridDim.x + blockIdx.x); };
    const auto shares_of = [&](long long units) { return (int)max(1ll, min((long long)gridDim.x * kWarps, units)); };
    long long iu, w1;  // units of this share that are to come
    {
        const long long units = carry * p.kv_heads;
        const int shares = shares_of(units);
        if (threadIdx.x == 0) all_units = units;
        iu = min(units, quotient(units * self(), shares));
        w1 = min(units, quotient(units * (self() + 1), shares));
    }
    __syncthreads();
    const K k{p, pl, starts, see};
    if (lane == 0) pl.seams[2 * self()] = make_int4(-1, 0, 0, 0);

    // ---- loads: the next step to load is ipos of a job (of request ir, head ig); lane l holds the pages and scales of the l-th step of a batch of 32
    int ir = k.find(iu), ig = 0, isteps = 0, ikeys = 0, which = 0;
    bool pending = false;  // that job has not been taken over by the steps below
    int istage = 0, ipos = 0, ibatch = 0, iend = 0, loaded = 0;
    int page0 = 0, page1 = 0;
    float4 sc = make_float4(0.f, 0.f, 0.f, 0.f);
    const int box = min(32, P);
    const auto next_job = [&]() {
        const Job j = k.open(iu, w1, ir);
        if (!j.starts && lane == 0) k.mark(j, iu, all_units, shares_of(all_units), self());
        iu += j.take;
        ir = j.r;
        ig = j.g;
        isteps = j.steps;
        ikeys = j.keys;
        ipos = ibatch = k.first_pos(j);
        iend = j.end;
        pending = true;
        if (lane == 0) ws.job[which ^ 1] = j;
        if (rr < j.cols && 128 * cc < p.head_dim * (int)sizeof(T)) {  // its queries, ahead of the loads of its codes
            int h;
            const int t = k.row_of(j, rr, h);
            asm volatile("prefetch.global.L1 [%0];" ::"l"((const char*)p.q.ptr + sizeof(T) * (h * p.q.stride_h + t * p.q.stride_t) + 128 * cc));
        }
    };
    const auto load_step = [&]() {
        if (ipos == ibatch) {
            const int key = 32 * (isteps - 1 - (ipos + lane));  // first key of this lane's step
            page0 = page1 = 0;
            sc = make_float4(0.f, 0.f, 0.f, 0.f);
            bool wrong = false;
            if (ipos + lane < iend) {
                const int* table = p.tables + ir * p.table_stride;
                const auto look = [&](int at) {
                    int page = table[at / P];
                    if (page < 0 || page >= p.pages) {
                        wrong = true;
                        page = 0;
                    }
                    return page;
                };
                if (key < ikeys) {
                    page0 = look(key);
                    page1 = P == 16 && key + 16 < ikeys ? look(key + 16) : page0;
                    sc.x = p.k_scale[page0 * p.k_scale_stride + ig];
                    sc.y = p.k_scale[page1 * p.k_scale_stride + ig];
                    sc.z = p.v_scale[page0 * p.v_scale_stride + ig];
                    sc.w = p.v_scale[page1 * p.v_scale_stride + ig];
                }
            }
            if (wrong) atomicOr(p.status, SBATTN_ST_BAD_PAGES);
            ibatch += 32;
        }
        if (lane == ((ipos - (ibatch - 32)) & 31)) {
            const int key = 32 * (isteps - 1 - ipos), row = ig * P + key % P;
            uint8_t* const dst = ring + istage * stage_bytes(DP);
            const bool load = key < ikeys, two = P == 16 && key + 16 < ikeys;
            mbar_expect_tx(&ws.full[istage], (load ? 2 * box * DP : 0) + (two ? 2 * box * DP : 0));
            if (load) {
                tma_load_3d(dst, &kmap, &ws.full[istage], 0, row, page0);
                tma_load_3d(dst + 32 * DP, &vmap, &ws.full[istage], 0, row, page0);
            }
            if (two) {
                tma_load_3d(dst + 16 * DP, &kmap, &ws.full[istage], 0, row, page1);
                tma_load_3d(dst + 48 * DP, &vmap, &ws.full[istage], 0, row, page1);
            }
            *(float4*)ws.scale[istage] = sc;  // read by this warp alone, behind a __syncwarp
        }
        ++ipos;
        ++loaded;
        if (++istage == ST) istage = 0;
    };

    // ---- steps
    int stage = 0;
    uint32_t parity = 0;
    bool alive = true, working = false;
    const int pk = key_of_row<DP>(rr), place = place_of<DP>(lane);
    int pos = 0, end = 0, steps = 0, cols = 0, keys = 0, least = 0;
    bool packed = false;
    uint32_t qh[2 * KW], ql[kSplitQ ? 2 * KW : 1];
    float acc[M][4];
    for (;;) {
        while (loaded < ST) {
            if (ipos < iend) load_step();
            else if (!pending && iu < w1) next_job();
            else break;
        }
        if (!working) {
            if (!pending) break;
            // the next job: its queries, scaled to at most 2^15
            which ^= 1;
            __syncwarp();
            const Job cj = ws.job[which];
            pending = false;
            working = true;
            pos = k.first_pos(cj);
            end = cj.end;
            steps = cj.steps;
            cols = cj.cols;
            keys = cj.keys;
            least = k.sees(cj, 0);  // keys that every column sees
            packed = cols <= kCols / 2;  // the weights' low terms in the other columns
            struct alignas(4 * sizeof(T)) Four {
                T a, b, c, d;
            } nq[KW];  // column rr, the d's of this lane's words
            int h = 0, t = 0;
            if (rr < cj.cols) t = k.row_of(cj, rr, h);
            const T* q = (const T*)p.q.ptr + h * p.q.stride_h + t * p.q.stride_t;
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                const int d = DP == 128 ? 16 * (cc + 4 * (w >> 2)) + 4 * (w & 3) : DP == 64 ? 16 * cc + 4 * w : 8 * cc + 4 * w;
                nq[w] = Four{T(0.f), T(0.f), T(0.f), T(0.f)};
                if (rr < cj.cols && pos < end) {
                    if (pl.quads) {
                        if (d < p.head_dim) nq[w] = *(const Four*)(q + d);
                    } else {
                        if (d < p.head_dim) nq[w].a = q[d];
                        if (d + 1 < p.head_dim) nq[w].b = q[d + 1];
                        if (d + 2 < p.head_dim) nq[w].c = q[d + 2];
                        if (d + 3 < p.head_dim) nq[w].d = q[d + 3];
                    }
                }
            }
            float top = 0.f;
            const auto take = [&](T x) {
                const float a = fabsf(to_f32(x));
                if (a <= 3.4028234664e38f) top = fmaxf(top, a);
            };
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                take(nq[w].a);
                take(nq[w].b);
                take(nq[w].c);
                take(nq[w].d);
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = top > 0.f ? max((int)(__float_as_uint(top) >> 23) - 127, -112) : 14;  // up to 2^(e + 1)
            const float up = pow2(14 - e);
#pragma unroll
            for (int i = 0; i < 2 * KW; ++i) {
                const Four& f = nq[i >> 1];
                const float a = to_f32(i & 1 ? f.c : f.a) * up, b = to_f32(i & 1 ? f.d : f.b) * up;
                qh[i] = pack_f16(a, b);
                if (kSplitQ) {
                    const __half2 hi = *(const __half2*)&qh[i];
                    const float la = a - __low2float(hi), lb = b - __high2float(hi);  // NaN behind an infinity: the low term of that is zero
                    ql[i] = pack_f16(fabsf(a) <= 65504.f ? la : 0.f, fabsf(b) <= 65504.f ? lb : 0.f);
                }
            }
            __syncwarp();
            if (cc == 0) {
                ws.temp[rr] = p.inv_temp * 1.44269504f * pow2(e - 14);
                ws.carry[rr] = make_float2(0.f, 0.f);
                ws.limit[rr] = rr < cj.cols ? k.sees(cj, rr) : 0;
            }
            __syncwarp();
#pragma unroll
            for (int m = 0; m < M; ++m) acc[m][0] = acc[m][1] = acc[m][2] = acc[m][3] = 0.f;
            continue;
        }
        if (pos < end) {
            const int key0 = 32 * (steps - 1 - pos);
            if (!mbar_wait(&ws.full[stage], parity, &gave_up)) {
                alive = false;
                break;
            }
            __syncwarp();
            const uint8_t* const kt = ring + stage * stage_bytes(DP);
            const uint8_t* const vt = kt + 32 * DP;
            // scores: 2 x 16 keys by 8 columns
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                float s[4] = {0.f, 0.f, 0.f, 0.f};
                // float32: matrix instructions round their sums towards zero, so the two halves of d and the low terms are summed apart
                float s2[kSplitQ ? 2 : 1][4] = {};
                const int ka = 16 * mt + pk, kb = ka + 8;
                alignas(16) uint32_t wa[KW], wb[KW];
                if constexpr (DP == 32) {
                    *(uint2*)wa = *(const uint2*)(kt + ka * 32 + cc * 8);
                    *(uint2*)wb = *(const uint2*)(kt + kb * 32 + cc * 8);
                } else {
#pragma unroll
                    for (int x = 0; x < KW / 4; ++x) {
                        *(uint4*)(wa + 4 * x) = *(const uint4*)(kt + chunk_at<DP>(ka, cc + 4 * x));
                        *(uint4*)(wb + 4 * x) = *(const uint4*)(kt + chunk_at<DP>(kb, cc + 4 * x));
                    }
                }
#pragma unroll
                for (int w = 0; w < KW; ++w) {
                    uint32_t a0, a1, a2, a3;
                    codes_to_f16(wa[w], a0, a2);
                    codes_to_f16(wb[w], a1, a3);
                    mma16816(kSplitQ && 2 * w >= KW ? s2[0] : s, a0, a1, a2, a3, qh[2 * w], qh[2 * w + 1]);
                    if constexpr (kSplitQ) mma16816(s2[1], a0, a1, a2, a3, ql[2 * w], ql[2 * w + 1]);
                }
                if constexpr (kSplitQ)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[i] = s[i] + s2[0][i] + s2[1][i];
                if (2 * cc < cols) {
                    float* const x0 = ws.x + 2 * cc * kColStride + ka;
                    x0[0] = s[0];
                    x0[kColStride] = s[1];
                    x0[8] = s[2];
                    x0[kColStride + 8] = s[3];
                }
            }
            __syncwarp();
            // weights: a lane has a key; in powers of two throughout
            const float ks = ws.scale[stage][lane >> 4], vs = ws.scale[stage][2 + (lane >> 4)];
            const auto weights = [&](auto count, int c0) {
                constexpr int C = decltype(count)::value;
                float weight[C], sum[C];
#pragma unroll
                for (int i = 0; i < C; ++i) {
                    const bool seen = key0 + lane < ws.limit[c0 + i];
                    const float x = ws.x[(c0 + i) * kColStride + lane] * (ws.temp[c0 + i] * ks);
                    const float e = ex2(-fabsf(x));
                    sum[i] = seen ? fmaxf(x, 0.f) + log2_1p(e) : 0.f;
                    weight[i] = seen ? (x >= 0.f ? 1.f : e) * rcp(1.f + e) * vs : 0.f;
                }
#pragma unroll
                for (int off = 1; off < 32; off <<= 1)
#pragma unroll
                    for (int i = 0; i < C; ++i) {
                        const float y = __shfl_down_sync(0xffffffffu, sum[i], off);
                        if (lane + off < 32) sum[i] += y;
                    }
                float right[C], total[C];
                float2 had[C];
                int e2[C];
#pragma unroll
                for (int i = 0; i < C; ++i) {
                    right[i] = __shfl_down_sync(0xffffffffu, sum[i], 1);
                    if (lane == 31) right[i] = 0.f;
                    total[i] = __shfl_sync(0xffffffffu, sum[i], 0);
                    had[i] = ws.carry[c0 + i];
                    right[i] = had[i].x + (had[i].y + right[i]);
                    weight[i] = weight[i] != 0.f ? weight[i] * ex2(-right[i]) : 0.f;
                    e2[i] = max((int)(__reduce_max_sync(0xffffffffu, __float_as_uint(weight[i]) & 0x7fffffffu) >> 23), 15);
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < C; ++i) {  // to at most 2^15, and in two terms
                    const float y = weight[i] * pow2(14 + 127 - e2[i]);
                    const __half hi = __float2half_rn(y), lo = __float2half_rn(fabsf(y) <= 65504.f ? y - __half2float(hi) : 0.f);
                    __half* const to = (__half*)(ws.x + (c0 + i) * kColStride) + place;
                    to[0] = hi;
                    to[packed ? kCols / 2 * kColStride * 2 : 32] = lo;
                    if (lane == 0) {
                        ws.factor[c0 + i] = pow2(e2[i] - 127 - 14);
                        const float now = had[i].x + total[i], part = now - had[i].x;  // two-sum
                        ws.carry[c0 + i] = make_float2(now, now <= 3.4028234664e38f ? had[i].y + ((had[i].x - (now - part)) + (total[i] - part)) : 0.f);
                    }
                }
            };
            if (cols == 1) weights(std::integral_constant<int, 1>(), 0);
            else
                for (int c0 = 0; c0 < cols; c0 += 4) weights(std::integral_constant<int, 4>(), c0);  // those behind the last see nothing
            __syncwarp();
            // weights times values
            const bool edge = key0 + 32 > least;
            bool mixed_nan = false;
            alignas(16) uint32_t vw[2][4][VW];
#pragma unroll
            for (int ks16 = 0; ks16 < 2; ++ks16)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = 16 * ks16 + key_of<DP>(cc, i);
                    uint32_t(&w)[VW] = vw[ks16][i];
                    if constexpr (DP == 128) *(uint4*)w = *(const uint4*)(vt + chunk_at<DP>(key, rr));
                    else if constexpr (DP == 64) *(uint2*)w = *(const uint2*)(vt + chunk_at<DP>(key, rr >> 1) + 8 * (rr & 1));
                    else w[0] = *(const uint32_t*)(vt + key * 32 + rr * 4);
                }
            if (edge)  // keys that some columns do not see: 0 * NaN would be NaN
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int key = key0 + 16 * (i >> 2) + key_of<DP>(cc, i & 3);
                    if (key < least) continue;
#pragma unroll
                    for (int x = 0; x < VW; ++x) {
                        uint32_t& w = vw[i >> 2][i & 3][x];
                        if (key >= keys) w = 0;
                        const uint32_t nan = (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
                        if (nan) mixed_nan = true;
                        w &= ~(nan * 255u);
                    }
                }
            const int fc = packed ? 2 * (cc & 1) : 2 * cc;
            const float f0 = ws.factor[fc], f1 = ws.factor[fc + 1];
            uint32_t bh[2][2], bl[2][2];
#pragma unroll
            for (int ks16 = 0; ks16 < 2; ++ks16) {
                const uint2 h = *(const uint2*)((const __half*)(ws.x + rr * kColStride) + 16 * ks16 + 4 * cc);
                bh[ks16][0] = h.x, bh[ks16][1] = h.y;
                if (!packed) {
                    const uint2 l = *(const uint2*)((const __half*)(ws.x + rr * kColStride) + 32 + 16 * ks16 + 4 * cc);
                    bl[ks16][0] = l.x, bl[ks16][1] = l.y;
                }
            }
#pragma unroll
            for (int w = 0; w < VW; ++w) {
                float t[2][4] = {};
#pragma unroll
                for (int ks16 = 0; ks16 < 2; ++ks16)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t a0, a1, a2, a3;
                        codes_to_f16(__byte_perm(vw[ks16][0][w], vw[ks16][1][w], half ? 0x7362 : 0x5140), a0, a1);
                        codes_to_f16(__byte_perm(vw[ks16][2][w], vw[ks16][3][w], half ? 0x7362 : 0x5140), a2, a3);
                        mma16816(t[half], a0, a1, a2, a3, bh[ks16][0], bh[ks16][1]);
                        if (!packed) mma16816(t[half], a0, a1, a2, a3, bl[ks16][0], bl[ks16][1]);
                    }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float(&a)[4] = acc[2 * w + half];
                    a[0] = fmaf(f0, t[half][0], a[0]);
                    a[1] = fmaf(f1, t[half][1], a[1]);
                    a[2] = fmaf(f0, t[half][2], a[2]);
                    a[3] = fmaf(f1, t[half][3], a[3]);
                }
            }
            if (edge && __any_sync(0xffffffffu, mixed_nan)) {  // NaN for the columns that do see them
                for (int key = max(0, least - key0); key < min(32, keys - key0); ++key)
#pragma unroll
                    for (int m = 0; m < M; ++m)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int d = rr * 4 * VW + 2 * m + i, at = DP == 32 ? key * 32 + d : chunk_at<DP>(key, d >> 4) + (d & 15);
                            if ((vt[at] & 127) == 127)
#pragma unroll
                                for (int c = 0; c < 2; ++c)
                                    if (key0 + key < ws.limit[fc + c]) acc[m][2 * i + c] = __int_as_float(0x7fc00000);
                        }
            }
            __syncwarp();
            ++pos;
            --loaded;
            if (++stage == ST) {
                stage = 0;
                parity ^= 1;
            }
            if (pos < end) continue;
        }
        // the share's part of this job: the result, or a partial one
        working = false;
        const Job cj = ws.job[which];
        const bool starts_here = cj.starts;
        if (packed)
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[m][i] += __shfl_xor_sync(0xffffffffu, acc[m][i], 2);
        float* const slot = pl.slots + ((size_t)self() * 2 + (starts_here ? 1 : 0)) * slot_floats(kCols, DP);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int col = 2 * cc + c, d0 = rr * 4 * VW;
            if (col >= cj.cols) continue;
            float x[2 * M];
#pragma unroll
            for (int m = 0; m < M; ++m) {
                x[2 * m] = acc[m][c];
                x[2 * m + 1] = acc[m][2 + c];
            }
            const float sum = ws.carry[col].x + ws.carry[col].y;
            if (starts_here && cj.ends) {
                k.store(cj, col, d0, x, sum, rr == 0);
            } else {
#pragma unroll
                for (int i = 0; i < M / 2; ++i) *(float4*)(slot + col * DP + d0 + 4 * i) = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
                if (rr == 0) slot[kCols * DP + col] = sum;
            }
        }
        __syncwarp();
    }
    if (!alive) {  // no load of this warp may arrive after it has left
        uint32_t ignored = 0;
        for (; loaded > 0; --loaded) {
            mbar_wait(&ws.full[stage], parity, &ignored);
            if (++stage == ST) {
                stage = 0;
                parity ^= 1;
            }
        }
        if (lane == 0) {
            pl.seams[2 * self()] = make_int4(-1, 0, 0, 0);
            atomicOr(p.status, SBATTN_ST_TIMEOUT);
        }
    }

    clear_rem<T>(p, kThreads);
}

int64_t grid_of(const SbCacheParams& p) {
    const int64_t all = (int64_t)sm_count() * blocks_per_sm(p.row);
    const int64_t shared = p.heads / p.kv_heads, tiles = ((int64_t)p.tokens * shared + kCols - 1) / kCols + p.requests;
    const int64_t steps = ((int64_t)p.width * p.page_tokens + 31) / 32;
    const double most = (double)tiles * (double)((steps > 0 ? steps : 1) + kJobCost) * p.kv_heads;  // no more units than this
    return most < (double)all ? (most < 1. ? 1 : (int64_t)most) : all;
}

template <typename T, int DP>
int launch(const SbCacheParams& p, cudaStream_t st) {
    const int64_t grid = grid_of(p);
    const Plan pl = make_plan(p, (int)grid * warps(DP));
    CUtensorMap km, vm;
    const int box = p.page_tokens < 32 ? p.page_tokens : 32;
    if (encode_page_map(&km, p.k_codes, DP, (int64_t)p.kv_heads * p.page_tokens, p.pages, p.k_stride, box, true) != 0 ||
        encode_page_map(&vm, p.v_codes, DP, (int64_t)p.kv_heads * p.page_tokens, p.pages, p.v_stride, box, true) != 0)
        return kMapEncodeFailed;
    int rc = ensure_kernel_attrs((const void*)cached_kernel<T, DP>, (int)Layout<DP>::bytes(SBATTN_MAX_REQUESTS), true);
    if (rc != 0) return rc;
    rc = launch_kernel(cached_kernel<T, DP>, dim3((unsigned)grid), dim3(32 * warps(DP)), Layout<DP>::bytes(p.requests), st, p, pl, km, vm);
    if (rc != 0) return rc;
    return launch_join<T, DP, kCols>(p, pl, st);
}

template <typename T>
int launch_row(const SbCacheParams& p, cudaStream_t st) {
    return p.row == 128 ? launch<T, 128>(p, st) : p.row == 64 ? launch<T, 64>(p, st) : launch<T, 32>(p, st);
}

}  // namespace

// Whether the kernel of sb_cached_tc.cu takes the call: 16-bit types, and enough queries per key on average over the requests.  Both ways, us a call, bfloat16, by
// queries (heads of a group times new tokens) of a request and key/value head:
//   16 requests of 2000 tokens, 8 heads, head dim 128      16: 52 / 61   24: 69 / 63   32: 85 / 64   64: 153 / 65   256: 531 / 95   1024: 1932 / 238
//   64 requests of 1000 tokens, 8 heads, head dim 128      16: 89 / 136  24: 127 / 138  32: 154 / 140  64: 284 / 141  256: 1023 / 183
//   1 request of 16 000 tokens, 8 heads, head dim 128      16: 43 / 40   24: 48 / 43   32: 54 / 45   64: 83 / 46    256: 270 / 65
//   16 requests of 2000 tokens, 8 heads, head dim 64       16: 43 / 51   24: 54 / 52   32: 68 / 54   64: 120 / 54
//   16 requests of 2000 tokens, 8 heads, head dim 32       16: 39 / 49   24: 49 / 50   32: 62 / 52   64: 108 / 52   256: 376 / 68   1024: 1407 / 178
//   64 requests of 1000 tokens, 8 heads, head dim 32       16: 64 / 103  24: 88 / 105  32: 113 / 107  64: 202 / 108  256: 720 / 128
// It starts more slowly, which decides where there is little work (the lengths are not known here, the room in the tables is):
//   1 request of 2000 tokens, 8 heads, head dim 128        32: 28 / 29  64: 28 / 30   128: 34 / 32  256: 50 / 39
//   1 request of 300 tokens, 4 heads, head dim 64          64: 14 / 19  128: 14 / 20  256: 16 / 23
// float16 turns at the same places:
//   16 requests of 2000 tokens, 8 heads, head dim 128      16: 51 / 61   24: 69 / 62   32: 84 / 63   64: 151 / 64   256: 524 / 93    1024: 1909 / 236
//   1 request of 2000 tokens, 8 heads, head dim 128        32: 27 / 28  64: 28 / 29   128: 34 / 32  256: 50 / 38
// One kernel takes the whole batch, by its mean: single tokens beside a few prompt pieces go where the mean does.
static bool many_queries(const SbCacheParams& p) {
    const int64_t columns = (int64_t)p.tokens * (p.heads / p.kv_heads);
    return p.dtype != SBATTN_F32 && p.ends && p.requests > 0 && columns >= 24 * (int64_t)p.requests &&
           (double)columns * p.kv_heads * p.width * p.page_tokens >= 2097152.;
}

size_t cached_workspace(const SbCacheParams& p) {
    if (p.heads == 0 || p.kv_heads == 0) return 0;
    if (many_queries(p)) return cached_tc_workspace(p);
    return plan_bytes(grid_of(p) * warps(p.row), kCols, p.row);
}

int launch_cached_fwd(const SbCacheParams& p, cudaStream_t st) {
    if (many_queries(p)) return launch_cached_tc(p, st);
    if (p.dtype == SBATTN_F32) return launch_row<float>(p, st);
    if (p.dtype == SBATTN_F16) return launch_row<__half>(p, st);
    return launch_row<__nv_bfloat16>(p, st);
}

}  // namespace sb
