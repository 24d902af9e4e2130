// Attention over the 8-bit paged cache where many queries share the keys (a conversation's next turn, a prompt in pieces): bfloat16 and float16.
// The line of work of sb_cached.cuh in tiles of 256 queries and steps of 128 keys, one share per block; the products on tcgen05.
//
// A tile is two halves of 128 queries (rows of tensor memory) against the same keys, which take turns as in sb_tc_fwd_pair.cu: while the row threads of
// one turn scores into weights, the tensor cores work for the other.  Codes become 16-bit operands once per block and step: keys float16 (exact; the queries
// are scaled by a power of two per row to at most 2^15, exact but for elements below 2^-31 of the row's largest, which lose 2^-39 of that), values bfloat16 (exact).  The scale of the keys' page goes into the factor of a
// score, that of the values' page into the weight before that becomes two bfloat16 terms (2^-16 of it is lost; float16 weights would lack the range for scales
// that differ from page to page), which the tensor cores multiply one after the other.  One term would do for bfloat16 results if all came from this kernel, as in
// the forward kernels, and takes 198 us for 219 (below); but the same request comes here or to sb_cached.cu by what its batch looks like, and 2^-8 of the weights show
// in its results (2-norm 2.4e-3 of float64 for 1.7e-3, the output's own rounding), 2^-16 do not.
//
// With e = 2^x and d = 1 + e, 1 - beta = 1 / d.  A thread owns a query; for a group of four keys entered with W, the product of 1 - beta to its right,
// the weight of key m is e_m (product of d to its left in the group) / (product of d of the group) W: one reciprocal per four keys.
// x is clamped at 30 (1 - beta = 2^-30), so that the product of a group stays below 2^121 and its reciprocal a normal number.
//
// Warps of a block (512 threads, 128 registers): 0-3 / 4-7 row warps of the first / second half, 8-11 / 12-14 convert the codes of the values / keys, which
// TMA brings to shared memory a step ahead, all of them the queries, 15 issues tcgen05.mma.
// The product with the values starts with the right 64 keys while rows work on the left ones (173 -> 163 us at head dim 64, 160 -> 152 at 32, nothing at 128).
// Tensor memory (512 columns): scores of the halves at 0 / 128 (the weights' two terms overwrite the scores of the same keys), sums at 256 / 384.
//
// Measured: 4 requests of 2000 ... 5000 tokens, 512 new ones each, 32 heads over 8, head dim 128: 219 us, 514 TFLOP/s (70 us at the rate of a bfloat16 GEMM; the low terms, not
// counted, are half as much again), where the kernel of sb_cached.cu takes 1 868. The special-function unit needs 2 560 cycles for a step of both halves, which takes about 6 100: issue slots
// are busy 54 % of the time, the tensor pipe 42 %, and with a quarter of the conversions (head dim 32) a step is not much shorter. Rows wait for their own results. Earlier forms, with one
// term of the weights: codes straight from global memory to the operands, unrolled: 302 us; three warps that convert keys and values, 168 registers: 386; codes by TMA and all
// loops rolled: 251; the rest is the queries' loads side by side, joins and shares.
// 4 requests of 4000 tokens, 512 new ones, the same heads: bfloat16 229 us, float16 227 (2 002 in the kernel of sb_cached.cu), head dim 64 188, 32 178 (1 408).  Errors of 18 calls of either
// type against float64 (2-norm): bfloat16 as the plain form's, o and rem; float16 (the output's own rounding is 2.1e-4) o as the plain form's, rem 2.18e-4 for its 2.13e-4 at
// 20 000 tokens, 2.33e-4 for 2.05e-4 at 60 000.
#include <type_traits>

#include "sb_cached.cuh"
#include "sb_tc_common.cuh"

namespace sb {

namespace {

using namespace sm100;
using namespace cached;
using bf16 = __nv_bfloat16;

constexpr int kThreads = 512, kMmaWarp = 15, kConverters = 7, kValueWarps = 4;
constexpr int kTile = 256, kStep = 128;  // queries of a tile, keys of a step
constexpr int kJobCost = 2;              // steps that a job costs besides its own
constexpr uint32_t kTmemCols = 512, kColS = 0, kColO = 256;
constexpr int kScaleSlots = 4;
// Who waits for which use of a barrier.  A wait names a phase by its parity alone: it is right where the barrier has completed all uses before the one that is meant,
// and at most that one.
//   Q_FULL (a use per job, two in turn), Q_EMPTY, K_*, RAW_*, READ_*, V_*: converters and the issuing warp go through every job and every step, in order.
//   S_READY, P_HALF, P_READY, O_READY, O_FREE of a half: used only by jobs that have columns in that half; whoever uses them counts those uses.
//   SC_FULL (a use per step, four in turn) and Q_FULL as the rows see them: rows of the second half pass over jobs of at most 128 columns without a wait, any number
//   of them, and would find either barrier uses behind.  So they wait for their scores first.  Scores of step s of job j are issued when the queries of j and the keys of s are there and
//   the products of step s - 1 have been issued, which had that step's values, scales and all before them.  And until these rows have given the weights of
//   step s, the scores of s + 2 are not issued, so that no scales of s + 4 and no queries of j + 2 have come.
enum Bar { Q_FULL0, Q_FULL1, Q_EMPTY, K_FULL, K_EMPTY, RAW_K, RAW_V, READ_K, READ_V, V_FULL0, V_FULL1, V_EMPTY0, V_EMPTY1, SC_FULL0, SC_FULL1, SC_FULL2, SC_FULL3,
           S_READY0, S_READY1, P_READY0, P_READY1, P_HALF0, P_HALF1, O_READY0, O_READY1, O_FREE0, O_FREE1, kNumBars };

struct Small {  // behind the tiles
    uint64_t bars[kNumBars];
    float temp[2][kTile];            // of the jobs in turn: inv_temp log2(e) by what the query was multiplied with
    float ks[kScaleSlots][8], vs[kScaleSlots][8];  // of the steps in turn: scales of 16 keys each
    uint32_t nan_job[4];             // of the jobs in turn: 1 + number of the job, if it has NaN among the values of keys that not all of its queries see
    Job job[8];                      // of the row warps: here, not in registers
    uint32_t tmem, abort;
};

// 16 keys: weights relative to an entering W of 1, and the products of 1 + e of the four groups of four; groups in pairs, one packed instruction for both
template <bool kMasked>
__device__ __forceinline__ void sweep(const uint32_t (&s)[16], float scale, int col0, int lim, float2 (&p)[2][4], float2 (&run)[2]) {
    const auto e_of = [](float x) {
        asm("min.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(30.f));
        return ex2_approx(x);
    };
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        run[h] = make_float2(1.f, 1.f);
#pragma unroll
        for (int m = 0; m < 4; m += 2) {
            const int i0 = 8 * h + m, i1 = i0 + 4;
            const float2 x0 = __fmul2_rn(make_float2(__uint_as_float(s[i0]), __uint_as_float(s[i0 + 1])), make_float2(scale, scale));
            const float2 x1 = __fmul2_rn(make_float2(__uint_as_float(s[i1]), __uint_as_float(s[i1 + 1])), make_float2(scale, scale));
            float2 ea = make_float2(e_of(x0.x), e_of(x1.x)), eb = make_float2(e_of(x0.y), e_of(x1.y));
            if (kMasked) {
                if (col0 + i0 >= lim) ea.x = 0.f;
                if (col0 + i1 >= lim) ea.y = 0.f;
                if (col0 + i0 + 1 >= lim) eb.x = 0.f;
                if (col0 + i1 + 1 >= lim) eb.y = 0.f;
            }
            p[h][m] = __fmul2_rn(ea, run[h]);
            run[h] = __ffma2_rn(run[h], ea, run[h]);
            p[h][m + 1] = __fmul2_rn(eb, run[h]);
            run[h] = __ffma2_rn(run[h], eb, run[h]);
        }
    }
}
// for every group 1 / (product of d), and W vs as it enters, from right to left; W <- what leaves the 16 keys on their left.  1 / (product of d) may be as small as
// 2^-120: made one factor with W it would be lost, and with it all of the stick that the group takes.  (W itself underflows where the weights
// behind it are below 2^-126.)  One factor per group, which this had been, took 195 us where two take 198 (4 requests of 2000 ... 5000 tokens, below; weights in one
// term), 152 for 159 at head dim 32.  W goes from group to group: by the product of the four reciprocals it loses 2.7e-4 of itself over 60 000 tokens for 2.0e-4 (the
// reciprocal is on average 1e-8 too small), for the same time; reciprocals put right by a Newton step leave 1e-5 and cost 2 to 5 %.
__device__ __forceinline__ void carries(const float2 (&run)[2], float vs, float& W, float2 (&r)[2], float2 (&g)[2]) {
    r[1] = make_float2(rcp_approx(run[1].x), rcp_approx(run[1].y));
    r[0] = make_float2(rcp_approx(run[0].x), rcp_approx(run[0].y));
#pragma unroll
    for (int h = 1; h >= 0; --h) {
        g[h].y = W * vs;
        W *= r[h].y;
        g[h].x = W * vs;
        W *= r[h].x;
    }
}
// into two bfloat16 terms, w the leading one
__device__ __forceinline__ void finish(const float2 (&p)[2][4], const float2 (&r)[2], const float2 (&g)[2], uint32_t (&w)[8], uint32_t (&low)[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int m = 0; m < 4; m += 2) {
            const float2 a = __fmul2_rn(__fmul2_rn(p[h][m], r[h]), g[h]), b = __fmul2_rn(__fmul2_rn(p[h][m + 1], r[h]), g[h]);  // the first product is at most one
            w[4 * h + m / 2] = pack_bf16(a.x, b.x);
            w[4 * h + 2 + m / 2] = pack_bf16(a.y, b.y);
            const uint32_t wx = w[4 * h + m / 2], wy = w[4 * h + 2 + m / 2];
            const float2 minus = make_float2(-1.f, -1.f);
            const float2 c = __ffma2_rn(make_float2(__uint_as_float(wx << 16), __uint_as_float(wy << 16)), minus, a);
            const float2 d = __ffma2_rn(make_float2(__uint_as_float(wx & 0xffff0000u), __uint_as_float(wy & 0xffff0000u)), minus, b);
            low[4 * h + m / 2] = pack_bf16(c.x, d.x);
            low[4 * h + 2 + m / 2] = pack_bf16(c.y, d.y);
        }
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

// One row of a step, 16 keys at a time from the right, one such group ahead: exponentials of the next keys (special functions) stand beside the weights
// of these (arithmetic), scores of the keys after them travel.  Weights go to columns of scores that have been read.  A loop, not its rounds one behind
// the other: the code of all roles has to stay in the instruction cache (12 % of the kernel).  us for 32 keys at a time, all exponentials and then all weights,
// with spilled registers / this, one term of the weights for bfloat16: 4 requests of 4000 tokens, 512 new ones, 32 heads over 8, bfloat16, head dim 128: 213 / 205, 64: 183 / 164, 32: 169 / 152,
// float16, 128: 266 / 226.  Jobs of few steps do not gain: 64 requests of 1000 tokens, 8 heads, head dim 128, 512 columns 277 / 276, 32 columns 131 / 131, head dim 32,
// 64 columns 93 / 96; with masked steps in this form too (twice the code) 285, 137 and 103.  More registers for rows by setmaxnreg did not help the first form.
template <bool kMasked>
__device__ __forceinline__ void row_step(uint32_t s_base, uint64_t* half_ready, const float* ks, const float* vs, float temp, int key0, int lim, float& W) {
    uint32_t u[2][16], w[8], low[8];
    float2 pw[2][2][4], run[2][2], r[2], g[2];
    const auto swept = [&](int b, int ch) {
        tmem_wait_ld(u[b]);
        sweep<kMasked>(u[b], ks[ch] * temp, key0 + 16 * ch, lim, pw[b], run[b]);
    };
    const auto out = [&](int b, int ch) {
        carries(run[b], vs[ch], W, r, g);
        finish(pw[b], r, g, w, low);
        tmem_st8(s_base + 16 * ch, w);  // in the columns of the same 16 keys' scores
        tmem_st8(s_base + 16 * ch + 8, low);
    };
    if (kMasked) {  // few steps of a job: short code counts for more
#pragma unroll 1
        for (int ch = 7; ch >= 0; --ch) {
            tmem_ld16(s_base + 16 * ch, u[0]);
            swept(0, ch);
            out(0, ch);
            if (ch == 4) {
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(half_ready);
            }
        }
        return;
    }
    tmem_ld16(s_base + 112, u[1]);
    swept(1, 7);
    tmem_ld16(s_base + 96, u[0]);
#pragma unroll 1
    for (int ch = 7; ch > 1; ch -= 2) {
        swept(0, ch - 1);
        tmem_ld16(s_base + 16 * (ch - 2), u[1]);
        out(1, ch);
        swept(1, ch - 2);
        tmem_ld16(s_base + 16 * (ch - 3), u[0]);
        out(0, ch - 1);
        if (ch == 5) {  // the right 64 keys' weights are there, and no score under them is still to be read
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(half_ready);
        }
    }
    swept(0, 0);
    out(1, 1);
    out(0, 0);
}

// ROW: bytes of a cached row, and columns of the results; DP: values of an operand's row.  Behind a row of 32 values the operands hold what shared memory happens to:
// the products for scores stop before it, and the columns of the sums that it reaches are not read.
template <typename T, int ROW>
__global__ void __launch_bounds__(kThreads, 1) cached_tc_kernel(const __grid_constant__ SbCacheParams p, const __grid_constant__ Plan pl, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    constexpr int DP = ROW < 64 ? 64 : ROW;
    using J = Jobs<T, ROW, kTile, kStep, kJobCost>;
    constexpr bool kHalf = std::is_same<T, __half>::value;
    constexpr int kHalfBytes = 128 * DP * 2, kBoxBytes = 128 * 128;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* const sQ = smem;                       // two halves
    uint8_t* const sK = sQ + 2 * kHalfBytes;        // one stage: it is free as soon as both halves have their scores
    uint8_t* const sV = sK + kHalfBytes;            // two stages
    uint8_t* const raw_k = sV + 2 * kHalfBytes;     // codes of a step
    uint8_t* const raw_v = raw_k + kStep * ROW;
    Small& sm = *(Small*)(raw_v + kStep * ROW);
    int* const starts = (int*)(&sm + 1);
    volatile uint32_t* const abort_flag = &sm.abort;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, see = p.attend_current ? 1 : 0, P = p.page_tokens;
    if (tid == 0) {
        for (int i = 0; i < kNumBars; ++i) {
            const bool by_all = i == Q_FULL0 || i == Q_FULL1, by_values = i == V_FULL0 || i == V_FULL1 || i == READ_V;
            const bool by_rows = i == P_READY0 || i == P_READY1 || i == P_HALF0 || i == P_HALF1 || i == O_FREE0 || i == O_FREE1;
            mbar_init(&sm.bars[i], by_all ? 32 * kConverters : i == K_FULL || i == READ_K ? 32 * (kConverters - kValueWarps) : by_values ? 32 * kValueWarps : by_rows ? 128 : i >= SC_FULL0 && i <= SC_FULL3 ? 2 : 1);
        }
        for (int i = 0; i < 4; ++i) sm.nan_job[i] = 0;
        sm.abort = (smem_u32(smem) & 1023u) ? 1u : 0u;  // the swizzled tiles need a 1024-byte aligned base
        fence_barrier_init();
    }
    if (tid == 0) {
        tma_prefetch_desc(&kmap);
        tma_prefetch_desc(&vmap);
    }
    if (warp == kMmaWarp) {
        tmem_alloc(&sm.tmem, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem;
    pdl_wait();
    pdl_launch_dependents();
    const long long carry = scan_requests<J, kThreads>(p, pl, starts, see);
    const long long units = *abort_flag ? 0 : carry * p.kv_heads;
    const long long shares = max(1ll, min((long long)gridDim.x, units)), self = blockIdx.x;
    const long long u0 = min(units, quotient(units * self, shares)), u1 = min(units, quotient(units * (self + 1), shares));
    const J k{p, pl, starts, see};
    const int r0 = k.find(u0);
    if (tid == 0) pl.seams[2 * self] = make_int4(-1, 0, 0, 0);

    if (warp >= 8 && warp < kMmaWarp) {
        // ------------------------------------------------------------------ codes and queries to operands
        const bool values = warp < 8 + kValueWarps;
        const int group = values ? kValueWarps : kConverters - kValueWarps, gw = values ? warp - 8 : warp - 8 - kValueWarps;
        constexpr int kPerRow = ROW / 16, kRowsALoad = 32 / kPerRow;  // 16-byte pieces of a row; rows a warp takes at a time
        const int chunk = lane % kPerRow, row0 = lane / kPerRow;
        const int flip = ROW == 128 ? (chunk >> 2) & 1 : 0;  // which half of 16 values is stored first: all banks once
        const CUtensorMap* const map = values ? &vmap : &kmap;
        uint64_t* const raw_full = &sm.bars[values ? RAW_V : RAW_K];
        uint8_t* const raw = values ? raw_v : raw_k;
        const float* const scales = values ? p.v_scale : p.k_scale;
        const int64_t scale_stride = values ? p.v_scale_stride : p.k_scale_stride;
        const int box = min(P, kStep), nb = kStep / box;  // keys of a load, loads of a step
        uint32_t ph_e = 3, ph_qe = 1, step = 0, jobs = 0, issued = 0;
        bool ok = true;
        for (long long u = u0; u < u1 && ok;) {
            const Job j = k.open(u, u1, r0);
            u += j.take;
            const int first = k.first_pos(j);
            if (first >= j.end) continue;
            const int least = k.sees(j, 0);
            int page = 0, batch = first;  // of the group's first warp, lane l: page and scale of load l % nb of step l / nb of a batch of 32 / nb
            float scale = 0.f;
            const auto load = [&](int pos) {  // by the group's first warp, when the whole group has read the codes before
                if (gw != 0) return;
                if (pos == batch) {
                    const int s = lane / nb, key = kStep * (j.steps - 1 - (pos + s)) + box * (lane % nb);
                    page = 0;
                    scale = 0.f;
                    if (pos + s < j.end && key < j.keys) {
                        page = p.tables[j.r * p.table_stride + key / P];
                        if (page < 0 || page >= p.pages) {
                            atomicOr(p.status, SBATTN_ST_BAD_PAGES);
                            page = 0;
                        }
                        scale = scales[page * scale_stride + j.g];
                    }
                    batch += 32 / nb;
                }
                const int l0 = nb * (pos - (batch - 32 / nb)), i = lane - l0, key0 = kStep * (j.steps - 1 - pos), key = key0 + box * i;
                if (i == 0) mbar_expect_tx(raw_full, min(nb, (j.keys - key0 + box - 1) / box) * box * ROW);
                __syncwarp();
                if (i >= 0 && i < nb) {
                    if (key < j.keys) tma_load_3d(raw + box * i * ROW, map, raw_full, 0, j.g * P + key % P, page);
                    float* const to = (values ? sm.vs : sm.ks)[issued % kScaleSlots] + i * (box / 16);
                    for (int e = 0; e < box / 16; ++e) to[e] = scale;
                }
                __syncwarp();
                if (i == 0) mbar_arrive(&sm.bars[SC_FULL0 + issued % kScaleSlots]);
                ++issued;
            };
            load(first);
            // the queries, when the last product with the ones before is done: 16 bytes a lane
            ok = mbar_wait(&sm.bars[Q_EMPTY], ph_qe & 1, abort_flag);
            ph_qe ^= 1;
            if (!ok) break;
            constexpr int kLanes = DP / 8, kRows = 32 / kLanes;  // lanes of a row, rows of a load
            constexpr int kAhead = 7;  // loads that travel together
            const int d = 8 * (lane % kLanes);
#pragma unroll 1
            for (int base = (warp - 8) * kRows + lane / kLanes; base < kTile; base += kAhead * kConverters * kRows) {
                uint4 w[kAhead];
#pragma unroll
                for (int n = 0; n < kAhead; ++n) {
                    const int c = base + n * kConverters * kRows;
                    w[n] = make_uint4(0u, 0u, 0u, 0u);
                    if (c >= j.cols || d >= p.head_dim) continue;
                    int h;
                    const int t = k.row_of(j, c, h);
                    const T* q = (const T*)p.q.ptr + h * p.q.stride_h + t * p.q.stride_t + d;
                    if (pl.octets) {
                        w[n] = *(const uint4*)q;
                    } else {
                        const auto at = [&](int i) { return d + i < p.head_dim ? (uint32_t)*(const uint16_t*)(q + i) : 0u; };
                        w[n] = make_uint4(at(0) | at(1) << 16, at(2) | at(3) << 16, at(4) | at(5) << 16, at(6) | at(7) << 16);
                    }
                }
#pragma unroll
                for (int n = 0; n < kAhead; ++n) {
                    const int c = base + n * kConverters * kRows, row = c & 127;
                    if (c >= kTile) break;
                    const uint32_t x[4] = {w[n].x, w[n].y, w[n].z, w[n].w};
                    float y[8], top = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (kHalf) y[i] = __half2float(__ushort_as_half((unsigned short)(x[i >> 1] >> 16 * (i & 1))));
                        else y[i] = __uint_as_float(i & 1 ? x[i >> 1] & 0xffff0000u : x[i >> 1] << 16);
                        const float a = fabsf(y[i]);
                        if (a <= 3.4028234664e38f) top = fmaxf(top, a);
                    }
#pragma unroll
                    for (int off = 1; off < kLanes; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                    const int e = top > 0.f ? min(max((int)(__float_as_uint(top) >> 23) - 127, -112), kHalf ? 14 : 127) : 14;  // up to 2^(e + 1); float16 is never made smaller
                    const float up = pow2(14 - e);
                    *(uint4*)(sQ + (c >> 7) * kHalfBytes + (d >> 6) * kBoxBytes + row * 128 + ((((d >> 3) & 7) ^ (row & 7)) << 4)) =
                        make_uint4(pack_f16(y[0] * up, y[1] * up), pack_f16(y[2] * up, y[3] * up), pack_f16(y[4] * up, y[5] * up), pack_f16(y[6] * up, y[7] * up));
                    if (d == 0) sm.temp[jobs & 1][c] = p.inv_temp * kLog2e * pow2(e - 14);
                }
            }
            fence_async_smem();
            mbar_arrive(&sm.bars[Q_FULL0 + (jobs & 1)]);

            for (int pos = first; pos < j.end; ++pos, ++step) {
                const int key0 = kStep * (j.steps - 1 - pos), st = values ? step & 1 : 0;
                ok = mbar_wait(raw_full, step & 1, abort_flag) && mbar_wait(&sm.bars[values ? V_EMPTY0 + st : K_EMPTY], (ph_e >> st) & 1, abort_flag);
                ph_e ^= 1u << st;
                if (!ok) break;
                uint8_t* const dst = values ? sV + st * kHalfBytes : sK;
                const bool edge = values && key0 + kStep > least;  // keys that some queries do not see: 0 * NaN would be NaN
                bool nan = false;
#pragma unroll 2
                for (int i = gw; i < kStep / kRowsALoad; i += group) {
                    const int row = kRowsALoad * i + row0;
                    uint4 x = *(const uint4*)(raw + row * ROW + 16 * chunk);
                    if (edge && key0 + row >= least) {
                        uint32_t* const w[4] = {&x.x, &x.y, &x.z, &x.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t bad = (((*w[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
                            if (bad && key0 + row < j.keys) nan = true;
                            *w[e] = key0 + row < j.keys ? *w[e] & ~(bad * 255u) : 0u;
                        }
                    }
                    uint32_t y[8];
                    codes_to_f16(x.x, y[0], y[1]);
                    codes_to_f16(x.y, y[2], y[3]);
                    codes_to_f16(x.z, y[4], y[5]);
                    codes_to_f16(x.w, y[6], y[7]);
                    if (values)
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float2 f = __half22float2(*(const __half2*)&y[e]);
                            y[e] = pack_bf16(f.x, f.y);
                        }
                    // 8 values (16 bytes) of a row: [128 rows][64 values] boxes, 128-byte swizzle
                    const uint4 a = make_uint4(y[0], y[1], y[2], y[3]), b = make_uint4(y[4], y[5], y[6], y[7]);
                    const int c0 = 2 * chunk + flip, c1 = c0 ^ 1;
                    *(uint4*)(dst + (c0 >> 3) * kBoxBytes + row * 128 + (((c0 & 7) ^ (row & 7)) << 4)) = flip ? b : a;
                    *(uint4*)(dst + (c1 >> 3) * kBoxBytes + row * 128 + (((c1 & 7) ^ (row & 7)) << 4)) = flip ? a : b;
                }
                if (nan) *(volatile uint32_t*)&sm.nan_job[jobs & 3] = jobs + 1;
                fence_async_smem();
                mbar_arrive(&sm.bars[values ? V_FULL0 + st : K_FULL]);
                mbar_arrive(&sm.bars[values ? READ_V : READ_K]);
                if (gw == 0) ok = mbar_wait(&sm.bars[values ? READ_V : READ_K], step & 1, abort_flag);  // the whole group has read the codes
                if (!ok) break;
                if (pos + 1 < j.end) load(pos + 1);
            }
            ++jobs;
        }
    } else if (warp == kMmaWarp) {
        // ------------------------------------------------------------------ products: the whole warp runs the loops, one lane issues
        const bool leader = elect_one();
        constexpr uint32_t idesc_s = make_idesc(128, kStep, 0, 0, 0), idesc_o = make_idesc(128, DP, 1, 0, 1);
        const SmemDesc dq = make_desc(smem_u32(sQ), 0, 1024), dk = make_desc(smem_u32(sK), 0, 1024), dv = make_desc(smem_u32(sV), kBoxBytes, 1024);
        uint32_t ph_p = 0, ph_of = 3, step = 0, jobs = 0;
        bool ok = true;
        const auto scores = [&](int t) {
            const SmemDesc a = {dq.lo + t * (kHalfBytes >> 4), dq.hi};
#pragma unroll
            for (int i = 0; i < ROW / 16; ++i) {
                const uint32_t off = (i >> 2) * kBoxBytes + (i & 3) * 32;
                if (i == 0) mma_ss<false>(leader, tmem + kColS + 128 * t, a, off, dk, off, idesc_s);
                else mma_ss<true>(leader, tmem + kColS + 128 * t, a, off, dk, off, idesc_s);
            }
            mma_commit(leader, &sm.bars[S_READY0 + t]);
        };
        for (long long u = u0; u < u1 && ok;) {
            const Job j = k.open(u, u1, r0);
            u += j.take;
            const int n = j.end - k.first_pos(j), halves = j.cols > 128 ? 2 : 1;
            if (n <= 0) continue;
            ok = mbar_wait(&sm.bars[Q_FULL0 + (jobs & 1)], (jobs >> 1) & 1, abort_flag) && mbar_wait(&sm.bars[K_FULL], step & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            for (int t = 0; t < halves; ++t) scores(t);
            mma_commit(leader, &sm.bars[K_EMPTY]);
            if (n == 1) mma_commit(leader, &sm.bars[Q_EMPTY]);
            for (int s = 0; s < n && ok; ++s, ++step) {
                const uint32_t st = step & 1;
                ok = mbar_wait(&sm.bars[V_FULL0 + st], (step >> 1) & 1, abort_flag);
                for (int t = 0; t < halves && ok; ++t) {
                    ok = mbar_wait(&sm.bars[P_HALF0 + t], (ph_p >> t) & 1, abort_flag);
                    if (ok && s == 0) {  // the sums before must have been read
                        ok = mbar_wait(&sm.bars[O_FREE0 + t], (ph_of >> t) & 1, abort_flag);
                        ph_of ^= 1u << t;
                    }
                    if (!ok) break;
                    tc_fence_after();
                    const SmemDesc b = {dv.lo + st * (kHalfBytes >> 4), dv.hi};
                    const uint32_t d = tmem + kColO + 128 * t, a = tmem + kColS + 128 * t;
#pragma unroll
                    for (int i = kStep / 16 - 1; i >= 0; --i) {
                        if (i == kStep / 32 - 1) {
                            ok = mbar_wait(&sm.bars[P_READY0 + t], (ph_p >> t) & 1, abort_flag);
                            ph_p ^= 1u << t;
                            if (!ok) break;
                            tc_fence_after();
                        }
                        if (i == kStep / 16 - 1) mma_ts_dyn(leader, d, a + 16 * i, b, i * 2048, idesc_o, s > 0);
                        else mma_ts<true>(leader, d, a + 16 * i, b, i * 2048, idesc_o);
                        mma_ts<true>(leader, d, a + 16 * i + 8, b, i * 2048, idesc_o);
                    }
                    if (!ok) break;
                    if (t == halves - 1) mma_commit(leader, &sm.bars[V_EMPTY0 + st]);
                    if (s + 1 == n) {
                        mma_commit(leader, &sm.bars[O_READY0 + t]);
                    } else {
                        if (t == 0) ok = mbar_wait(&sm.bars[K_FULL], (step + 1) & 1, abort_flag);
                        if (!ok) break;
                        tc_fence_after();
                        scores(t);
                        if (t == halves - 1) {
                            mma_commit(leader, &sm.bars[K_EMPTY]);
                            if (s + 2 == n) mma_commit(leader, &sm.bars[Q_EMPTY]);
                        }
                    }
                }
            }
            ++jobs;
        }
    } else if (warp < 8) {
        // ------------------------------------------------------------------ rows
        const int half = warp >> 2, c = 32 * warp + lane;  // column of the tile
        const uint32_t base = tmem + ((uint32_t)((warp & 3) * 32) << 16), s_base = base + kColS + 128 * half, o_base = base + kColO + 128 * half;
        uint32_t step = 0, jobs = 0, ph_s = 0, ph_o = 0;
        bool ok = true;
        for (long long u = u0; u < u1 && ok;) {
            const Job j = k.open(u, u1, r0);
            if (!j.starts && tid == 0) k.mark(j, u, units, shares, self);
            u += j.take;
            const int first = k.first_pos(j), n = max(0, j.end - first);
            const bool mine = c < j.cols, live = n > 0 && 128 * half < j.cols;
            float W = 1.f;
            bool nans = false;
            __syncwarp();
            if (lane == 0) sm.job[warp] = j;
            __syncwarp();
            if (live) {
                float temp = 0.f;
                const int lim = mine ? k.sees(j, c) : 0, least = k.sees(j, 128 * half);
                for (int pos = first; pos < j.end; ++pos, ++step) {
                    const int key0 = kStep * (j.steps - 1 - pos), slot = step % kScaleSlots;
                    // the scores first: with them, and not before, the two barriers that a half without columns skips are at the use that is meant
                    ok = mbar_wait(&sm.bars[S_READY0 + half], ph_s, abort_flag) && mbar_wait(&sm.bars[SC_FULL0 + slot], (step / kScaleSlots) & 1, abort_flag);
                    ph_s ^= 1;
                    if (ok && pos == first) {
                        ok = mbar_wait(&sm.bars[Q_FULL0 + (jobs & 1)], (jobs >> 1) & 1, abort_flag);
                        temp = sm.temp[jobs & 1][c];
                    }
                    if (!ok) break;
                    tc_fence_after();
                    const bool masked = key0 + kStep > least;
                    if (masked) row_step<true>(s_base, &sm.bars[P_HALF0 + half], sm.ks[slot], sm.vs[slot], temp, key0, lim, W);
                    else row_step<false>(s_base, &sm.bars[P_HALF0 + half], sm.ks[slot], sm.vs[slot], temp, 0, 0, W);
                    tmem_wait_st();
                    tc_fence_before();
                    mbar_arrive(&sm.bars[P_READY0 + half]);
                }
                if (!ok) break;
                if (mine && p.v.ptr) {  // for the end of the job
                    int h;
                    const int t = k.row_of(sm.job[warp], c, h);
                    const char* v = (const char*)p.v.ptr + 2 * (sm.job[warp].g * p.v.stride_h + t * p.v.stride_t);
                    for (int b = 0; b < 2 * p.head_dim; b += 128) asm volatile("prefetch.global.L1 [%0];" ::"l"(v + b));
                }
                ok = mbar_wait(&sm.bars[O_READY0 + half], ph_o, abort_flag);
                ph_o ^= 1;
                if (!ok) break;
                tc_fence_after();
                nans = *(volatile uint32_t*)&sm.nan_job[jobs & 3] == jobs + 1;
            } else {
                step += n;
            }
            const Job e = sm.job[warp];
            const bool starts_here = e.starts, whole = e.starts && e.ends;
            float* const slot = pl.slots + ((size_t)self * 2 + (starts_here ? 1 : 0)) * slot_floats(kTile, ROW);
            const float sum = -lg2_approx(W);
            if (mine && whole) k.template store<1>(e, c, p.head_dim, {0.f}, sum, true);  // rem alone
            if (mine && !whole) slot[kTile * ROW + c] = sum;
#pragma unroll 1
            for (int d0 = 0; d0 < ROW; d0 += 16) {  // 32 columns at a time: 1 to 3 % more, the steps' registers suffer
                uint32_t v[16];
                if (live) {
                    tmem_ld16(o_base + d0, v);
                    tmem_wait_ld(v);
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = 0u;
                }
                if (live && d0 + 16 == ROW) {
                    tc_fence_before();
                    mbar_arrive(&sm.bars[O_FREE0 + half]);
                }
                if (!mine) continue;
                float (&x)[16] = *(float (*)[16]) & v;
                if (nans) {  // rare: NaN in a value that this query sees
                    const int lim = k.sees(e, c);
                    for (int key = max(k.sees(e, 0), kStep * (e.steps - e.end)); key < min(lim, kStep * (e.steps - first)); ++key) {
                        const int page = p.tables[e.r * p.table_stride + key / P];
                        if (page < 0 || page >= p.pages) continue;
                        const uint8_t* code = (const uint8_t*)p.v_codes + page * p.v_stride + ((int64_t)e.g * P + key % P) * ROW + d0;
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if ((code[i] & 127) == 127) x[i] = __int_as_float(0x7fc00000);
                    }
                }
                if (whole) {
                    k.template store<16>(e, c, d0, x, sum, false);
                } else {
#pragma unroll
                    for (int i = 0; i < 16; i += 4) *(float4*)(slot + c * ROW + d0 + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
                }
            }
            if (n > 0) ++jobs;
        }
    }
    if (*abort_flag && tid == 0) pl.seams[2 * self] = make_int4(-1, 0, 0, 0);
    tc_teardown(abort_flag, p.status, tmem, kTmemCols, kMmaWarp);
    clear_rem<T>(p, kThreads);
}

template <int ROW>
constexpr size_t smem_bytes(int requests) { return 5 * 128 * (ROW < 64 ? 64 : ROW) * 2 + 2 * kStep * ROW + sizeof(Small) + sizeof(int) * ((size_t)requests + 1); }
static_assert(smem_bytes<128>(SBATTN_MAX_REQUESTS) + 1024 <= 232448, "shared memory of a block");

template <typename T, int ROW>
int launch(const SbCacheParams& p, cudaStream_t st) {
    const Plan pl = make_plan(p, sm_count());
    CUtensorMap km, vm;
    const int box = p.page_tokens < kStep ? p.page_tokens : kStep;
    if (encode_page_map(&km, p.k_codes, ROW, (int64_t)p.kv_heads * p.page_tokens, p.pages, p.k_stride, box, false) != 0 ||
        encode_page_map(&vm, p.v_codes, ROW, (int64_t)p.kv_heads * p.page_tokens, p.pages, p.v_stride, box, false) != 0)
        return kMapEncodeFailed;
    int rc = ensure_kernel_attrs((const void*)cached_tc_kernel<T, ROW>, (int)smem_bytes<ROW>(SBATTN_MAX_REQUESTS), true);
    if (rc != 0) return rc;
    rc = launch_kernel(cached_tc_kernel<T, ROW>, dim3((unsigned)pl.shares), dim3(kThreads), smem_bytes<ROW>(p.requests), st, p, pl, km, vm);
    return rc != 0 ? rc : launch_join<T, ROW, kTile>(p, pl, st);
}

}  // namespace

size_t cached_tc_workspace(const SbCacheParams& p) { return plan_bytes(sm_count(), kTile, p.row); }

template <typename T>
static int launch_row(const SbCacheParams& p, cudaStream_t st) {
    return p.row == 128 ? launch<T, 128>(p, st) : p.row == 64 ? launch<T, 64>(p, st) : launch<T, 32>(p, st);
}
int launch_cached_tc(const SbCacheParams& p, cudaStream_t st) { return p.dtype == SBATTN_F16 ? launch_row<__half>(p, st) : launch_row<bf16>(p, st); }

}  // namespace sb
