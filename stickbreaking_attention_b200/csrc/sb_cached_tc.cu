// Attention over the 8-bit paged cache where many queries share the keys (a conversation's next turn, a prompt in pieces): bfloat16, rows of 64 or
// 128 bytes.  The line of work of sb_cached.cuh in tiles of 256 queries and steps of 128 keys, one share per block; the products on tcgen05.
//
// A tile is two halves of 128 queries (rows of tensor memory) against the same keys, which take turns as in sb_tc_fwd_pair.cu: while the row threads of
// one turn scores into weights, the tensor cores work for the other.  Codes become 16-bit operands once per block and step: keys float16 (exact; the queries
// are scaled by a power of two per row to at most 2^15, exact too), values bfloat16 (exact).  The scale of the keys' page goes into the factor of a
// score, that of the values' page into the weight before it is rounded to bfloat16: one rounding of the weights, as in the forward
// kernels, and bfloat16's range.
//
// With e = 2^x and d = 1 + e, 1 - beta = 1 / d.  A thread owns a query; for a group of four keys entered with W, the product of 1 - beta to its right,
// the weight of key m is e_m (product of d to its left in the group) W / (product of d of the group): one reciprocal per four keys.
// x is clamped at 30 (1 - beta = 2^-30), so that the product of a group stays below 2^121.
//
// Warps of a block (416 threads): 0-3 / 4-7 row warps of the first / second half, 8-11 load codes and queries and convert them, 12 issues tcgen05.mma.
// Tensor memory (512 columns): scores of the halves at 0 / 128 (weights overwrite the right half of their scores), sums at 256 / 384.
#include "sb_cached.cuh"
#include "sb_tc_common.cuh"

namespace sb {

namespace {

using namespace sm100;
using namespace cached;
using bf16 = __nv_bfloat16;

constexpr int kThreads = 416, kConverters = 128, kMmaWarp = 12;
constexpr int kTile = 256, kStep = 128;  // queries of a tile, keys of a step
constexpr uint32_t kTmemCols = 512, kColS = 0, kColO = 256, kColP = 64;
constexpr int kScaleSlots = 4;
enum Bar { Q_FULL0, Q_FULL1, Q_EMPTY, K_FULL0, K_FULL1, K_EMPTY0, K_EMPTY1, V_FULL0, V_FULL1, V_EMPTY0, V_EMPTY1, SC_FULL0, SC_FULL1, SC_FULL2, SC_FULL3,
           S_READY0, S_READY1, P_READY0, P_READY1, O_READY0, O_READY1, O_FREE0, O_FREE1, kNumBars };

struct Small {  // behind the tiles
    uint64_t bars[kNumBars];
    float temp[2][kTile];            // of the jobs in turn: inv_temp log2(e) by what the query was multiplied with
    float ks[kScaleSlots][8], vs[kScaleSlots][8];  // of the steps in turn: scales of 16 keys each
    uint32_t nan_job[2];             // 1 + number of the job that has NaN among the values of keys that not all of its queries see
    uint32_t tmem, abort;
};

// one chunk of 32 keys: weights relative to an entering W of 1, and the products of 1 + e of the eight groups of four
template <bool kMasked>
__device__ __forceinline__ void sweep(const uint32_t (&s)[32], float scale0, float scale1, int col0, int lim, float2 (&p)[4][4], float2 (&run)[4]) {
    const auto e_of = [](float x) {
        asm("min.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(30.f));
        return ex2_approx(x);
    };
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        const float sc = h < 2 ? scale0 : scale1;
        run[h] = make_float2(1.f, 1.f);
#pragma unroll
        for (int m = 0; m < 4; m += 2) {
            const int i0 = 8 * h + m, i1 = i0 + 4;
            const float2 x0 = __fmul2_rn(make_float2(__uint_as_float(s[i0]), __uint_as_float(s[i0 + 1])), make_float2(sc, sc));
            const float2 x1 = __fmul2_rn(make_float2(__uint_as_float(s[i1]), __uint_as_float(s[i1 + 1])), make_float2(sc, sc));
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
// from right to left: the factor of every group; W <- what leaves the chunk on its left
__device__ __forceinline__ void carries(const float2 (&run)[4], float& W, float2 (&f)[4]) {
#pragma unroll
    for (int h = 3; h >= 0; --h) {
        f[h].y = W * rcp_approx(run[h].y);
        f[h].x = f[h].y * rcp_approx(run[h].x);
        W = f[h].x;
    }
}
__device__ __forceinline__ void finish(const float2 (&p)[4][4], const float2 (&f)[4], float vs0, float vs1, uint32_t (&w)[16]) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        const float2 v = h < 2 ? make_float2(vs0, vs0) : make_float2(vs1, vs1);  // not into f, which may be as small as 2^-120
#pragma unroll
        for (int m = 0; m < 4; m += 2) {
            const float2 a = __fmul2_rn(__fmul2_rn(p[h][m], f[h]), v), b = __fmul2_rn(__fmul2_rn(p[h][m + 1], f[h]), v);
            w[4 * h + m / 2] = pack_bf16(a.x, b.x);
            w[4 * h + 2 + m / 2] = pack_bf16(a.y, b.y);
        }
    }
}

template <int DP>
__global__ void __launch_bounds__(kThreads, 1) cached_tc_kernel(const __grid_constant__ SbCacheParams p, const __grid_constant__ Plan pl) {
    using J = Jobs<bf16, DP, kTile, kStep>;
    constexpr int kHalfBytes = 128 * DP * 2, kBoxBytes = 128 * 128;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* const sQ = smem;                       // two halves
    uint8_t* const sK = sQ + 2 * kHalfBytes;        // two stages
    uint8_t* const sV = sK + 2 * kHalfBytes;
    Small& sm = *(Small*)(sV + 2 * kHalfBytes);
    int* const starts = (int*)(&sm + 1);
    volatile uint32_t* const abort_flag = &sm.abort;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, see = p.attend_current ? 1 : 0, P = p.page_tokens;
    if (tid == 0) {
        for (int i = 0; i < kNumBars; ++i) {
            const bool by_converters = i == Q_FULL0 || i == Q_FULL1 || i == K_FULL0 || i == K_FULL1 || i == V_FULL0 || i == V_FULL1;
            const bool by_rows = i == P_READY0 || i == P_READY1 || i == O_FREE0 || i == O_FREE1;
            mbar_init(&sm.bars[i], by_converters ? kConverters : by_rows ? 128 : i >= SC_FULL0 && i <= SC_FULL3 ? 4 : 1);
        }
        sm.nan_job[0] = sm.nan_job[1] = 0;
        sm.abort = (smem_u32(smem) & 1023u) ? 1u : 0u;  // the swizzled tiles need a 1024-byte aligned base
        fence_barrier_init();
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
    const long long u0 = min(units, units * self / shares), u1 = min(units, units * (self + 1) / shares);
    const J k{p, pl, starts, see};
    const int r0 = k.find(u0);
    if (tid == 0) pl.seams[self] = make_int4(-1, 0, 0, 0);

    if (warp >= 8 && warp < kMmaWarp) {
        // ------------------------------------------------------------------ codes and queries to operands
        constexpr int kPasses = DP / 16, kPerRow = DP / 16;  // 16-byte loads of a step and lane, for keys and for values; of a row
        const int cw = warp - 8, ct = tid - 256;
        const int chunk = lane % kPerRow, row0 = 32 * cw + lane / kPerRow, dr = 32 / kPerRow;  // rows row0 + dr i
        const int flip = DP == 128 ? (chunk >> 2) & 1 : 0;  // which half of 16 values is stored first: all banks once
        const auto place = [&](int row, int half) {  // 8 values (16 bytes) of a row: [128 rows][64 values] boxes, 128-byte swizzle
            const int c16 = 2 * chunk + half;
            return (c16 >> 3) * kBoxBytes + row * 128 + (((c16 & 7) ^ (row & 7)) << 4);
        };
        uint4 kx[kPasses], vx[kPasses];
        float sk[2], sv[2];
        uint32_t ph_ke = 3, ph_ve = 3, ph_qe = 1, step = 0, jobs = 0;
        bool ok = true;
        for (long long u = u0; u < u1 && ok;) {
            const Job j = k.open(u, u1, r0);
            u += j.end - j.pos;
            const int first = k.first_pos(j);
            if (first >= j.end) continue;
            const int least = k.sees(j, 0);
            const int* const table = p.tables + j.r * p.table_stride;
            const auto load = [&](int pos) {
                const int key0 = kStep * (j.steps - 1 - pos);
                int page[2];
#pragma unroll
                for (int g = 0; g < 2; ++g) {  // this warp's 32 keys lie in one page, or in two of 16 tokens
                    const int key = key0 + 32 * cw + 16 * g;
                    page[g] = 0;
                    sk[g] = sv[g] = 0.f;
                    if (key >= j.keys) continue;
                    page[g] = table[key / P];
                    if (page[g] < 0 || page[g] >= p.pages) {
                        if (lane == 0) atomicOr(p.status, SBATTN_ST_BAD_PAGES);
                        page[g] = 0;
                    }
                    sk[g] = p.k_scale[page[g] * p.k_scale_stride + j.g];
                    sv[g] = p.v_scale[page[g] * p.v_scale_stride + j.g];
                }
#pragma unroll
                for (int i = 0; i < kPasses; ++i) {
                    const int row = row0 + dr * i, key = key0 + row;
                    kx[i] = vx[i] = make_uint4(0u, 0u, 0u, 0u);
                    if (key < j.keys) {
                        const int64_t at = ((int64_t)j.g * P + key % P) * DP + 16 * chunk, pg = (row & 16) ? page[1] : page[0];
                        kx[i] = *(const uint4*)((const uint8_t*)p.k_codes + pg * p.k_stride + at);
                        vx[i] = *(const uint4*)((const uint8_t*)p.v_codes + pg * p.v_stride + at);
                    }
                }
            };
            load(first);
            // the queries, when the last product with the ones before is done
            ok = mbar_wait(&sm.bars[Q_EMPTY], ph_qe & 1, abort_flag);
            ph_qe ^= 1;
            if (!ok) break;
            for (int c = ct; c < kTile; c += kConverters) {
                int h = 0, t = 0;
                if (c < j.cols) t = k.row_of(j, c, h);
                const bf16* q = (const bf16*)p.q.ptr + h * p.q.stride_h + t * p.q.stride_t;
                const auto eight = [&](int d, uint32_t (&w)[4]) {
                    w[0] = w[1] = w[2] = w[3] = 0u;
                    if (c >= j.cols) return;
                    if (pl.octets) {
                        if (d < p.head_dim) {
                            const uint4 x = *(const uint4*)(q + d);
                            w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (d + i < p.head_dim) w[i >> 1] |= (uint32_t)__bfloat16_as_ushort(q[d + i]) << (16 * (i & 1));
                    }
                };
                const auto lo = [](uint32_t w) { return __uint_as_float(w << 16); };
                const auto hi = [](uint32_t w) { return __uint_as_float(w & 0xffff0000u); };
                float top = 0.f;
#pragma unroll 4
                for (int d = 0; d < DP; d += 8) {
                    uint32_t w[4];
                    eight(d, w);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float a = fabsf(lo(w[i])), b = fabsf(hi(w[i]));
                        if (a <= 3.4028234664e38f) top = fmaxf(top, a);
                        if (b <= 3.4028234664e38f) top = fmaxf(top, b);
                    }
                }
                const int e = top > 0.f ? max((int)(__float_as_uint(top) >> 23) - 127, -112) : 14;  // up to 2^(e + 1)
                const float up = pow2(14 - e);
                uint8_t* const dst = sQ + (c >> 7) * kHalfBytes;
                const int row = c & 127;
#pragma unroll 4
                for (int d = 0; d < DP; d += 8) {
                    uint32_t w[4];
                    eight(d, w);
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = pack_f16(lo(w[i]) * up, hi(w[i]) * up);
                    *(uint4*)(dst + (d >> 6) * kBoxBytes + row * 128 + ((((d >> 3) & 7) ^ (row & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                }
                sm.temp[jobs & 1][c] = p.inv_temp * kLog2e * pow2(e - 14);
            }
            fence_async_smem();
            mbar_arrive(&sm.bars[Q_FULL0 + (jobs & 1)]);

            for (int pos = first; pos < j.end; ++pos, ++step) {
                const int key0 = kStep * (j.steps - 1 - pos), st = step & 1, slot = step % kScaleSlots;
                if (key0 + kStep > least) {  // keys that some queries do not see: 0 * NaN would be NaN
                    bool nan = false;
#pragma unroll
                    for (int i = 0; i < kPasses; ++i) {
                        if (key0 + row0 + dr * i < least) continue;
                        uint32_t* const w = (uint32_t*)&vx[i];
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const uint32_t bad = (((w[x] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
                            if (bad) nan = true;
                            w[x] &= ~(bad * 255u);
                        }
                    }
                    if (nan) *(volatile uint32_t*)&sm.nan_job[jobs & 1] = jobs + 1;
                }
                __syncwarp();
                if (lane == 0) {
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        sm.ks[slot][2 * cw + g] = sk[g];
                        sm.vs[slot][2 * cw + g] = sv[g];
                    }
                    mbar_arrive(&sm.bars[SC_FULL0 + slot]);
                }
                ok = mbar_wait(&sm.bars[K_EMPTY0 + st], (ph_ke >> st) & 1, abort_flag);
                ph_ke ^= 1u << st;
                if (!ok) break;
#pragma unroll
                for (int i = 0; i < kPasses; ++i) {
                    uint32_t y[8];
                    codes_to_f16(kx[i].x, y[0], y[1]);
                    codes_to_f16(kx[i].y, y[2], y[3]);
                    codes_to_f16(kx[i].z, y[4], y[5]);
                    codes_to_f16(kx[i].w, y[6], y[7]);
                    const uint4 a = make_uint4(y[0], y[1], y[2], y[3]), b = make_uint4(y[4], y[5], y[6], y[7]);
                    uint8_t* const dst = sK + st * kHalfBytes;
                    *(uint4*)(dst + place(row0 + dr * i, flip)) = flip ? b : a;
                    *(uint4*)(dst + place(row0 + dr * i, flip ^ 1)) = flip ? a : b;
                }
                fence_async_smem();
                mbar_arrive(&sm.bars[K_FULL0 + st]);
                ok = mbar_wait(&sm.bars[V_EMPTY0 + st], (ph_ve >> st) & 1, abort_flag);
                ph_ve ^= 1u << st;
                if (!ok) break;
#pragma unroll
                for (int i = 0; i < kPasses; ++i) {
                    uint32_t y[8];
                    codes_to_f16(vx[i].x, y[0], y[1]);
                    codes_to_f16(vx[i].y, y[2], y[3]);
                    codes_to_f16(vx[i].z, y[4], y[5]);
                    codes_to_f16(vx[i].w, y[6], y[7]);
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const float2 f = __half22float2(*(const __half2*)&y[x]);
                        y[x] = pack_bf16(f.x, f.y);
                    }
                    const uint4 a = make_uint4(y[0], y[1], y[2], y[3]), b = make_uint4(y[4], y[5], y[6], y[7]);
                    uint8_t* const dst = sV + st * kHalfBytes;
                    *(uint4*)(dst + place(row0 + dr * i, flip)) = flip ? b : a;
                    *(uint4*)(dst + place(row0 + dr * i, flip ^ 1)) = flip ? a : b;
                }
                fence_async_smem();
                mbar_arrive(&sm.bars[V_FULL0 + st]);
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
        const auto scores = [&](int t, uint32_t st) {
            const SmemDesc a = {dq.lo + t * (kHalfBytes >> 4), dq.hi}, b = {dk.lo + st * (kHalfBytes >> 4), dk.hi};
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {
                const uint32_t off = (i >> 2) * kBoxBytes + (i & 3) * 32;
                if (i == 0) mma_ss<false>(leader, tmem + kColS + 128 * t, a, off, b, off, idesc_s);
                else mma_ss<true>(leader, tmem + kColS + 128 * t, a, off, b, off, idesc_s);
            }
            mma_commit(leader, &sm.bars[S_READY0 + t]);
        };
        for (long long u = u0; u < u1 && ok;) {
            const Job j = k.open(u, u1, r0);
            u += j.end - j.pos;
            const int n = j.end - k.first_pos(j), halves = j.cols > 128 ? 2 : 1;
            if (n <= 0) continue;
            ok = mbar_wait(&sm.bars[Q_FULL0 + (jobs & 1)], (jobs >> 1) & 1, abort_flag) && mbar_wait(&sm.bars[K_FULL0 + (step & 1)], (step >> 1) & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            for (int t = 0; t < halves; ++t) scores(t, step & 1);
            mma_commit(leader, &sm.bars[K_EMPTY0 + (step & 1)]);
            if (n == 1) mma_commit(leader, &sm.bars[Q_EMPTY]);
            for (int s = 0; s < n && ok; ++s, ++step) {
                const uint32_t st = step & 1, next = st ^ 1;
                ok = mbar_wait(&sm.bars[V_FULL0 + st], (step >> 1) & 1, abort_flag);
                for (int t = 0; t < halves && ok; ++t) {
                    ok = mbar_wait(&sm.bars[P_READY0 + t], (ph_p >> t) & 1, abort_flag);
                    ph_p ^= 1u << t;
                    if (ok && s == 0) {  // the sums before must have been read
                        ok = mbar_wait(&sm.bars[O_FREE0 + t], (ph_of >> t) & 1, abort_flag);
                        ph_of ^= 1u << t;
                    }
                    if (!ok) break;
                    tc_fence_after();
                    const SmemDesc b = {dv.lo + st * (kHalfBytes >> 4), dv.hi};
                    const uint32_t d = tmem + kColO + 128 * t, a = tmem + kColS + 128 * t + kColP;
#pragma unroll
                    for (int i = 0; i < kStep / 16; ++i) {
                        if (i == 0) mma_ts_dyn(leader, d, a, b, 0, idesc_o, s > 0);
                        else mma_ts<true>(leader, d, a + i * 8, b, i * 2048, idesc_o);
                    }
                    if (t == halves - 1) mma_commit(leader, &sm.bars[V_EMPTY0 + st]);
                    if (s + 1 == n) {
                        mma_commit(leader, &sm.bars[O_READY0 + t]);
                    } else {
                        if (t == 0) ok = mbar_wait(&sm.bars[K_FULL0 + next], ((step + 1) >> 1) & 1, abort_flag);
                        if (!ok) break;
                        tc_fence_after();
                        scores(t, next);
                        if (t == halves - 1) {
                            mma_commit(leader, &sm.bars[K_EMPTY0 + next]);
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
            if (j.pos > 0 && tid == 0) {  // the first job of this share: the join kernel's blocks of this seam take it if it started in the share before
                const long long start = u - j.pos, last = start + j.steps, before = units * (self - 1) / shares;
                if (start >= before) pl.seams[self] = make_int4(j.r, j.g, j.tile, (int)((last * shares - 1) / units));
            }
            u += j.end - j.pos;
            const int first = k.first_pos(j), n = max(0, j.end - first);
            const bool mine = c < j.cols, live = n > 0 && 128 * half < j.cols;
            float W = 1.f;
            if (live) {
                ok = mbar_wait(&sm.bars[Q_FULL0 + (jobs & 1)], (jobs >> 1) & 1, abort_flag);
                if (!ok) break;
                const float temp = sm.temp[jobs & 1][c];
                const int lim = mine ? k.sees(j, c) : 0, least = k.sees(j, 128 * half);
                for (int pos = first; pos < j.end; ++pos, ++step) {
                    const int key0 = kStep * (j.steps - 1 - pos), slot = step % kScaleSlots;
                    ok = mbar_wait(&sm.bars[SC_FULL0 + slot], (step / kScaleSlots) & 1, abort_flag) && mbar_wait(&sm.bars[S_READY0 + half], ph_s, abort_flag);
                    ph_s ^= 1;
                    if (!ok) break;
                    tc_fence_after();
                    const bool masked = key0 + kStep > least;
                    uint32_t x[32], w[16];
                    tmem_ld32(s_base + 96, x);
                    tmem_wait_ld(x);
#pragma unroll
                    for (int ch = 3; ch >= 0; --ch) {
                        const float k0 = sm.ks[slot][2 * ch] * temp, k1 = sm.ks[slot][2 * ch + 1] * temp;
                        float2 pw[4][4], run[4], f[4];
                        if (masked) sweep<true>(x, k0, k1, key0 + 32 * ch, lim, pw, run);
                        else sweep<false>(x, k0, k1, 0, 0, pw, run);
                        if (ch > 0) tmem_ld32(s_base + 32 * (ch - 1), x);
                        carries(run, W, f);
                        finish(pw, f, sm.vs[slot][2 * ch], sm.vs[slot][2 * ch + 1], w);
                        if (ch > 0) tmem_wait_ld(x);  // the weights overwrite columns of the chunk to the left
                        tmem_st16(s_base + kColP + 16 * ch, w);
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    mbar_arrive(&sm.bars[P_READY0 + half]);
                }
                if (!ok) break;
                ok = mbar_wait(&sm.bars[O_READY0 + half], ph_o, abort_flag);
                ph_o ^= 1;
                if (!ok) break;
                tc_fence_after();
            } else {
                step += n;
            }
            const bool starts_here = j.pos == 0, whole = starts_here && j.end == j.steps;
            const bool nans = live && *(volatile uint32_t*)&sm.nan_job[jobs & 1] == jobs + 1;
            float* const slot = pl.slots + ((size_t)self * 2 + (starts_here ? 1 : 0)) * slot_floats(kTile, DP);
            const float sum = -lg2_approx(W);
            if (mine && whole) k.template store<1>(j, c, p.head_dim, {0.f}, sum, true);  // rem alone
            if (mine && !whole) slot[kTile * DP + c] = sum;
#pragma unroll 1
            for (int d0 = 0; d0 < DP; d0 += 32) {
                uint32_t v[32];
                if (live) {
                    tmem_ld32(o_base + d0, v);
                    tmem_wait_ld(v);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = 0u;
                }
                if (live && d0 + 32 == DP) {
                    tc_fence_before();
                    mbar_arrive(&sm.bars[O_FREE0 + half]);
                }
                if (!mine) continue;
                float (&x)[32] = *(float (*)[32]) & v;
                if (nans) {  // rare: NaN in a value that this query sees
                    const int lim = k.sees(j, c);
                    for (int key = max(k.sees(j, 0), kStep * (j.steps - j.end)); key < min(lim, kStep * (j.steps - first)); ++key) {
                        const int page = p.tables[j.r * p.table_stride + key / P];
                        if (page < 0 || page >= p.pages) continue;
                        const uint8_t* code = (const uint8_t*)p.v_codes + page * p.v_stride + ((int64_t)j.g * P + key % P) * DP + d0;
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if ((code[i] & 127) == 127) x[i] = __int_as_float(0x7fc00000);
                    }
                }
                if (whole) {
                    k.template store<32>(j, c, d0, x, sum, false);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) *(float4*)(slot + c * DP + d0 + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
                }
            }
            if (n > 0) ++jobs;
        }
    }
    if (*abort_flag && tid == 0) pl.seams[self] = make_int4(-1, 0, 0, 0);
    tc_teardown(abort_flag, p.status, tmem, kTmemCols, kMmaWarp);
    clear_rem<bf16>(p, kThreads);
}

template <int DP>
constexpr size_t smem_bytes(int requests) { return 6 * 128 * DP * 2 + sizeof(Small) + sizeof(int) * ((size_t)requests + 1); }
static_assert(smem_bytes<128>(SBATTN_MAX_REQUESTS) + 1024 <= 232448, "shared memory of a block");

template <int DP>
int launch(const SbCacheParams& p, cudaStream_t st) {
    const Plan pl = make_plan(p, sm_count());
    int rc = ensure_kernel_attrs((const void*)cached_tc_kernel<DP>, (int)smem_bytes<DP>(SBATTN_MAX_REQUESTS), true);
    if (rc != 0) return rc;
    rc = launch_kernel(cached_tc_kernel<DP>, dim3((unsigned)pl.shares), dim3(kThreads), smem_bytes<DP>(p.requests), st, p, pl);
    return rc != 0 ? rc : launch_join<bf16, DP, kTile>(p, pl, st);
}

}  // namespace

size_t cached_tc_workspace(const SbCacheParams& p) { return plan_bytes(sm_count(), kTile, p.row); }

int launch_cached_tc(const SbCacheParams& p, cudaStream_t st) { return p.row == 128 ? launch<128>(p, st) : launch<64>(p, st); }

}  // namespace sb
