// A whole mixture-of-experts layer for a few tokens in one cooperative launch (lq_dev_moe_ffn):
//
//   logits[t, e] = x_t . router_e + bias_e; the top_e experts by logit (ties to the lower index), softmax weights
//   out_t = sum_j w_tj * down_j . (silu(gate_j . x_t) * (up_j . x_t))
//
// cpu_moe_forward's route -> experts -> combine (crates/larql-compute/src/cpu/ops/moe/forward.rs:24-140) over dense
// experts (every feature), the router's product included.  Experts are MXFP4, NVFP4 or FP8_B128, gate and up
// [inter, hidden], down [hidden, inter].
//
// What bounds it is reading the chosen experts' weights once.  One CTA per SM walks its share of the work in phases,
// a grid barrier between them:
//   route   the T x E router products (f64 sums: which of two near logits is larger decides a whole expert), spread
//           over the grid; after the barrier every CTA picks the experts itself (the same result everywhere);
//   gate/up units of 16 features of one expert for one group of its tokens: act = silu(gate) * up, f32, to global;
//   down    units of 16 or 32 output rows, one result per (token, expert) pair;
//   combine the pairs' weighted results in selection order.
// A producer warp streams the units' rows through a ring in shared memory (bulk copies); it needs only the routing,
// so it runs ahead across the barrier between gate/up and down.  The products run on the tensor cores (mma.sync
// m16n8k16, f16 x f16 -> f32): weights are the 16 rows of A, tokens the 8 columns of B.  The codes of all three
// formats are exact in f16; an f32 activation is brought to [2^14, 2^15) by a power of two per token and split
// in two f16 terms (22 bits), which take two columns; bf16 activations take one (f16 carries all of their 8 bits).
// Scales: e8m0 (per row and 32) and FP8 blocks on the f32 accumulators, e4m3 (per row and 16) multiplied into the f16
// codes, which is exact (2 + 4 significant bits).  The contraction is split over the 8 warps of a CTA and added
// up in a fixed order: results do not depend on timing.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/larql_cuda.h"
#include "codecs.cuh"
#include "kernels.h"

namespace lq {

namespace {

constexpr int ML_WARPS = 8, ML_CONSUMERS = ML_WARPS * 32, ML_THREADS = ML_CONSUMERS + 32;
constexpr int ML_MAX_STAGES = 12;
constexpr int ML_RED_COL = 20;  // floats between two columns of a warp's partial sums (16 rows + padding against conflicts)

struct MlSmem {
    uint64_t full[ML_MAX_STAGES], empty[ML_MAX_STAGES];
    uint64_t sfull[2], sempty[2];
    double red[ML_WARPS];
    float amax[16][ML_WARPS];   // per token of the group: the warps' parts of its largest |value|
    float unscale[16];          // per token of the group: the power of two its values were divided by
    int gtok[16], gpair[16];    // the group's tokens and (token, slot) pairs
    int n_active, n_groups;
    int active[MOE_LAYER_MAX_EXPERTS];
    int gpre[MOE_LAYER_MAX_EXPERTS + 1];     // groups before the active expert
    unsigned mask[MOE_LAYER_MAX_EXPERTS][2]; // tokens that chose the expert
    int idx[MOE_LAYER_MAX_PAIRS];
    float w[MOE_LAYER_MAX_PAIRS];
    int failed;
};

__device__ __forceinline__ float ld_as_f32(const void* p, int type, size_t at) {
    if (type == LQ_T_F32) return static_cast<const float*>(p)[at];
    if (type == LQ_T_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]);
    return __half2float(static_cast<const __half*>(p)[at]);
}

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(ML_CONSUMERS) : "memory"); }

// Grid barrier: the last CTA to arrive opens the next generation.  Bounded; false when it gave up.
__device__ bool grid_arrive_and_wait(unsigned* bar, unsigned n) {
    unsigned gen;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(gen) : "l"(bar + 1) : "memory");
    __threadfence();
    if (atomicAdd(bar, 1u) == n - 1) {
        bar[0] = 0;
        __threadfence();
        atomicAdd(bar + 1, 1u);
        return true;
    }
    const long long t0 = clock64();
    for (unsigned it = 1;; ++it) {
        unsigned now;
        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(now) : "l"(bar + 1) : "memory");
        if (now != gen) return true;
        if ((it & 255u) == 0 && clock64() - t0 > (1ll << 31)) return false;
    }
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Eight e2m1 codes (low nibble first) -> four f16 pairs.
__device__ __forceinline__ void e2m1x8(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
}
__device__ __forceinline__ uint32_t e4m3x2_f16(uint32_t two) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short)two));
    return h;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Bytes of `cols` codes, and of a row's scales.
template <int FMT>
__host__ __device__ constexpr int code_bytes(int cols) { return FMT == LQ_FMT_FP8_B128 ? cols : cols / 2; }
template <int FMT>
__host__ __device__ constexpr int row_scale_bytes(int cols) {
    return FMT == LQ_FMT_MXFP4 ? cols / 32 : (FMT == LQ_FMT_NVFP4 ? cols / 16 : 0);
}
// Distance of two rows of a stage: the eight rows of a fragment load fall into different banks (4 bytes a thread for
// FP4, 8 for FP8).
template <int FMT>
__host__ __device__ constexpr int stage_pitch(int kc) {
    const int b = code_bytes<FMT>(kc);
    return FMT == LQ_FMT_FP8_B128 ? (b % 64 == 0 ? b + 32 : b) : (b % 32 == 0 ? b + 16 : b);
}
// Distance of two columns of the activations: two columns (a phase of a 16-byte load) fall into different banks.
__host__ __device__ constexpr int act_pitch(int k) { return (2 * k) % 128 == 0 ? 2 * k + 64 : 2 * k; }
// Columns of the contraction per stage: at most 1024 (512 for FP8), in equal parts, whole 32s.
template <int FMT>
__host__ __device__ constexpr int chunk_cols(int k) {
    const int most = FMT == LQ_FMT_FP8_B128 ? 512 : 1024, n = (k + most - 1) / most;
    return ((k + n - 1) / n + 31) / 32 * 32;
}

// One phase's products as the kernel walks them.
struct Walk {
    int k, chunk, n_chunks, pitch;  // contraction, columns per stage, stages per unit, bytes between stage rows
    int units_per_group, tiles;     // 16-row tiles per unit: 2 (gate + up, or 32 rows) or 1
    int is_down;
};

template <int FMT>
__device__ __forceinline__ Walk walk_of(const MoeLayer& L, bool down, int n_groups) {
    Walk w;
    w.is_down = down;
    w.k = down ? L.inter : L.hidden;
    w.chunk = chunk_cols<FMT>(w.k);
    w.n_chunks = (w.k + w.chunk - 1) / w.chunk;
    w.pitch = stage_pitch<FMT>(w.chunk);
    if (!down) {
        w.tiles = 2;
        w.units_per_group = L.inter / 16;
    } else {
        // 32 rows a unit share the loads of the activations; 16 when there are too few units to even the SMs out
        w.tiles = (long long)n_groups * (L.hidden / 32) >= 8ll * gridDim.x ? 2 : 1;
        w.units_per_group = L.hidden / (16 * w.tiles);
    }
    return w;
}

// Active expert of group gi (groups are numbered expert by expert).
__device__ __forceinline__ int expert_of(const MlSmem& sh, int gi, int from) {
    while (gi >= sh.gpre[from + 1]) ++from;
    return from;
}

template <int FMT, int NT, int TERMS>
__global__ void __launch_bounds__(ML_THREADS, 1) moe_layer_kernel(const MoeLayer L) {
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int TG = NT * 8 / TERMS;  // tokens per group
    constexpr int RED = 2 * NT * 8 * ML_RED_COL;  // floats of a warp's partial sums
    MlSmem& sh = *reinterpret_cast<MlSmem*>(smem);
    uint8_t* p = smem + (sizeof(MlSmem) + 127) / 128 * 128;
    float* red = reinterpret_cast<float*>(p);                 // [2][ML_WARPS][RED]
    p += 2 * ML_WARPS * RED * 4;
    uint8_t* xs = p;                                          // [NT * 8] columns of f16
    p += (size_t)NT * 8 * max(act_pitch(L.hidden), act_pitch(L.inter));
    uint8_t* sbuf = p;                                        // [2] scales of a unit's rows
    const int sbytes = max(row_scale_bytes<FMT>(L.hidden), row_scale_bytes<FMT>(L.inter)) * 32;
    p += 2 * sbytes;
    uint8_t* ring = p;                                        // [n_stages][32 rows]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int T = L.tokens, E = L.experts, K = L.top_e;

    if (tid == 0) {
        for (int i = 0; i < L.n_stages; ++i) {
            mbar_init(&sh.full[i], 1);
            mbar_init(&sh.empty[i], ML_WARPS);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.sfull[i], 1);
            mbar_init(&sh.sempty[i], ML_WARPS);
        }
        sh.failed = 0;
        fence_mbar_init();
    }
    for (int i = tid; i < 2 * E; i += ML_THREADS) sh.mask[i >> 1][i & 1] = 0;

    // ---- route ----
    {
        const int items = T * E;
        const bool whole = items <= 2 * (int)gridDim.x;  // a product per CTA, or per warp
        const int step = whole ? gridDim.x : gridDim.x * (ML_THREADS / 32);
        const int n_thr = whole ? ML_THREADS : 32, me = whole ? tid : lane;
        for (int it = whole ? blockIdx.x : blockIdx.x * (ML_THREADS / 32) + warp; it < items; it += step) {
            const int t = it / E, e = it - t * E;
            double s = 0.0;
            for (int i = me; i < L.hidden; i += n_thr)
                s = fma((double)ld_as_f32(L.x, L.type, (size_t)t * L.hidden + i), (double)ld_as_f32(L.router, L.router_type, (size_t)e * L.hidden + i), s);
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            if (whole) {
                __syncthreads();
                if (lane == 0) reinterpret_cast<double*>(red)[warp] = s;
                __syncthreads();
                s = 0.0;
                for (int i = 0; i < ML_THREADS / 32; ++i) s += reinterpret_cast<double*>(red)[i];
            }
            if (me == 0) L.logits[it] = (float)(s + (L.bias ? (double)ld_as_f32(L.bias, L.router_type, e) : 0.0));
        }
    }
    __syncthreads();
    if (tid == 0 && !grid_arrive_and_wait(L.barrier, gridDim.x)) sh.failed = 1;
    __syncthreads();
    for (int t = warp; t < T; t += ML_THREADS / 32) {
        // a warp per token: K rounds of the largest (logit, lowest index) left
        constexpr int PER = MOE_LAYER_MAX_EXPERTS / 32;
        unsigned long long key[PER];
        float lg[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = i * 32 + lane;
            lg[i] = e < E ? __ldcg(L.logits + (size_t)t * E + e) : -INFINITY;
            uint32_t u = __float_as_uint(lg[i]);
            u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
            if (lg[i] != lg[i]) u = 1;  // a NaN is taken last; the weights become NaN all the same
            key[i] = e < E ? ((unsigned long long)u << 32) | (uint32_t)(0xffffffffu - e) : 0ull;
        }
        float mx = -INFINITY, sum = 0.0f, mine = 0.0f;
        int chosen = 0;
        for (int j = 0; j < K; ++j) {
            unsigned long long best = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) best = max(best, key[i]);
            for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
            const int e = (int)(0xffffffffu - (uint32_t)best);
            float l = 0.0f;
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (i == (e >> 5)) {
                    l = lg[i];
                    if (lane == (e & 31)) key[i] = 0;
                }
            l = __shfl_sync(0xffffffffu, l, e & 31);
            if (j == 0) mx = l;
            if (j == lane) {
                mine = expf(l - mx);
                chosen = e;
            }
        }
        if (L.renormalise) {
            sum = lane < K ? mine : 0.0f;
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (i * 32 + lane < E) sum += expf(lg[i] - mx);
        }
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane < K) {
            const float w = mine / sum;
            sh.idx[t * K + lane] = chosen;
            sh.w[t * K + lane] = w;
            atomicOr(&sh.mask[chosen][t >> 5], 1u << (t & 31));
            if (blockIdx.x == 0) {
                if (L.idx_out) L.idx_out[(size_t)t * K + lane] = (uint32_t)chosen;
                if (L.w_out) L.w_out[(size_t)t * K + lane] = w;
            }
        }
    }
    __syncthreads();
    if (warp == 0) {  // the chosen experts in order, and their token groups
        int n = 0, groups = 0;
        for (int e0 = 0; e0 < E; e0 += 32) {
            const int e = e0 + lane;
            const int cnt = e < E ? __popc(sh.mask[e][0]) + __popc(sh.mask[e][1]) : 0;
            const int g = (cnt + TG - 1) / TG;
            int pre = g;
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, pre, o);
                if (lane >= o) pre += v;
            }
            const unsigned on = __ballot_sync(0xffffffffu, cnt > 0);
            if (cnt > 0) {
                const int at = n + __popc(on & ((1u << lane) - 1));
                sh.active[at] = e;
                sh.gpre[at] = groups + pre - g;
            }
            n += __popc(on);
            groups += __shfl_sync(0xffffffffu, pre, 31);
        }
        if (lane == 0) {
            sh.gpre[n] = groups;
            sh.n_active = n;
            sh.n_groups = groups;
        }
    }
    __syncthreads();
    const int n_groups = sh.n_groups;

    if (warp == ML_WARPS) {
        // ---- producer: the rows of both phases' units, in order ----
        bool ok = true;
        int n = 0, un = 0;  // stages and units so far
        for (int ph = 0; ph < 2 && ok; ++ph) {
            const Walk w = walk_of<FMT>(L, ph == 1, n_groups);
            const long long total = (long long)n_groups * w.units_per_group;
            const long long ua = total * blockIdx.x / gridDim.x, ub = total * (blockIdx.x + 1) / gridDim.x;
            int a = 0;
            for (long long u = ua; u < ub && ok; ++u) {
                const int gi = (int)(u / w.units_per_group), tile = (int)(u - (long long)gi * w.units_per_group);
                a = expert_of(sh, gi, a);
                const MoeExpert& ex = L.table[sh.active[a]];
                const size_t row_bytes = (size_t)code_bytes<FMT>(w.k);
                if (row_scale_bytes<FMT>(w.k)) {
                    const int s = un & 1;
                    if (un >= 2) ok = __all_sync(0xffffffffu, mbar_wait(&sh.sempty[s], (uint32_t)(un / 2 - 1) & 1u));
                    if (!ok) break;
                    if (lane == 0) {
                        const uint32_t bytes = 16u * row_scale_bytes<FMT>(w.k);
                        mbar_expect_tx(&sh.sfull[s], bytes * w.tiles);
                        for (int i = 0; i < w.tiles; ++i) {
                            const uint8_t* src = w.is_down ? ex.scales[2] + (size_t)(tile * w.tiles + i) * bytes : ex.scales[i] + (size_t)tile * bytes;
                            tma_bulk_g2s(sbuf + s * sbytes + i * bytes, src, bytes, &sh.sfull[s]);
                        }
                    }
                }
                ++un;
                for (int c = 0; c < w.n_chunks; ++c, ++n) {
                    const int st = n % L.n_stages, k0 = c * w.chunk;
                    if (n >= L.n_stages) ok = __all_sync(0xffffffffu, mbar_wait(&sh.empty[st], (uint32_t)(n / L.n_stages - 1) & 1u));
                    if (!ok) break;
                    const uint32_t bytes = (uint32_t)code_bytes<FMT>(min(w.chunk, w.k - k0));
                    if (lane == 0) mbar_expect_tx(&sh.full[st], bytes * 16u * w.tiles);
                    __syncwarp();
                    if (lane < 16 * w.tiles) {
                        const uint8_t* m = w.is_down ? ex.codes[2] : ex.codes[lane >> 4];
                        const size_t row = w.is_down ? (size_t)tile * 16 * w.tiles + lane : (size_t)tile * 16 + (lane & 15);
                        tma_bulk_g2s(ring + (size_t)st * L.stage_bytes + lane * w.pitch, m + row * row_bytes + code_bytes<FMT>(k0), bytes,
                                     &sh.full[st]);
                    }
                }
            }
        }
        if (!ok) {  // the copies in flight have to land before the block's shared memory goes away
            for (int v = max(0, n - L.n_stages); v < n; ++v) mbar_wait(&sh.full[v % L.n_stages], (uint32_t)(v / L.n_stages) & 1u);
            if (row_scale_bytes<FMT>(L.hidden))
                for (int v = max(0, un - 2); v < un; ++v) mbar_wait(&sh.sfull[v & 1], (uint32_t)(v / 2) & 1u);
            sh.failed = 1;
        }
    } else {
        // ---- consumers ----
        const int g = lane >> 2, t4 = lane & 3;
        bool ok = true;  // a wait that ran out is not waited for again; barriers and arrivals are kept
        int n = 0, un = 0;
        for (int ph = 0; ph < 2; ++ph) {
            const Walk w = walk_of<FMT>(L, ph == 1, n_groups);
            const int xpitch = act_pitch(w.k), srow = row_scale_bytes<FMT>(w.k);
            const long long total = (long long)n_groups * w.units_per_group;
            const long long ua = total * blockIdx.x / gridDim.x, ub = total * (blockIdx.x + 1) / gridDim.x;
            int a = 0, cur = -1, cnt = 0;
            for (long long u = ua; u < ub; ++u, ++un) {
                const int gi = (int)(u / w.units_per_group), tile = (int)(u - (long long)gi * w.units_per_group);
                a = expert_of(sh, gi, a);
                const int e = sh.active[a];
                const MoeExpert& ex = L.table[e];
                if (gi != cur) {
                    // the group's tokens: which they are, and their activations as columns of f16
                    cur = gi;
                    const int first = (gi - sh.gpre[a]) * TG;
                    const unsigned long long m0 = sh.mask[e][0] | ((unsigned long long)sh.mask[e][1] << 32);
                    cnt = min(TG, __popcll(m0) - first);
                    consumers_sync();  // everyone is done with the previous group
                    if (tid < cnt) {
                        unsigned long long m = m0;
                        for (int i = 0; i < first + tid; ++i) m &= m - 1;
                        const int t = __ffsll((long long)m) - 1;
                        int j = 0;
                        while (sh.idx[t * K + j] != e) ++j;
                        sh.gtok[tid] = t;
                        sh.gpair[tid] = t * K + j;
                    }
                    consumers_sync();
                    // the warps share the rows out: `per` warps a token
                    const int per = cnt >= 5 ? 1 : (cnt >= 3 ? 2 : (cnt == 2 ? 4 : 8)), at_once = ML_WARPS / per;
                    for (int i0 = 0; i0 < cnt; i0 += at_once) {
                        const int i = i0 + warp / per, part = (warp % per) * 32 + lane;
                        if (i < cnt) {
                            float m = 0.0f;
                            for (int k = part; k < w.k; k += per * 32) {
                                const float v = w.is_down ? __ldcg(L.act + (size_t)sh.gpair[i] * w.k + k) : ld_as_f32(L.x, L.type, (size_t)sh.gtok[i] * w.k + k);
                                m = fmaxf(m, fabsf(v));
                            }
                            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                            if (lane == 0) sh.amax[i][warp % per] = m;
                        }
                    }
                    consumers_sync();
                    for (int i0 = 0; i0 < cnt; i0 += at_once) {
                        const int i = i0 + warp / per, part = (warp % per) * 32 + lane;
                        if (i < cnt) {
                            float m = 0.0f;
                            for (int q = 0; q < per; ++q) m = fmaxf(m, sh.amax[i][q]);
                            // exponent of the largest value -> 2^14 (kept where both powers of two are normal numbers)
                            const int ex2 = min(max((int)(__float_as_uint(m) >> 23), 15), 254);
                            const float down = __uint_as_float((uint32_t)(127 + 14 + 127 - ex2) << 23);
                            if (warp % per == 0 && lane == 0) sh.unscale[i] = __uint_as_float((uint32_t)(ex2 - 14) << 23);
                            for (int k = part; k < w.k; k += per * 32) {
                                const float v = (w.is_down ? __ldcg(L.act + (size_t)sh.gpair[i] * w.k + k) : ld_as_f32(L.x, L.type, (size_t)sh.gtok[i] * w.k + k)) * down;
                                const __half hi = __float2half_rn(v);
                                *reinterpret_cast<__half*>(xs + (size_t)(i * TERMS) * xpitch + 2 * k) = hi;
                                if (TERMS == 2)
                                    *reinterpret_cast<__half*>(xs + (size_t)(i * TERMS + 1) * xpitch + 2 * k) = __float2half_rn(v - __half2float(hi));
                            }
                        }
                    }
                    consumers_sync();
                }
                float acc[2][NT][4];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int q = 0; q < 4; ++q) acc[i][j][q] = 0.0f;
                if (FMT != LQ_FMT_FP8_B128 && ok) ok = __all_sync(0xffffffffu, mbar_wait(&sh.sfull[un & 1], (uint32_t)(un / 2) & 1u));
                const uint8_t* sc = sbuf + (un & 1) * sbytes;
                for (int c = 0; c < w.n_chunks; ++c, ++n) {
                    const int st = n % L.n_stages, k0 = c * w.chunk, blocks = min(w.chunk, w.k - k0) / 32;
                    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&sh.full[st], (uint32_t)(n / L.n_stages) & 1u));
                    const uint8_t* rows = ring + (size_t)st * L.stage_bytes;
                    for (int b = warp; b < blocks; b += ML_WARPS) {
                        const int kb = k0 / 32 + b;  // block of 32 columns of the row
                        uint4 xb[NT];
#pragma unroll
                        for (int j = 0; j < NT; ++j)
                            xb[j] = *reinterpret_cast<const uint4*>(xs + (size_t)(j * 8 + g) * xpitch + kb * 64 + t4 * 16);
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            if (i >= w.tiles) break;
                            const uint8_t* r0 = rows + (i * 16 + g) * w.pitch;
                            const uint8_t* r1 = r0 + 8 * w.pitch;
                            uint32_t h0[4], h1[4];
                            if (FMT == LQ_FMT_FP8_B128) {
                                const uint2 q0 = *reinterpret_cast<const uint2*>(r0 + b * 32 + t4 * 8);
                                const uint2 q1 = *reinterpret_cast<const uint2*>(r1 + b * 32 + t4 * 8);
                                h0[0] = e4m3x2_f16(q0.x), h0[1] = e4m3x2_f16(q0.x >> 16), h0[2] = e4m3x2_f16(q0.y), h0[3] = e4m3x2_f16(q0.y >> 16);
                                h1[0] = e4m3x2_f16(q1.x), h1[1] = e4m3x2_f16(q1.x >> 16), h1[2] = e4m3x2_f16(q1.y), h1[3] = e4m3x2_f16(q1.y >> 16);
                            } else {
                                e2m1x8(*reinterpret_cast<const uint32_t*>(r0 + b * 16 + t4 * 4), h0);
                                e2m1x8(*reinterpret_cast<const uint32_t*>(r1 + b * 16 + t4 * 4), h1);
                            }
                            const uint8_t* s0 = sc + (i * 16 + g) * srow;
                            const uint8_t* s1 = s0 + 8 * srow;
                            if (FMT == LQ_FMT_NVFP4) {
                                const uint32_t f0 = s0[2 * kb + (t4 >> 1)], f1 = s1[2 * kb + (t4 >> 1)];
                                const uint32_t m0 = e4m3x2_f16(f0 | (f0 << 8)), m1 = e4m3x2_f16(f1 | (f1 << 8));
#pragma unroll
                                for (int q = 0; q < 4; ++q) {
                                    h0[q] = mul_f16x2(h0[q], m0);
                                    h1[q] = mul_f16x2(h1[q], m1);
                                }
#pragma unroll
                                for (int j = 0; j < NT; ++j) {
                                    mma_f16(acc[i][j], h0[0], h1[0], h0[1], h1[1], xb[j].x, xb[j].y);
                                    mma_f16(acc[i][j], h0[2], h1[2], h0[3], h1[3], xb[j].z, xb[j].w);
                                }
                            } else {
                                float f0, f1;
                                if (FMT == LQ_FMT_MXFP4) {
                                    f0 = e8m0_to_f32(s0[kb]);
                                    f1 = e8m0_to_f32(s1[kb]);
                                } else {
                                    const int row = w.is_down ? (tile * w.tiles + i) * 16 : tile * 16;
                                    const float* fs = reinterpret_cast<const float*>(ex.scales[w.is_down ? 2 : i]);
                                    f0 = f1 = __ldg(fs + (size_t)(row >> 7) * ((w.k + 127) >> 7) + (kb >> 2));
                                }
#pragma unroll
                                for (int j = 0; j < NT; ++j) {
                                    float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                                    mma_f16(d, h0[0], h1[0], h0[1], h1[1], xb[j].x, xb[j].y);
                                    mma_f16(d, h0[2], h1[2], h0[3], h1[3], xb[j].z, xb[j].w);
                                    acc[i][j][0] = fmaf(d[0], f0, acc[i][j][0]);
                                    acc[i][j][1] = fmaf(d[1], f0, acc[i][j][1]);
                                    acc[i][j][2] = fmaf(d[2], f1, acc[i][j][2]);
                                    acc[i][j][3] = fmaf(d[3], f1, acc[i][j][3]);
                                }
                            }
                        }
                    }
                    __syncwarp();
                    if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&sh.empty[st])) : "memory");
                }
                if (FMT != LQ_FMT_FP8_B128 && lane == 0)
                    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&sh.sempty[un & 1])) : "memory");
                // the warps' parts, in warp order
                float* mine = red + ((size_t)(un & 1) * ML_WARPS + warp) * RED;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        float* q = mine + (i * NT * 8 + j * 8 + 2 * t4) * ML_RED_COL + g;
                        q[0] = acc[i][j][0];
                        q[ML_RED_COL] = acc[i][j][1];
                        q[8] = acc[i][j][2];
                        q[ML_RED_COL + 8] = acc[i][j][3];
                    }
                consumers_sync();
                const float* all = red + (size_t)(un & 1) * ML_WARPS * RED;
                auto sum = [&](int i, int tok, int row, float scale) {
                    float s = 0.0f;
                    for (int q = 0; q < ML_WARPS; ++q)
#pragma unroll
                        for (int m = 0; m < TERMS; ++m) s += all[(size_t)q * RED + (i * NT * 8 + tok * TERMS + m) * ML_RED_COL + row];
                    return s * scale;
                };
                if (!w.is_down) {
                    const int row = tid & 15, tok = tid >> 4;
                    if (tok < cnt) {
                        const float un_x = sh.unscale[tok];
                        const float gate = sum(0, tok, row, un_x) * ex.ts[0], up = sum(1, tok, row, un_x) * ex.ts[1];
                        L.act[(size_t)sh.gpair[tok] * L.inter + tile * 16 + row] = gate / (1.0f + expf(-gate)) * up;
                    }
                } else {
                    for (int i = 0; i < w.tiles; ++i) {
                        const int row = tid & 15, tok = tid >> 4;
                        // the routing weight goes into the power of two, so that only the weighted output has to be in range
                        if (tok < cnt)
                            L.pair_out[(size_t)sh.gpair[tok] * L.hidden + (tile * w.tiles + i) * 16 + row] =
                                sum(i, tok, row, sh.unscale[tok] * sh.w[sh.gpair[tok]]) * ex.ts[2];
                    }
                }
            }
            consumers_sync();
            if (tid == 0 && !grid_arrive_and_wait(L.barrier, gridDim.x)) sh.failed = 1;
            consumers_sync();
        }
        if (!ok && lane == 0) sh.failed = 1;
        // ---- combine ----
        const long long n_out = (long long)T * L.hidden;
        for (long long i = (long long)blockIdx.x * ML_CONSUMERS + tid; i < n_out; i += (long long)gridDim.x * ML_CONSUMERS) {
            const int t = (int)(i / L.hidden), h = (int)(i - (long long)t * L.hidden);
            float s = 0.0f;
            for (int j = 0; j < K; ++j) s += __ldcg(L.pair_out + (size_t)(t * K + j) * L.hidden + h);
            if (L.type == LQ_T_F32) static_cast<float*>(L.out)[i] = s;
            else if (L.type == LQ_T_BF16) static_cast<__nv_bfloat16*>(L.out)[i] = __float2bfloat16_rn(s);
            else static_cast<__half*>(L.out)[i] = __float2half_rn(s);
        }
    }
    __syncthreads();
    if (tid == 0 && sh.failed) set_err(L.err, DEV_ERR_TMA_TIMEOUT);
}

template <int FMT, int NT, int TERMS>
size_t fixed_smem(int hidden, int inter) {
    const size_t red = 2 * ML_WARPS * (2 * NT * 8 * ML_RED_COL) * 4;
    const size_t sb = 2 * (size_t)std::max(row_scale_bytes<FMT>(hidden), row_scale_bytes<FMT>(inter)) * 32;
    return (sizeof(MlSmem) + 127) / 128 * 128 + red + (size_t)NT * 8 * std::max(act_pitch(hidden), act_pitch(inter)) + sb;
}

template <int FMT, int NT, int TERMS>
cudaError_t launch_layer(MoeLayer L, int sm_count, cudaStream_t st) {
    const size_t most = 227 * 1024, fixed = fixed_smem<FMT, NT, TERMS>(L.hidden, L.inter);
    L.stage_bytes = 32 * std::max(stage_pitch<FMT>(chunk_cols<FMT>(L.hidden)), stage_pitch<FMT>(chunk_cols<FMT>(L.inter)));
    if (fixed + 2 * (size_t)L.stage_bytes > most) return cudaErrorInvalidConfiguration;
    L.n_stages = (int)std::min<size_t>(ML_MAX_STAGES, (most - fixed) / L.stage_bytes);
    const void* fn = (const void*)moe_layer_kernel<FMT, NT, TERMS>;
    cudaError_t e = set_max_dyn_smem(fn, (int)most);
    if (e != cudaSuccess) return e;
    void* args[] = {&L};
    return cudaLaunchCooperativeKernel(fn, dim3(sm_count), dim3(ML_THREADS), args, fixed + (size_t)L.n_stages * L.stage_bytes, st);
}

template <int FMT>
cudaError_t launch_fmt(const MoeLayer& L, int sm_count, cudaStream_t st) {
    // Two column tiles (16 columns) when the tokens fill more than one and the activations leave room for a ring.
    const int terms = L.type == LQ_T_BF16 ? 1 : 2;
    const bool wide = L.tokens * terms > 8 &&
                      (terms == 1 ? fixed_smem<FMT, 2, 1>(L.hidden, L.inter) : fixed_smem<FMT, 2, 2>(L.hidden, L.inter)) <= 150 * 1024;
    if (terms == 1) return wide ? launch_layer<FMT, 2, 1>(L, sm_count, st) : launch_layer<FMT, 1, 1>(L, sm_count, st);
    return wide ? launch_layer<FMT, 2, 2>(L, sm_count, st) : launch_layer<FMT, 1, 2>(L, sm_count, st);
}

}  // namespace

template <int FMT>
static bool fits(int hidden, int inter) {
    const int pitch = std::max(stage_pitch<FMT>(chunk_cols<FMT>(hidden)), stage_pitch<FMT>(chunk_cols<FMT>(inter)));
    return fixed_smem<FMT, 1, 2>(hidden, inter) + 2 * 32 * (size_t)pitch <= 227 * 1024;
}
bool moe_layer_supported(int fmt, int hidden, int inter) {
    if (hidden <= 0 || inter <= 0 || hidden % 32 || inter % 32 || hidden > 8192 || inter > 8192) return false;
    switch (fmt) {
        case LQ_FMT_MXFP4: return fits<LQ_FMT_MXFP4>(hidden, inter);
        case LQ_FMT_NVFP4: return fits<LQ_FMT_NVFP4>(hidden, inter);
        case LQ_FMT_FP8_B128: return fits<LQ_FMT_FP8_B128>(hidden, inter);
    }
    return false;
}

cudaError_t launch_moe_layer(int fmt, const MoeLayer& L, int sm_count, cudaStream_t st) {
    switch (fmt) {
        case LQ_FMT_MXFP4: return launch_fmt<LQ_FMT_MXFP4>(L, sm_count, st);
        case LQ_FMT_NVFP4: return launch_fmt<LQ_FMT_NVFP4>(L, sm_count, st);
        case LQ_FMT_FP8_B128: return launch_fmt<LQ_FMT_FP8_B128>(L, sm_count, st);
    }
    return cudaErrorInvalidValue;
}

}  // namespace lq
