// A whole mixture-of-experts layer for a few tokens in one cooperative launch (lq_dev_moe_ffn):
//
//   logits[t, e] = x_t . router_e + bias_e; the top_e experts by logit (ties to the lower index), softmax weights
//   out_t = sum_j w_tj * down_j . (silu(gate_j . x_t) * (up_j . x_t))
//
// cpu_moe_forward's route -> experts -> combine (crates/larql-compute/src/cpu/ops/moe/forward.rs:24-140) over dense
// experts (every feature), the router's product included.  Experts are MXFP4, NVFP4 or FP8_B128, gate and up
// [inter, hidden], down [hidden, inter].
//
// What bounds it is reading the chosen experts' weights once.  One CTA per SM walks its share of the work:
//   route    the T x E router products (twice f32's precision: which of two near logits is larger decides a whole
//            expert), spread over the grid; then every CTA picks the experts itself;
//   gate/up  units of 16 features of one expert for one group of its tokens: act = silu(gate) * up, f32, to global;
//   down     units of 32 output rows, as soon as the expert's activations are complete (a counter per group, no
//            grid barrier); when the last unit of all is done, the tokens' results are added up in selection order.
// Warps have three jobs.  A producer streams the units' rows through a ring in shared memory (one tile copy per 16
// rows); it needs only the routing, so it runs ahead from gate/up into down while the activations are still on
// their way.  16 compute warps multiply, each its part of the contraction, and leave their sums in shared memory.
// Finishers add the parts up in a fixed order (results do not depend on timing), apply the activation or the
// routing weight, and publish what they finished of a group when they leave it (a fence and an atomic cost a
// microsecond, as much as a unit's multiplication).
//
// The products run on the tensor cores (mma.sync m16n8k16, f16 x f16 -> f32): weights are the 16 rows of A, tokens the 8
// columns of B.  The codes of all three formats are exact in f16.  An activation is brought to [2^14, 2^15) by a
// power of two per token and held as two f16 terms (22 bits), in both products and for every type; only a bf16 x takes a
// single one, which has all of its bits.  The terms are a column each, or, in a group of more than four tokens, two sets of
// columns multiplied one after the other into the same sums.  Scales: e8m0 (per row and 32) and FP8 blocks multiply the
// f32 sums of 32 products, e4m3 (per row and 16) the f16 codes, which is exact (2 + 4 bits).  (One term between the products of a bf16 layer saves about 5 us in the two cases of several tokens below and keeps
// 11 bits of an activation.)
// Measured: 32 MXFP4 experts of 2880 x 2880, 4 a token: 16 bf16 tokens 107 us for 373 MB, 3.5 TB/s; one f32 token 33 us for
// 53 MB.  64 FP8 experts of 3840 x 800, 6 a token: 37 bf16 tokens 168 us for 576 MB, 3.4 TB/s.  The copies alone take 55, 9
// and 93 us: the compute warps' conversions and latencies bound it (integer pipe 47 %, an instruction in 56 % of the
// cycles, tensor pipe 19 %), and for one token the routing's exchange between the CTAs and the two phases' starts.
// (Tried: e4m3 terms and m16n8k32 e4m3 products, which need no conversion of FP8 codes: that form is converted to f16
// behind the instruction, 32 cycles of a scheduler against 2 x 8.)
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/larql_cuda.h"
#include "codecs.cuh"
#include "kernels.h"
#include "tc5.cuh"

namespace lq {

namespace {

constexpr int ML_WARPS = 16, ML_CONSUMERS = ML_WARPS * 32, ML_FINISH = 3, ML_THREADS = ML_CONSUMERS + 32 * (1 + ML_FINISH);
constexpr int ML_MAX_STAGES = 12;
// A warp's partial sums: 16 rows per column, the upper and lower 8 swapped in every second pair of columns so that the
// lanes of a store (8 rows of four columns 2t) meet in a bank two at most.
__device__ __forceinline__ int red_at(int col, int row) { return col * 16 + (row ^ ((col & 2) << 2)); }

struct MlSmem {
    uint64_t full[ML_MAX_STAGES], empty[ML_MAX_STAGES];
    uint64_t rfull[ML_FINISH], rempty[ML_FINISH];  // partial sums of a unit: written by every compute warp / read
    float2 part[ML_THREADS / 32];
    float unscale[8];           // per token of the group: the power of two its values were divided by
    int gtok[8], gpair[8];      // the group's tokens and (token, slot) pairs
    int n_groups, cnt;
    unsigned x_bits;            // one token: its largest |value|
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

// Eight consecutive elements, loaded first and converted later so that loads of several operands overlap.  WIDE: the
// address is a multiple of 16 bytes.
struct Raw8 {
    uint4 a, b;
};
template <bool WIDE>
__device__ __forceinline__ Raw8 ld8(const void* p, int type, size_t at) {
    Raw8 r;
    if (WIDE) {
        const uint4* q = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) + at * (type == LQ_T_F32 ? 4 : 2));
        r.a = __ldcg(q);
        r.b = type == LQ_T_F32 ? __ldcg(q + 1) : make_uint4(0, 0, 0, 0);
    } else if (type == LQ_T_F32) {
        const uint32_t* q = static_cast<const uint32_t*>(p) + at;
        r.a = make_uint4(q[0], q[1], q[2], q[3]);
        r.b = make_uint4(q[4], q[5], q[6], q[7]);
    } else {
        const uint16_t* q = static_cast<const uint16_t*>(p) + at;
        r.a = make_uint4(q[0] | (uint32_t)q[1] << 16, q[2] | (uint32_t)q[3] << 16, q[4] | (uint32_t)q[5] << 16, q[6] | (uint32_t)q[7] << 16);
        r.b = make_uint4(0, 0, 0, 0);
    }
    return r;
}
__device__ __forceinline__ void to_f32(const Raw8& r, int type, float (&v)[8]) {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
    if (type == LQ_T_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
    } else if (type == LQ_T_BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(ML_CONSUMERS) : "memory"); }

// Bounded polls (about a second): an mbarrier phase, and a counter that other CTAs raise to at least `target`.  The producer
// and the finishers sleep between polls (LAZY): four warps polling flat out took a quarter of the integer pipe's
// cycles from the conversions of the compute warps.
template <bool LAZY>
__device__ __forceinline__ bool ml_wait(uint64_t* bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    for (uint32_t it = 1;; ++it) {
        if (LAZY) __nanosleep(100);
        if (mbar_try_wait(bar, parity)) return true;
        if ((it & 255u) == 0 && clock64() - t0 > (1ll << 31)) return false;
    }
}
__device__ bool wait_count(const unsigned* word, unsigned target) {
    const long long t0 = clock64();
    for (uint32_t it = 1;; ++it) {
        unsigned now;
        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(now) : "l"(word) : "memory");
        if (now >= target) return true;
        if ((it & 255u) == 0 && clock64() - t0 > (1ll << 31)) return false;
    }
}
__device__ __forceinline__ unsigned add_release(unsigned* word, unsigned n) {
    unsigned before;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], %2;" : "=r"(before) : "l"(word), "r"(n) : "memory");
    return before;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_new(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// Four 8 x 16-byte pieces of shared memory, lane l naming row l % 8 of piece l / 8: a lane gets word l % 4 of row l / 4.
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
// Loads by shared-memory address (ordered against the waits, like them volatile).
__device__ __forceinline__ uint32_t lds_u8(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint4 lds_128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
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

// A sum kept as an f32 and its error: products and additions split by the error-free transformations of Dekker and
// Knuth (the dot product of Ogita, Rump and Oishi), as precise as if it were summed in twice f32's precision.
__device__ __forceinline__ float2 pair_add(float2 a, float b) {
    const float s = __fadd_rn(a.x, b), t = __fsub_rn(s, a.x);
    const float e = __fadd_rn(__fsub_rn(a.x, __fsub_rn(s, t)), __fsub_rn(b, t));
    return make_float2(s, __fadd_rn(a.y, e));
}
__device__ __forceinline__ float2 pair_fma(float2 a, float x, float y) {
    const float p = __fmul_rn(x, y), e = __fmaf_rn(x, y, -p);
    a = pair_add(a, p);
    a.y = __fadd_rn(a.y, e);
    return a;
}

// Bytes of `cols` codes, and of a row's scales.
template <int FMT>
__host__ __device__ constexpr int code_bytes(int cols) { return FMT == LQ_FMT_FP8_B128 ? cols : cols / 2; }
template <int FMT>
__host__ __device__ constexpr int row_scale_bytes(int cols) {
    return FMT == LQ_FMT_MXFP4 ? cols / 32 : (FMT == LQ_FMT_NVFP4 ? cols / 16 : 0);
}
// Distance of two columns of the activations: two columns (a phase of a 16-byte load) fall into different banks.
__host__ __device__ constexpr int act_pitch(int k) { return (2 * k) % 128 == 0 ? 2 * k + 64 : 2 * k; }
// Columns per activation of a group of cnt tokens: its terms if eight columns hold them, else one, and the second terms lie
// in a second set of columns.
__host__ __device__ constexpr int group_columns(int cnt, int terms) { return terms == 2 && cnt <= 4 ? 2 : 1; }
__host__ __device__ constexpr int second_set(int cnt, int terms, int pitch) { return terms == 2 && cnt > 4 ? 8 * pitch : 0; }
// Bytes of a group's columns, of one phase or the other.
__host__ __device__ constexpr int act_bytes(int x_terms, int group, int hidden, int inter) {
    const int x = 8 * act_pitch(hidden) + second_set(group, x_terms, act_pitch(hidden));
    const int a = 8 * act_pitch(inter) + second_set(group, 2, act_pitch(inter));
    return x > a ? x : a;
}
// Columns of the contraction per stage: equal parts of at most 46 blocks of 32 (22 for FP8, and for long rows, whose
// activations take most of shared memory), an even number of them.  A stage holds one block more of every row, back to
// back as the tile copy lays them: an odd number of 16-byte pieces per row puts the eight rows of a fragment load into
// different banks (FP8 rows, 32 bytes a block, keep a two-way conflict).
template <int FMT>
__host__ __device__ constexpr int chunk_cols(int k) {
    const int blocks = k / 32, most = FMT == LQ_FMT_FP8_B128 || k > 4096 ? 22 : 46, n = (blocks + most - 1) / most;
    return (((blocks + n - 1) / n + 1) & ~1) * 32;
}
template <int FMT>
__host__ __device__ constexpr int stage_cols(int k) { return chunk_cols<FMT>(k) + 32; }

// One phase's products as the kernel walks them.
struct Walk {
    int k, chunk, n_chunks, pitch;  // contraction, columns per stage, stages per unit, bytes between stage rows
    int units_per_group;            // a unit is two tiles of 16 rows: gate and up, or 32 rows of down
    int is_down;
    int terms;                      // f16 terms per activation
    uint8_t* scales;                // [slots] scales of a unit's rows
    int slots;
    int first, end;                 // this CTA's units
};

template <int FMT>
__device__ __forceinline__ Walk walk_of(const MoeLayer& L, bool down, int n_groups, uint8_t* sbuf) {
    Walk w;
    w.scales = sbuf + (down ? 32 * L.scale_slots[0] * row_scale_bytes<FMT>(L.hidden) : 0);
    w.slots = L.scale_slots[down];
    w.is_down = down;
    w.terms = down ? 2 : L.x_terms;
    w.k = down ? L.inter : L.hidden;
    w.chunk = L.chunk[down];
    w.n_chunks = L.n_chunks[down];
    w.pitch = code_bytes<FMT>(w.chunk + 32);
    // (units of 16 rows of down, which share the load out more evenly, were slower: both tiles take one load of the activations,
    // and the code for one tile costs registers; one bf16 token on 32 MXFP4 experts of 2880 x 2880 33.3 against 31.5 us, 16
    // tokens 126 against 108)
    w.units_per_group = down ? L.hidden / 32 : L.inter / 16;
    // (at most 1024 groups of 512 units, 2^10 CTAs: 32 bits hold the products)
    const unsigned total = (unsigned)(n_groups * w.units_per_group);
    w.first = (int)(total * blockIdx.x / gridDim.x);
    w.end = (int)(total * (blockIdx.x + 1) / gridDim.x);
    return w;
}

// Eight activations times a power of two, into columns of f16: one term, or a value and its rest `rest` bytes on.
template <int FMT>
__device__ __forceinline__ void put_columns(const float (&v)[8], float scale, uint8_t* dst, int rest, int k) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const float x0 = v[2 * q] * scale, x1 = v[2 * q + 1] * scale;
        const __half2 h = __floats2half2_rn(x0, x1);
        const float2 f = __half22float2(h);
        const __half2 l = __floats2half2_rn(x0 - f.x, x1 - f.y);
        hi[q] = *reinterpret_cast<const uint32_t*>(&h);
        lo[q] = *reinterpret_cast<const uint32_t*>(&l);
    }
    if (FMT == LQ_FMT_FP8_B128) {
        // a lane's 8 columns of a block: 4 of either half (what its two code words hold)
        uint8_t* q = dst + 2 * (k & ~31) + ((k & 15) >> 2) * 16 + ((k >> 4) & 1) * 8;
        *reinterpret_cast<uint2*>(q) = make_uint2(hi[0], hi[1]);
        *reinterpret_cast<uint2*>(q + 16) = make_uint2(hi[2], hi[3]);
        if (rest) {
            *reinterpret_cast<uint2*>(q + rest) = make_uint2(lo[0], lo[1]);
            *reinterpret_cast<uint2*>(q + rest + 16) = make_uint2(lo[2], lo[3]);
        }
    } else {
        *reinterpret_cast<uint4*>(dst + 2 * k) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if (rest) *reinterpret_cast<uint4*>(dst + rest + 2 * k) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
}
// The power of two that brings values of at most |bits| to [2^14, 2^15), and the one that takes it back (kept where both
// are normal numbers).  An infinity makes the whole token NaN, like a NaN.
__device__ __forceinline__ float down_scale(uint32_t bits) {
    const int e = min(max((int)(bits >> 23), 15), 254);
    return bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)(127 + 14 + 127 - e) << 23);
}
__device__ __forceinline__ float up_scale(uint32_t bits) {
    return __uint_as_float((uint32_t)(min(max((int)(bits >> 23), 15), 254) - 14) << 23);
}

// Active expert of group gi (groups are numbered expert by expert).
__device__ __forceinline__ int expert_of(const MlSmem& sh, int gi, int from) {
    while (gi >= sh.gpre[from + 1]) ++from;
    return from;
}

// The experts of token t, into shared memory: a warp takes top_e rounds of the largest logit left, the lowest index
// among equals.  Every CTA does it for every token (a publication by one would cost the others a microsecond more).
template <int PER>
__device__ void route_token(const MoeLayer& L, MlSmem& sh, int t, int lane) {
    const int E = L.experts, K = L.top_e;
    uint32_t key[PER];  // logits as integers of the same order; 0: taken (a NaN, 1, comes last: the weights are NaN then)
    float mx = -INFINITY, sum = 0.0f, mine = 0.0f;
    int chosen = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        key[i] = 0;
        if (i * 32 < E && i * 32 + lane < E) {
            const float l = __ldcg(L.logits + (size_t)t * E + i * 32 + lane);
            const uint32_t u = __float_as_uint(l);
            key[i] = l != l ? 1u : ((u & 0x80000000u) ? ~u : (u | 0x80000000u));
        }
    }
    auto value = [](uint32_t k) { return k == 1u ? __uint_as_float(0x7fc00000u) : __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k); };
    for (int j = 0; j < K; ++j) {
        uint32_t best = 0, at = 0xffffffffu;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (i * 32 < E && key[i] > best) {
                best = key[i];
                at = i * 32 + lane;
            }
        const uint32_t top = __reduce_max_sync(0xffffffffu, best);
        const uint32_t e = __reduce_min_sync(0xffffffffu, best == top ? at : 0xffffffffu);
        if (j == 0) {
            mx = value(top);
            if (!L.renormalise) {  // the sum over all experts, before any is taken out
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    if (i * 32 < E && i * 32 + lane < E) sum += expf(value(key[i]) - mx);
            }
        }
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (i * 32 < E && i * 32 + lane == e) key[i] = 0;
        if (j == lane) {
            mine = expf(value(top) - mx);
            chosen = (int)e;
        }
    }
    if (L.renormalise) sum = lane < K ? mine : 0.0f;
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

// SETS: groups may have a second set of columns.
template <int FMT, bool SETS>
__global__ void __launch_bounds__(ML_THREADS, 1) moe_layer_kernel(const __grid_constant__ MoeLayer L) {
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int RED = 8 * 16;  // floats of a warp's partial sums of 16 rows
    MlSmem& sh = *reinterpret_cast<MlSmem*>(smem);
    uint8_t* p = smem + (sizeof(MlSmem) + 127) / 128 * 128;
    float* red = reinterpret_cast<float*>(p);                 // [finish][ML_WARPS][2 tiles][RED]
    p += L.finish * ML_WARPS * 2 * RED * 4;
    uint8_t* xs = p;                                          // a group's columns of f16
    p += act_bytes(L.x_terms, L.group, L.hidden, L.inter);
    uint8_t* sbuf = p;                                        // scales of the units' rows, [scale_slots] per phase
    p += 32 * (L.scale_slots[0] * row_scale_bytes<FMT>(L.hidden) + L.scale_slots[1] * row_scale_bytes<FMT>(L.inter));
    uint8_t* ring = smem + (p - smem + 127) / 128 * 128;      // [n_stages][32 rows]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int T = L.tokens, E = L.experts, K = L.top_e;
    const int TG = L.group;  // tokens per group
    const bool x_wide = (reinterpret_cast<uintptr_t>(L.x) & 15) == 0;  // (rows are multiples of 32 elements)

    if (tid == 0) {
        for (int i = 0; i < L.n_stages; ++i) {
            mbar_init(&sh.full[i], 1);
            mbar_init(&sh.empty[i], ML_WARPS);
        }
        for (int i = 0; i < ML_FINISH; ++i) {
            mbar_init(&sh.rfull[i], ML_WARPS);
            mbar_init(&sh.rempty[i], 1);
        }
        sh.failed = 0;
        sh.x_bits = 0;
        fence_mbar_init();
    }
    for (int i = tid; i < 2 * E; i += ML_THREADS) sh.mask[i >> 1][i & 1] = 0;
    __syncthreads();

    // ---- route: an item is one token's product with one expert's row, worked on by as many warps as there are to spare ----
    {
        constexpr int WARPS = ML_THREADS / 32;
        const int items = T * E;
        const bool r_wide = (reinterpret_cast<uintptr_t>(L.router) & 15) == 0;
        // (1 | 4 | 20 warps an item: 32 items 41 | 35 | 34 us, 256 75 | 69 | 70, 1024 146 | 143 | 149, 4096 215 | 220 | 249)
        const int W = items <= (int)gridDim.x ? WARPS : (items <= 5 * (int)gridDim.x ? 4 : (items <= 10 * (int)gridDim.x ? 2 : 1));
        const int per_cta = WARPS / W, sub = warp / W, part = (warp % W) * 32 + lane;
        const int rounds = (items + (int)gridDim.x * per_cta - 1) / ((int)gridDim.x * per_cta);
        for (int r = 0; r < rounds; ++r) {
            const int it = (r * per_cta + sub) * gridDim.x + blockIdx.x;
            const bool on = it < items && sub < per_cta;  // (warps beyond the last whole item have none)
            const int t = on ? it / E : 0, e = on ? it - t * E : 0;
            float2 s = make_float2(0.0f, 0.0f);
            float m = 0.0f;
            if (on) {
                auto products = [&](auto wide) {
#pragma unroll 2
                    for (int i = part * 8; i < L.hidden; i += W * 256) {
                        const Raw8 rr = ld8<decltype(wide)::value>(L.router, L.router_type, (size_t)e * L.hidden + i);
                        const Raw8 xr = ld8<decltype(wide)::value>(L.x, L.type, (size_t)t * L.hidden + i);
                        float rv[8], xv[8];
                        to_f32(rr, L.router_type, rv);
                        to_f32(xr, L.type, xv);
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            s = pair_fma(s, xv[j], rv[j]);
                            m = fmaxf(m, fabsf(xv[j]));
                        }
                    }
                };
                if (x_wide && r_wide) products(std::true_type{});
                else products(std::false_type{});
                // the token's largest |value|, for its power of two (bits of non-negative floats order as integers)
                if (e == 0) {
                    const unsigned top = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
                    if (lane == 0) atomicMax(L.x_max + t, top);
                }
            }
            auto fold = [&](int from) {
                for (int o = from; o > 0; o >>= 1) {
                    const float ox = __shfl_down_sync(0xffffffffu, s.x, o), oy = __shfl_down_sync(0xffffffffu, s.y, o);
                    s = pair_add(s, ox);
                    s.y = __fadd_rn(s.y, oy);
                }
            };
            fold(16);
            if (W > 1) {
                if (lane == 0) sh.part[warp] = s;
                __syncthreads();
                s = lane < W ? sh.part[sub * W + lane] : make_float2(0.0f, 0.0f);
                if (warp % W == 0) fold(16);
                __syncthreads();
            }
            if (on && warp % W == 0 && lane == 0) {
                if (L.bias) s = pair_add(s, ld_as_f32(L.bias, L.router_type, e));
                // (the errors of a sum that left f32's range, as with a bias of -inf that masks an expert, are NaN)
                L.logits[it] = fabsf(s.x) < INFINITY ? __fadd_rn(s.x, s.y) : s.x;
                add_release(L.route_done, 1u);
            }
        }
        if (T == 1) {
            // one token: every group's activations are the same; make its columns now, while the other CTAs' products arrive
            Raw8 raw[2];
            float v[8];
            uint32_t m = 0;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int k = (tid + q * ML_THREADS) * 8;
                if (k >= L.hidden) continue;
                raw[q] = x_wide ? ld8<true>(L.x, L.type, k) : ld8<false>(L.x, L.type, k);
                to_f32(raw[q], L.type, v);
#pragma unroll
                for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
            }
            m = __reduce_max_sync(0xffffffffu, m);
            if (lane == 0) atomicMax(&sh.x_bits, m);
            __syncthreads();
            const uint32_t bits = sh.x_bits;
            if (tid == 0) sh.unscale[0] = up_scale(bits);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int k = (tid + q * ML_THREADS) * 8;
                if (k >= L.hidden) continue;
                to_f32(raw[q], L.type, v);
                put_columns<FMT>(v, down_scale(bits), xs, L.x_terms == 2 ? act_pitch(L.hidden) : 0, k);
            }
        }
        if (tid == 0 && !wait_count(L.route_done, (unsigned)items)) sh.failed = 1;
    }
    __syncthreads();
    if (sh.failed) {  // no routing to go by: leave (the counters are cleared by the host)
        if (tid == 0) set_err(L.err, DEV_ERR_TMA_TIMEOUT);
        return;
    }
    for (int t = warp; t < T; t += ML_THREADS / 32) {
        if (E <= 32) route_token<1>(L, sh, t, lane);
        else if (E <= 64) route_token<2>(L, sh, t, lane);
        else route_token<MOE_LAYER_MAX_EXPERTS / 32>(L, sh, t, lane);
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
            sh.n_groups = groups;
        }
    }
    __syncthreads();
    const int n_groups = sh.n_groups;

    if (warp == ML_WARPS) {
        // ---- producer: the rows of both phases' units, in order, by one elected thread (behind a branch on the lane each copy takes
        // several times as long: its operands have to be the same in the whole warp) ----
        if (elect_one()) {
            bool ok = true;
            int n = 0, st = 0;  // stages so far, the ring's next place
            uint32_t lap = 0;   // parity of the ring's lap (an empty barrier's first wait, for parity 1, passes)
            for (int ph = 0; ph < 2 && ok; ++ph) {
                const Walk w = walk_of<FMT>(L, ph == 1, n_groups, sbuf);
                const int ua = w.first, ub = w.end;
                if (ua >= ub) continue;
                int gi = ua / w.units_per_group, tile = ua - gi * w.units_per_group, a = -1;
                const CUtensorMap *m0 = nullptr, *m1 = nullptr;
                const uint8_t *sc0 = nullptr, *sc1 = nullptr;
                int slot = 0;
                const uint32_t sbytes16 = 16u * row_scale_bytes<FMT>(w.k), code16 = 16u * w.pitch;
                for (int u = ua; u < ub && ok; ++u) {
                    if (a < 0 || tile == w.units_per_group) {
                        if (a >= 0) ++gi, tile = 0;
                        a = expert_of(sh, gi, max(a, 0));
                        const MoeExpert& ex = L.table[sh.active[a]];
                        m0 = &ex.map[w.is_down ? 2 : 0], m1 = &ex.map[w.is_down ? 2 : 1];
                        tma_acquire_map(m0);
                        if (!w.is_down) tma_acquire_map(m1);
                        sc0 = ex.scales[w.is_down ? 2 : 0], sc1 = ex.scales[w.is_down ? 2 : 1];
                    }
                    const int row0 = tile * (w.is_down ? 32 : 16), row1 = w.is_down ? row0 + 16 : row0;
                    for (int c = 0; c < w.n_chunks; ++c, ++n) {
                        ok = ml_wait<true>(&sh.empty[st], lap ^ 1u);
                        if (!ok) break;
                        // (columns past the row's end arrive as zeros and count as bytes)
                        const bool with_scales = sbytes16 && c == 0;
                        mbar_expect_tx(&sh.full[st], (code16 + (with_scales ? sbytes16 : 0u)) * 2u);
                        uint8_t* dst = ring + (size_t)st * L.stage_bytes;
                        const int x = code_bytes<FMT>(c * w.chunk) / 4;
                        tma_load_2d(dst, m0, x, row0, &sh.full[st]);
                        tma_load_2d(dst + code16, m1, x, row1, &sh.full[st]);
                        if (with_scales) {
                            // the unit's scales come with its first stage.  Their slot is free: the stage this one replaces was
                            // consumed, and scale_slots units do not fit between the two
                            uint8_t* sd = w.scales + slot * 2 * sbytes16;
                            tma_bulk_g2s(sd, sc0 + (size_t)(row0 >> 4) * sbytes16, sbytes16, &sh.full[st]);
                            tma_bulk_g2s(sd + sbytes16, sc1 + (size_t)(row1 >> 4) * sbytes16, sbytes16, &sh.full[st]);
                        }
                        if (++st == L.n_stages) st = 0, lap ^= 1u;
                    }
                    ++tile;
                    if (++slot == w.slots) slot = 0;
                }
            }
            if (!ok) {  // the copies in flight have to land before the block's shared memory goes away
                for (int v = max(0, n - L.n_stages); v < n; ++v) ml_wait<true>(&sh.full[v % L.n_stages], (uint32_t)(v / L.n_stages) & 1u);
                sh.failed = 1;
            }
        }
        __syncwarp();
    } else {
        // ---- compute warps and finishers walk the same units ----
        const bool computes = warp < ML_WARPS;
        const int g = lane >> 2, t4 = lane & 3;
        bool ok = true;  // a wait that ran out is not waited for again; barriers, arrivals and counters are kept
        int st = 0, rb = 0;               // next place of the ring, buffer of the unit's sums
        uint32_t lap = 0, rlap = 0;       // parities of their laps
        for (int ph = 0; ph < 2; ++ph) {
            const Walk w = walk_of<FMT>(L, ph == 1, n_groups, sbuf);
            const int xpitch = act_pitch(w.k), srow = row_scale_bytes<FMT>(w.k);
            const int ua = w.first, ub = w.end;
            if (ua >= ub) continue;
            int gi = ua / w.units_per_group, tile = ua - gi * w.units_per_group, a = expert_of(sh, gi, 0);
            if (!computes) {
                // ---- finishers: every finish-th unit, each with a buffer of its own (it sees all of its phases) ----
                const int buf = warp - ML_WARPS - 1;
                unsigned units = 0, top = 0;  // of this group, not yet published: units, lane i's pair's largest |value|
                int pair = 0;
                auto publish = [&]() {
                    if (units == 0) return;
                    if (!w.is_down && top) atomicMax(L.act_max + pair, top);
                    __threadfence();
                    __syncwarp();
                    if (lane == 0) add_release(w.is_down ? L.down_done : L.group_done + gi, units);
                    units = top = 0;
                };
                for (int u = ua; u < ub; ++u, ++tile) {
                    if (tile == w.units_per_group) {
                        if (!w.is_down) publish();
                        ++gi, tile = 0;
                        a = expert_of(sh, gi, a);
                    }
                    const bool mine = rb == buf;
                    const uint32_t parity = rlap;
                    if (++rb == L.finish) rb = 0, rlap ^= 1u;
                    if (!mine) continue;
                    ++units;
                    const MoeExpert& ex = L.table[sh.active[a]];
                    const float ts0 = ex.ts[w.is_down ? 2 : 0], ts1 = ex.ts[w.is_down ? 2 : 1];
                    if (ok) ok = __all_sync(0xffffffffu, ml_wait<true>(&sh.rfull[buf], parity));
                    const int cnt = sh.cnt;
                    if (lane < cnt) pair = sh.gpair[lane];  // (lane i publishes what belongs to token i of the group)
                    const float* all = red + buf * ML_WARPS * 2 * RED;
                    // a lane takes four rows of one column in both tiles; a token's two terms may lie in two columns
                    const int per = group_columns(cnt, w.terms);
                    const int col = lane >> 2, quad = lane & 3, i = col / per;
                    const bool live = i < cnt && (per == 1 || (col & 1) == 0);
                    const int at = sh.gpair[i < cnt ? i : 0];
                    // (the routing weight goes into the power of two, so that only the weighted output has to be in range)
                    const float scale = sh.unscale[i < cnt ? i : 0] * (w.is_down ? sh.w[at] : 1.0f);
                    auto sums = [&](const float* part, float f) {  // the warps' parts in order
                        const float* from = part + red_at(col, 4 * quad);
                        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                        for (int q = 0; q < ML_WARPS; ++q) {
                            const float4 u = *reinterpret_cast<const float4*>(from + q * 2 * RED);
                            v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
                        }
                        if (per == 2) {
                            v.x += __shfl_xor_sync(0xffffffffu, v.x, 4), v.y += __shfl_xor_sync(0xffffffffu, v.y, 4);
                            v.z += __shfl_xor_sync(0xffffffffu, v.z, 4), v.w += __shfl_xor_sync(0xffffffffu, v.w, 4);
                        }
                        return make_float4(v.x * scale * f, v.y * scale * f, v.z * scale * f, v.w * scale * f);
                    };
                    const float4 a0 = sums(all, ts0), a1 = sums(all + RED, ts1);
                    if (!w.is_down) {
                        auto silu = [](float g, float u) { return g / (1.0f + expf(-g)) * u; };
                        const float4 act = make_float4(silu(a0.x, a1.x), silu(a0.y, a1.y), silu(a0.z, a1.z), silu(a0.w, a1.w));
                        if (live) __stcg(reinterpret_cast<float4*>(L.act + (size_t)at * L.inter + tile * 16 + 4 * quad), act);
                        // the pairs' largest |value| (a NaN's bits are above every number's)
                        auto bits = [](float v) { return __float_as_uint(v) & 0x7fffffffu; };
                        unsigned m = max(max(bits(act.x), bits(act.y)), max(bits(act.z), bits(act.w)));
                        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
                        m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
                        const unsigned mine = __shfl_sync(0xffffffffu, m, lane * per * 4 & 31);
                        if (lane < cnt) top = max(top, mine);  // (columns past the group hold anything)
                    } else if (live) {
                        float* o = L.pair_out + (size_t)at * L.hidden + tile * 32 + 4 * quad;
                        __stcg(reinterpret_cast<float4*>(o), a0);
                        __stcg(reinterpret_cast<float4*>(o + 16), a1);
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive_one(&sh.rempty[buf]);
                }
                publish();
                continue;
            }
            // A compute warp takes every 16th block of the contraction, of both tiles.
            constexpr bool F8 = FMT == LQ_FMT_FP8_B128;
            const int tile2 = 16 * w.pitch, scale2 = 16 * srow;
            int cur = -1, slot = 0;
            uint32_t rest = 0;  // distance of the second set of columns (0: there is none)
            for (int u = ua; u < ub; ++u, ++tile) {
                if (tile == w.units_per_group) {
                    ++gi, tile = 0;
                    a = expert_of(sh, gi, a);
                }
                const int e = sh.active[a];
                if (gi != cur) {
                    // the group's tokens: which they are, and their activations as columns of f16
                    cur = gi;
                    const int first = (gi - sh.gpre[a]) * TG;
                    const unsigned long long m0 = sh.mask[e][0] | ((unsigned long long)sh.mask[e][1] << 32);
                    const int cnt = min(TG, __popcll(m0) - first);
                    const int columns = group_columns(cnt, w.terms);
                    if (SETS) rest = second_set(cnt, w.terms, xpitch);
                    // the finishers are done with the previous group's units, the compute warps with its activations
                    for (int v = 0; v < L.finish; ++v)
                        if (ok) ok = __all_sync(0xffffffffu, ml_wait<false>(&sh.rempty[v], v < rb ? rlap : rlap ^ 1u));
                    consumers_sync();
                    if (tid < cnt) {
                        unsigned long long m = m0;
                        for (int i = 0; i < first + tid; ++i) m &= m - 1;
                        const int t = __ffsll((long long)m) - 1;
                        int j = 0;
                        while (sh.idx[t * K + j] != e) ++j;
                        sh.gtok[tid] = t;
                        sh.gpair[tid] = t * K + j;
                        sh.cnt = cnt;
                    }
                    // down: the activations of the whole group, from every CTA that made some of them
                    if (w.is_down && tid == 0 && ok && !wait_count(L.group_done + gi, (unsigned)(L.inter / 16))) sh.failed = 1;
                    consumers_sync();
                    // the warps share the rows out: `per` warps a token
                    const int per = cnt >= 5 ? 2 : (cnt >= 3 ? 4 : (cnt == 2 ? 8 : 16));
                    const int i = warp / per, part = (warp % per) * 32 + lane;
                    if (i < cnt && !(T == 1 && ph == 0)) {  // (a single token's columns were made while the routing was on its way)
                        const void* src = w.is_down ? L.act : L.x;
                        const int type = w.is_down ? LQ_T_F32 : L.type;
                        const bool wide = w.is_down || x_wide;
                        const size_t row = (size_t)(w.is_down ? sh.gpair[i] : sh.gtok[i]) * w.k;
                        auto fetch = [&](int k) { return wide ? ld8<true>(src, type, row + k) : ld8<false>(src, type, row + k); };
                        Raw8 next[2];  // (on their way while the largest value is looked up)
#pragma unroll
                        for (int q = 0; q < 2; ++q)
                            if (part * 8 + q * per * 256 < w.k) next[q] = fetch(part * 8 + q * per * 256);
                        const unsigned bits = __ldcg(w.is_down ? L.act_max + sh.gpair[i] : L.x_max + sh.gtok[i]);
                        const float scale = down_scale(bits);
                        if (part == 0) sh.unscale[i] = up_scale(bits);
                        for (int k = part * 8; k < w.k; k += per * 256) {
                            float v[8];
                            to_f32(next[0], type, v);
                            next[0] = next[1];
                            if (k + per * 512 < w.k) next[1] = fetch(k + per * 512);
                            put_columns<FMT>(v, scale, xs + (size_t)(i * columns) * xpitch, columns == 2 ? xpitch : (int)rest, k);
                        }
                    }
                    consumers_sync();
                }
                float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, acc2[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                const uint32_t s0 = smem_u32(w.scales) + (uint32_t)(slot * 32 * srow + g * srow);
                const float *fs = nullptr, *fs2 = nullptr;
                if (F8) {
                    const int row_blocks = (w.k + 127) >> 7, row = tile * (w.is_down ? 32 : 16);
                    fs = reinterpret_cast<const float*>(L.table[e].scales[w.is_down ? 2 : 0]) + (size_t)(row >> 7) * row_blocks;
                    // (32 rows of a down unit start at a multiple of 32: one row of scale blocks)
                    fs2 = w.is_down ? fs : reinterpret_cast<const float*>(L.table[e].scales[1]) + (size_t)(row >> 7) * row_blocks;
                }
                // fragment rows: FP4: lanes 0-15 name the rows of the first tile, 16-31 those of the second; FP8: the halves
                // of a block
                const uint32_t frag = smem_u32(ring) + (uint32_t)((lane & 15) * w.pitch + (lane >> 4) * (F8 ? 16 : tile2));
                const uint32_t xcol = smem_u32(xs) + (uint32_t)(g * xpitch + t4 * 16);
                if (++slot == w.slots) slot = 0;
                for (int c = 0; c < w.n_chunks; ++c) {
                    const int kb0 = c * (w.chunk / 32), blocks = min(w.chunk / 32, w.k / 32 - kb0);
                    if (ok) ok = __all_sync(0xffffffffu, ml_wait<false>(&sh.full[st], lap));
                    // addresses of the warp's first block; the others lie at constant distances
                    const uint32_t ra = frag + (uint32_t)(st * L.stage_bytes + warp * (F8 ? 32 : 16));
                    const uint32_t sa = s0 + (FMT == LQ_FMT_NVFP4 ? 2 * (kb0 + warp) + (t4 >> 1) : kb0 + warp), sb = sa + 8 * srow;
                    const uint32_t sc = sa + scale2, sd = sc + 8 * srow;
                    const uint32_t xa = xcol + (uint32_t)((kb0 + warp) * 64);
                    // one step: block warp + at of both tiles, with the second set of columns (SECOND)
                    auto step = [&](auto second_tag, int at) {
                        constexpr bool SECOND = decltype(second_tag)::value;
                        // lo and hi: the f16 pairs of rows g and g + 8 of the first and the second tile
                        uint32_t lo[2][4], hi[2][4];
                        float f0[2] = {0.0f, 0.0f}, f1[2] = {0.0f, 0.0f};
                        if (F8) {
                            uint32_t r[2][4];
                            ldmatrix4(r[0], ra + at * 32);
                            ldmatrix4(r[1], ra + tile2 + at * 32);
                            f0[0] = f1[0] = __ldg(fs + ((kb0 + warp + at) >> 2));
                            f0[1] = f1[1] = __ldg(fs2 + ((kb0 + warp + at) >> 2));
#pragma unroll
                            for (int q = 0; q < 2; ++q) {
                                lo[q][0] = e4m3x2_f16(r[q][0]), lo[q][1] = e4m3x2_f16(r[q][0] >> 16);
                                lo[q][2] = e4m3x2_f16(r[q][2]), lo[q][3] = e4m3x2_f16(r[q][2] >> 16);
                                hi[q][0] = e4m3x2_f16(r[q][1]), hi[q][1] = e4m3x2_f16(r[q][1] >> 16);
                                hi[q][2] = e4m3x2_f16(r[q][3]), hi[q][3] = e4m3x2_f16(r[q][3] >> 16);
                            }
                        } else {
                            constexpr int SB = FMT == LQ_FMT_NVFP4 ? 2 : 1;  // scales per block
                            uint32_t r[4];
                            ldmatrix4(r, ra + at * 16);
                            const uint32_t u[4] = {lds_u8(sa + at * SB), lds_u8(sb + at * SB), lds_u8(sc + at * SB), lds_u8(sd + at * SB)};
                            if (FMT == LQ_FMT_MXFP4) {
                                // 2^(byte - 127), 0 for 0 (e8m0_to_f32; a NaN scale was refused when the layer was made)
                                f0[0] = __uint_as_float(u[0] << 23), f1[0] = __uint_as_float(u[1] << 23);
                                f0[1] = __uint_as_float(u[2] << 23), f1[1] = __uint_as_float(u[3] << 23);
                            }
#pragma unroll
                            for (int q = 0; q < 2; ++q) {
                                e2m1x8(r[2 * q], lo[q]);
                                e2m1x8(r[2 * q + 1], hi[q]);
                                if (FMT == LQ_FMT_NVFP4) {
                                    const uint32_t m0 = e4m3x2_f16(u[2 * q] | (u[2 * q] << 8)), m1 = e4m3x2_f16(u[2 * q + 1] | (u[2 * q + 1] << 8));
#pragma unroll
                                    for (int i = 0; i < 4; ++i) {
                                        lo[q][i] = mul_f16x2(lo[q][i], m0);
                                        hi[q][i] = mul_f16x2(hi[q][i], m1);
                                    }
                                }
                            }
                        }
                        const uint32_t xj = xa + at * 64;
                        const uint4 x = lds_128(xj);
                        if (FMT == LQ_FMT_NVFP4) {
                            mma_f16(acc, lo[0][0], hi[0][0], lo[0][1], hi[0][1], x.x, x.y);
                            mma_f16(acc2, lo[1][0], hi[1][0], lo[1][1], hi[1][1], x.x, x.y);
                            mma_f16(acc, lo[0][2], hi[0][2], lo[0][3], hi[0][3], x.z, x.w);
                            mma_f16(acc2, lo[1][2], hi[1][2], lo[1][3], hi[1][3], x.z, x.w);
                            if (SECOND) {
                                const uint4 y = lds_128(xj + rest);
                                mma_f16(acc, lo[0][0], hi[0][0], lo[0][1], hi[0][1], y.x, y.y);
                                mma_f16(acc2, lo[1][0], hi[1][0], lo[1][1], hi[1][1], y.x, y.y);
                                mma_f16(acc, lo[0][2], hi[0][2], lo[0][3], hi[0][3], y.z, y.w);
                                mma_f16(acc2, lo[1][2], hi[1][2], lo[1][3], hi[1][3], y.z, y.w);
                            }
                        } else {
                            float d[4], h[4];
                            mma_f16_new(d, lo[0][0], hi[0][0], lo[0][1], hi[0][1], x.x, x.y);
                            mma_f16_new(h, lo[1][0], hi[1][0], lo[1][1], hi[1][1], x.x, x.y);
                            mma_f16(d, lo[0][2], hi[0][2], lo[0][3], hi[0][3], x.z, x.w);
                            mma_f16(h, lo[1][2], hi[1][2], lo[1][3], hi[1][3], x.z, x.w);
                            if (SECOND) {
                                const uint4 y = lds_128(xj + rest);
                                mma_f16(d, lo[0][0], hi[0][0], lo[0][1], hi[0][1], y.x, y.y);
                                mma_f16(h, lo[1][0], hi[1][0], lo[1][1], hi[1][1], y.x, y.y);
                                mma_f16(d, lo[0][2], hi[0][2], lo[0][3], hi[0][3], y.z, y.w);
                                mma_f16(h, lo[1][2], hi[1][2], lo[1][3], hi[1][3], y.z, y.w);
                            }
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                acc[q] = fmaf(d[q], q < 2 ? f0[0] : f1[0], acc[q]);
                                acc2[q] = fmaf(h[q], q < 2 ? f0[1] : f1[1], acc2[q]);
                            }
                        }
                    };
                    const int left = blocks - warp;  // (at most 46 blocks a stage, 22 for FP8)
                    auto steps = [&](auto second) {
#pragma unroll
                        for (int i = 0; i < (F8 ? 2 : 3); ++i)
                            if (i * ML_WARPS < left) step(second, i * ML_WARPS);
                    };
                    // (apart: a branch inside a step would keep it from overlapping with the next)
                    if (SETS && rest) steps(std::integral_constant<bool, SETS>{});
                    else steps(std::false_type{});
                    __syncwarp();
                    if (lane == 0) mbar_arrive_one(&sh.empty[st]);
                    if (++st == L.n_stages) st = 0, lap ^= 1u;
                }
                if (ok) ok = __all_sync(0xffffffffu, ml_wait<false>(&sh.rempty[rb], rlap ^ 1u));
                float* mine = red + (rb * ML_WARPS + warp) * 2 * RED;
                const int col = 2 * t4, at[4] = {red_at(col, g), red_at(col + 1, g), red_at(col, g + 8), red_at(col + 1, g + 8)};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    mine[at[q]] = acc[q];
                    mine[RED + at[q]] = acc2[q];
                }
                __syncwarp();
                if (lane == 0) mbar_arrive_one(&sh.rfull[rb]);
                if (++rb == L.finish) rb = 0, rlap ^= 1u;
            }
        }
        if (!ok && lane == 0) sh.failed = 1;
    }
    // ---- the tokens' results, when every unit of every CTA is there ----
    const int n_units = n_groups * walk_of<FMT>(L, true, n_groups, sbuf).units_per_group;
    if (tid == 0 && !wait_count(L.down_done, (unsigned)n_units)) sh.failed = 1;
    __syncthreads();
    for (int i = blockIdx.x * ML_THREADS + tid; i < T * (L.hidden / 4); i += gridDim.x * ML_THREADS) {
        const int t = i / (L.hidden / 4), h = (i - t * (L.hidden / 4)) * 4;
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int j = 0; j < K; ++j) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(L.pair_out + (size_t)(t * K + j) * L.hidden + h));
            s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
        }
        const size_t at = (size_t)t * L.hidden + h;
        const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (L.type == LQ_T_F32) static_cast<float*>(L.out)[at + q] = v[q];
            else if (L.type == LQ_T_BF16) static_cast<__nv_bfloat16*>(L.out)[at + q] = __float2bfloat16_rn(v[q]);
            else static_cast<__half*>(L.out)[at + q] = __float2half_rn(v[q]);
        }
    }
    __syncthreads();
    if (tid == 0) {
        if (sh.failed) set_err(L.err, DEV_ERR_TMA_TIMEOUT);
        __threadfence();
        sh.failed = add_release(L.exits, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (sh.failed) {  // the last CTA: nobody waits any more, the words are zeroed for the next launch
        for (int i = tid; i < MOE_LAYER_SYNC_WORDS; i += ML_THREADS) L.exits[i] = 0;
    }
}

// Shared memory beside the ring and the scales, a unit's scales, a stage.
size_t fixed_smem(int finish, int x_terms, int group, int hidden, int inter) {
    return 128 + (sizeof(MlSmem) + 127) / 128 * 128 + finish * (size_t)ML_WARPS * 2 * 8 * 16 * 4 +
           (size_t)act_bytes(x_terms, group, hidden, inter);
}
template <int FMT>
int stage_size(int hidden, int inter) {
    return 32 * std::max(code_bytes<FMT>(stage_cols<FMT>(hidden)), code_bytes<FMT>(stage_cols<FMT>(inter)));
}
// How shared memory is dealt out.
struct Plan {
    int stages, finish;  // of the ring; finishers at work (a buffer of partial sums each)
    int slots[2];        // scales of units, per phase
    size_t bytes;
};
// The most stages that fit, with fewer finishers where that leaves under three.  Between a unit's first stage and the stage it
// replaces lie at most stages / chunks units of a phase: so many slots its scales need, and one.
template <int FMT>
Plan plan_ring(int x_terms, int group, int hidden, int inter) {
    auto chunks = [](int k) { return (k + chunk_cols<FMT>(k) - 1) / chunk_cols<FMT>(k); };
    Plan p = {};
    for (int finish = ML_FINISH; finish >= 1; --finish) {
        for (int n = ML_MAX_STAGES; n >= 2; --n) {
            const int slots[2] = {(n + chunks(hidden) - 1) / chunks(hidden) + 1, (n + chunks(inter) - 1) / chunks(inter) + 1};
            const size_t scales = 32 * ((size_t)slots[0] * row_scale_bytes<FMT>(hidden) + (size_t)slots[1] * row_scale_bytes<FMT>(inter));
            const size_t bytes = fixed_smem(finish, x_terms, group, hidden, inter) + scales + (size_t)n * stage_size<FMT>(hidden, inter);
            if (bytes <= 227 * 1024) {
                if (n > p.stages) p = Plan{n, finish, {slots[0], slots[1]}, bytes};
                break;
            }
        }
        if (p.stages >= 3) break;
    }
    return p;
}

template <int FMT, bool SETS>
cudaError_t launch_layer(MoeLayer L, int sm_count, cudaStream_t st) {
    const Plan p = plan_ring<FMT>(L.x_terms, L.group, L.hidden, L.inter);
    if (p.stages == 0) return cudaErrorInvalidConfiguration;
    L.n_stages = p.stages, L.finish = p.finish, L.scale_slots[0] = p.slots[0], L.scale_slots[1] = p.slots[1];
    L.stage_bytes = stage_size<FMT>(L.hidden, L.inter);
    for (int i = 0; i < 2; ++i) {
        const int k = i ? L.inter : L.hidden;
        L.chunk[i] = chunk_cols<FMT>(k);
        L.n_chunks[i] = (k + L.chunk[i] - 1) / L.chunk[i];
    }
    const void* fn = (const void*)moe_layer_kernel<FMT, SETS>;
    cudaError_t e = set_max_dyn_smem(fn, 227 * 1024);
    if (e != cudaSuccess) return e;
    void* args[] = {&L};
    return cudaLaunchCooperativeKernel(fn, dim3(sm_count), dim3(ML_THREADS), args, p.bytes, st);
}

template <int FMT>
cudaError_t launch_fmt(MoeLayer L, int sm_count, cudaStream_t st) {
    L.x_terms = L.type == LQ_T_BF16 ? 1 : 2;
    // An expert with more tokens than a group holds is read once per group; a second set of columns doubles a group's products,
    // a bf16 layer's behind gate/up only.  Groups of 8 instead of 4 tokens by the tokens an expert is likely to have, where
    // shared memory takes the second set.  Measured with 4 | 8, 32 MXFP4 experts of 2880 x 2880, 4 a token: bf16, 16 tokens
    // 107 | 114 us, 24 135 | 132, 32 150 | 138; f32, 24 tokens 136 | 144, 32 151 | 151, 64 241 | 204; 64 FP8 experts of
    // 3840 x 800, 6 a token, 37 tokens: bf16 186 | 173, f32 189 | 195.
    const bool many = 2 * L.tokens * L.top_e > (L.x_terms == 1 ? 5 : 7) * L.experts && L.tokens > 4;
    L.group = 8;
    if (many && plan_ring<FMT>(L.x_terms, L.group, L.hidden, L.inter).stages > 0)
        return launch_layer<FMT, true>(L, sm_count, st);
    L.group = 4;
    return launch_layer<FMT, false>(L, sm_count, st);
}

}  // namespace

template <int FMT>
static bool fits(int hidden, int inter) {
    return plan_ring<FMT>(2, 4, hidden, inter).stages > 0;
}
bool moe_layer_supported(int fmt, int hidden, int inter) {
    if (hidden <= 0 || inter <= 0 || hidden % 32 || inter % 32 || hidden > 8192 || inter > 8192) return false;
    if (fmt == LQ_FMT_NVFP4 && (hidden > 6144 || inter > 6144)) return false;
    switch (fmt) {
        case LQ_FMT_MXFP4: return fits<LQ_FMT_MXFP4>(hidden, inter);
        case LQ_FMT_NVFP4: return fits<LQ_FMT_NVFP4>(hidden, inter);
        case LQ_FMT_FP8_B128: return fits<LQ_FMT_FP8_B128>(hidden, inter);
    }
    return false;
}

// Whether any e8m0 scale of the layer is 255, a NaN: block (expert, matrix) looks through that matrix's scales.
__global__ void moe_nan_scale_kernel(const MoeExpert* table, int hidden, int inter, int* found) {
    const size_t n = (size_t)hidden * inter / 32 / 16;  // (rows and columns are multiples of 32)
    const uint4* s = reinterpret_cast<const uint4*>(table[blockIdx.x].scales[blockIdx.y]);
    unsigned bad = 0;
    for (size_t i = threadIdx.x; i < n; i += blockDim.x) {
        const uint4 v = s[i];
        bad |= __vcmpeq4(v.x, 0xffffffffu) | __vcmpeq4(v.y, 0xffffffffu) | __vcmpeq4(v.z, 0xffffffffu) | __vcmpeq4(v.w, 0xffffffffu);
    }
    if (bad) *found = 1;
}
cudaError_t launch_moe_nan_scale(const MoeExpert* table, int experts, int hidden, int inter, int* found, cudaStream_t st) {
    moe_nan_scale_kernel<<<dim3(experts, 3), 512, 0, st>>>(table, hidden, inter, found);
    return cudaGetLastError();
}

template <int FMT>
static cudaError_t encode_maps(MoeExpert* ex, int hidden, int inter) {
    for (int i = 0; i < 3; ++i) {
        const size_t rows = i == 2 ? hidden : inter, bytes = (size_t)code_bytes<FMT>(i == 2 ? inter : hidden);
        const cudaError_t e = encode_tile_map(&ex->map[i], CU_TENSOR_MAP_DATA_TYPE_UINT32, ex->codes[i], rows, bytes / 4, bytes, 16,
                                              code_bytes<FMT>(stage_cols<FMT>(i == 2 ? inter : hidden)) / 4, CU_TENSOR_MAP_SWIZZLE_NONE);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}
cudaError_t moe_encode_maps(int fmt, MoeExpert* ex, int hidden, int inter) {
    switch (fmt) {
        case LQ_FMT_MXFP4: return encode_maps<LQ_FMT_MXFP4>(ex, hidden, inter);
        case LQ_FMT_NVFP4: return encode_maps<LQ_FMT_NVFP4>(ex, hidden, inter);
        case LQ_FMT_FP8_B128: return encode_maps<LQ_FMT_FP8_B128>(ex, hidden, inter);
    }
    return cudaErrorInvalidValue;
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
