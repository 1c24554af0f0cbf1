// Matrix product in 8-bit floating point with one scale per block of 128 (lq_dev_fp8_matmul), and the quantisation
// of its activations (lq_dev_fp8_quantize):
//
//   out[t, r] = sum_b sx[t, b] * sw[r / 128, b] * sum_{k in block b} qx[t, k] * qw[r, k]
//
// with qx, qw in e4m3, sx one f32 per token and 128 columns, sw one f32 per 128 x 128 block of the weight.  The
// scales change along the contraction, so a block's 128-long partial product (four K = 32 steps of tcgen05.mma
// kind::f8f6f4, f32 accumulators in tensor memory) is read back, multiplied by its scale and added to an f32
// accumulator in registers, while the tensor core works on the next block in another accumulator buffer.  The
// products are exact, their sum over a block is held in f32 with the tensor core's rounding (they span 2^-18 to 2^18); the
// two scales' product is rounded to f32, and a block's sum enters by one f32 fused multiply-add.
//
// Two kernels, chosen by estimates of their time (way_of has the rule and what both measured):
//   fp8_few_kernel    rows of the weight are the 128 lanes of an accumulator, tokens its 16, 32 or 64 columns.  What
//                     bounds it is reading the weight, so the (row tile, k block) units are dealt out evenly over
//                     the SMs in one contiguous run each, and tiles that end inside a run are joined through a
//                     workspace by the last CTA to finish its piece, always in the order of k: results do not
//                     depend on timing.
//   fp8_many_kernel   tokens are the lanes, 256 rows of the weight the columns: the scale of a lane and block is one
//                     number per thread, one fused multiply-add per value.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "../../include/larql_cuda.h"
#include "kernels.h"
#include "tc5.cuh"

namespace lq {

namespace {

constexpr float F8_MAX = 448.0f;
constexpr float F8_MIN_SCALE = 1.17549435e-38f;  // 2^-126: a zero block gets a scale too

__device__ __forceinline__ float ld_f32(const float* p) { return *p; }
__device__ __forceinline__ float ld_f32(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float ld_f32(const __half* p) { return __half2float(*p); }

__device__ __forceinline__ float max_nan(float a, float b) {  // a NaN wins: it must reach the scale
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// The correctly rounded quotient x / s, from r = 1 / s correctly rounded: a product, its exact remainder, one correction
// (Markstein's theorem).  Valid where no step under- or overflows; quotients below 2^-10 may be off, their code is 0
// either way.
__device__ __forceinline__ float quotient(float x, float s, float r) {
    const float q = __fmul_rn(x, r);
    return __fmaf_rn(__fmaf_rn(-q, s, x), r, q);
}
// Minus the quotients of two elements, two f32 an instruction: with the signs this way round the correction keeps a zero's
// (x = -0: +0; q itself would lose it).
__device__ __forceinline__ float2 minus_quotients(float x0, float x1, float s, float r) {
    float2 n;
    asm("{\n\t.reg .b64 x, s, r, q, e;\n\t"
        "mov.b64 x, {%2, %3};\n\tmov.b64 s, {%4, %4};\n\tmov.b64 r, {%5, %5};\n\t"
        "mul.rn.f32x2 q, x, r;\n\tfma.rn.f32x2 e, q, s, x;\n\tfma.rn.f32x2 q, e, r, q;\n\t"
        "mov.b64 {%0, %1}, q;\n\t}"
        : "=f"(n.x), "=f"(n.y)
        : "f"(x0), "f"(x1), "f"(s), "f"(-r));
    return n;
}

// Eight consecutive elements as they lie, their conversion, and the bits of their largest |value| as an f32 (as integers:
// a NaN's are above every number's).
template <class T>
struct Eight {
    uint4 a, b;
};
template <class T, bool VEC>
__device__ __forceinline__ Eight<T> load8(const T* p, int n) {
    Eight<T> r;
    r.a = r.b = make_uint4(0, 0, 0, 0);
    if (VEC) {
        r.a = __ldg(reinterpret_cast<const uint4*>(p));
        if (sizeof(T) == 4) r.b = __ldg(reinterpret_cast<const uint4*>(p) + 1);
    } else {
        T v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : T(0.0f);
        memcpy(&r.a, v, 16);
        if (sizeof(T) == 4) memcpy(&r.b, reinterpret_cast<const uint8_t*>(v) + sizeof(T) * 8 - 16, 16);
    }
    return r;
}
template <class T>
__device__ __forceinline__ void values8(const Eight<T>& r, float (&v)[8]) {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (std::is_same<T, float>::value) v[i] = __uint_as_float(w[i]);
        else if (std::is_same<T, __nv_bfloat16>::value) v[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        else v[i] = __half2float(__ushort_as_half((unsigned short)(w[i / 2] >> (16 * (i & 1)))));
    }
}
// Largest |value| of a block of 128, 16 threads' eights: 16-bit types two at a time as integers of the same order.
template <class T>
__device__ __forceinline__ float block_amax(const Eight<T>& r) {
    if (std::is_same<T, float>::value) {
        const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7fffffffu);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        return __uint_as_float(m);
    }
    uint32_t m = __vmaxu2(__vmaxu2(r.a.x & 0x7fff7fffu, r.a.y & 0x7fff7fffu), __vmaxu2(r.a.z & 0x7fff7fffu, r.a.w & 0x7fff7fffu));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
    m = max(m >> 16, m & 0xffffu);
    return std::is_same<T, __nv_bfloat16>::value ? __uint_as_float(m << 16) : __half2float(__ushort_as_half((unsigned short)m));
}

// n / d for n below 2^30 and d below 2^24 by a multiplication: m = ceil(2^(32 + s) / d) with 2^s <= d is off by less than d of
// 2^(32 + s), and n times that stays below 2^(32 + s).
struct Divisor {
    uint32_t m, s;  // m 0: d is 1
    static Divisor make(uint32_t d) {
        if (d == 1) return Divisor{0, 0};
        uint32_t s = 31 - __builtin_clz(d);
        if ((d & (d - 1)) == 0) --s;  // (2^(32 + s) / d has to fit 32 bits)
        return Divisor{(uint32_t)(((1ull << (32 + s)) + d - 1) / d), s};
    }
    __device__ __forceinline__ int of(int n) const { return m ? (int)(__umulhi((uint32_t)n, m) >> s) : n; }
};

// 16 threads per (token, block of 128), 8 consecutive elements each; QU such blocks are on their way at a time (1 where
// there are few, else 2: 4096 x 8192 bf16 23.6 us, with 4 1.4 more, with 8 9).  The quotients are the correctly rounded ones
// (and not x times 1 / s): the codes are defined by them, and the tests hold them to the definition bit for bit.
// Instructions bound it, about 135 for a thread's eight elements: 4.3 TB/s of the 102 MB it reads and writes.
template <class T, bool VEC, int QU>
__global__ void __launch_bounds__(256) fp8_quantize_kernel(const T* __restrict__ x, long long x_stride, int units, int kb_n,
                                                           int cols, uint8_t* __restrict__ codes, long long code_pitch,
                                                           float* __restrict__ scales, int wide_store, Divisor by_kb) {
    pdl_wait();  // (before the next kernel may start: what it reads early was complete when this one began)
    pdl_launch_next();
    const int sub = threadIdx.x & 15;
    for (int u0 = blockIdx.x * (16 * QU); u0 < units; u0 += gridDim.x * (16 * QU)) {
        Eight<T> r[QU];
        int t[QU], kb[QU];
        const int first = u0 + (threadIdx.x >> 4);
        t[0] = by_kb.of(first);
        kb[0] = first - t[0] * kb_n;
#pragma unroll
        for (int n = 0; n < QU; ++n) {
            if (n) {  // 16 blocks on
                t[n] = t[n - 1], kb[n] = kb[n - 1] + 16;
                while (kb[n] >= kb_n) kb[n] -= kb_n, ++t[n];
            }
            const int k0 = kb[n] * 128 + sub * 8;
            r[n].a = r[n].b = make_uint4(0, 0, 0, 0);
            if (first + n * 16 < units && k0 < cols) r[n] = load8<T, VEC>(x + t[n] * x_stride + k0, cols - k0);
        }
#pragma unroll
        for (int n = 0; n < QU; ++n) {
            const float m = block_amax(r[n]);
            float v[8], s;
            values8(r[n], v);
            uint32_t w[4], flip = 0;
            if (m > 0x1p-90f && m < 0x1p100f) {
                s = quotient(m, F8_MAX, 1.0f / F8_MAX);  // (a constant, correctly rounded)
                const float inv = __frcp_rn(s);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 n = minus_quotients(v[2 * i], v[2 * i + 1], s, inv);
                    w[i] = e4m3x2(n.x, n.y);
                }
                flip = 0x80808080u;
            } else {  // zero, tiny, huge, infinite or NaN
                s = max_nan(__fdiv_rn(m, F8_MAX), F8_MIN_SCALE);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = e4m3x2(__fdiv_rn(v[2 * i], s), __fdiv_rn(v[2 * i + 1], s));
            }
            const int k0 = kb[n] * 128 + sub * 8;
            if (first + n * 16 >= units || k0 >= cols) continue;
            if (sub == 0) scales[(size_t)t[n] * kb_n + kb[n]] = s;
            uint8_t* q = codes + t[n] * code_pitch + k0;
            if (wide_store) {  // cols (and the pitch) are multiples of 8
                *reinterpret_cast<uint2*>(q) = make_uint2((w[0] | (w[1] << 16)) ^ flip, (w[2] | (w[3] << 16)) ^ flip);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (k0 + i < cols) q[i] = (uint8_t)((w[i >> 1] ^ flip) >> (8 * (i & 1)));
            }
        }
    }
}

template <class T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ void store_as(void* out, int type, size_t at, float v) {
    if (type == LQ_T_F32) static_cast<float*>(out)[at] = v;
    else if (type == LQ_T_BF16) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
    else static_cast<__half*>(out)[at] = __float2half_rn(v);
}

// What both kernels are told.
struct F8Args {
    const float* sx;   // [tokens][kb_n]
    const float* sw;   // [ceil(rows / 128)][kb_n]
    void* out;
    long long out_stride;
    int out_type;
    int tokens, rows, kb_n;
    int whole;         // few-token kernel: a CTA's run is whole tiles (nothing to join)
    int chained;       // the kernel before this one on the stream is the tokens' quantisation
    float* part;       // few-token kernel: [grid][2][NT][128] partial tiles
    unsigned* done;    // few-token kernel: k blocks finished per tile (zero between launches)
    int* err;
};

// ------------------------------------------------------------ few tokens ----
// What bounds it: with every SM at work the memory (16 tokens x 28672 -> 8192, 237 MB: 50 us with the quantisation, 4.7
// TB/s); with less than a tile per SM the thread that issues the tensor-core instructions, 0.23 us per block of 16 columns
// (250 x 2880 -> 2880: 13 us with the quantisation).  That thread and the loading one loop inside elect.sync's branch:
// behind a branch on the lane every instruction takes several times as long (0.30 us a block).
constexpr int few_stage_bytes(int nt) { return 128 * 128 + nt * 128; }
constexpr int few_stages(int nt) { return nt == 16 ? 11 : (nt == 32 ? 10 : 8); }  // (an accumulator of nt columns each)
constexpr int few_promo_warps(int nt) { return nt / 4; }  // 16 columns a warp
constexpr int few_threads(int nt) { return 128 + 32 * few_promo_warps(nt); }  // (two warps idle: a warp reads the TMEM lanes of its rank of 4)

template <int NT>
struct FewSmem {
    // a stage is its tiles and its accumulator: loaded (full), multiplied (done), added up by every promoting warp (empty)
    uint64_t full[few_stages(NT)], done[few_stages(NT)], empty[few_stages(NT)];
    alignas(16) float sx[few_promo_warps(NT)][2][NT];  // the scales of a k block's tokens, per warp
    uint32_t tmem;
    int failed;
    int last;
};

template <int NT>
__global__ void __launch_bounds__(few_threads(NT), 1)
fp8_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const F8Args a) {
    constexpr int STAGES = few_stages(NT), STAGE = few_stage_bytes(NT), PW = few_promo_warps(NT);
    constexpr int COLS = NT * 4 / PW;  // columns (tokens) per promoting warp: all of them with one warpgroup
    constexpr uint32_t TMEM_COLS = NT * STAGES <= 256 ? 256 : 512;
    static_assert(NT * STAGES <= 512, "tensor memory");
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    FewSmem<NT>& sh = *reinterpret_cast<FewSmem<NT>*>(ring + STAGES * STAGE);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int tok_tiles = (a.tokens + NT - 1) / NT, row_tiles = (a.rows + 127) / 128;
    const long long units = (long long)row_tiles * tok_tiles * a.kb_n;
    const long long tiles = (long long)row_tiles * tok_tiles;
    const long long u0 = a.whole ? tiles * blockIdx.x / gridDim.x * a.kb_n : units * blockIdx.x / gridDim.x;
    const long long u1 = a.whole ? tiles * (blockIdx.x + 1) / gridDim.x * a.kb_n : units * (blockIdx.x + 1) / gridDim.x;
    // position of a unit, stepped along: row tile, token tile (innermost after k), k block
    struct Pos {
        int row, tok, kb;
    };
    const long long tile0 = u0 / a.kb_n;
    const Pos begin{(int)(tile0 / tok_tiles), (int)(tile0 % tok_tiles), (int)(u0 - tile0 * a.kb_n)};
    auto next = [&](Pos& p) {
        if (++p.kb == a.kb_n) {
            p.kb = 0;
            if (++p.tok == tok_tiles) p.tok = 0, ++p.row;
        }
    };
    const int head = (int)min(u1 - u0, (long long)STAGES);

    if (tid == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&sh.full[i], 1);
            mbar_init(&sh.done[i], 1);
            mbar_init(&sh.empty[i], PW);
        }
        sh.failed = 0;
        fence_mbar_init();
        // the first weight tiles, before anything else: the weight does not depend on the kernel before this one where that
        // is the tokens' quantisation (which has waited for all that came before it)
        tma_prefetch_map(&map_x);
        if (!a.chained) pdl_wait();
        Pos p = begin;
        for (int st = 0; st < head; ++st, next(p)) {
            mbar_expect_tx(&sh.full[st], STAGE);
            tma_load_2d(ring + st * STAGE, &map_w, p.kb * 128, p.row * 128, &sh.full[st]);
        }
    }
    if (warp == 1) tmem_alloc(&sh.tmem, TMEM_COLS);
    tc5_fence_before();
    __syncthreads();
    tc5_fence_after();
    const uint32_t tmem = sh.tmem;

    if (warp == 0) {
        // ---- producer: weight and token tiles of the run's units ----
        if (elect_one()) {
            Pos p = begin;
            pdl_wait();
            for (int st = 0; st < head; ++st, next(p))
                tma_load_2d(ring + st * STAGE + 128 * 128, &map_x, p.kb * 128, p.tok * NT, &sh.full[st]);
            bool ok = true;
            long long u = u0 + head;
            int st = head == STAGES ? 0 : head;
            uint32_t lap = 0;  // parity of the lap whose reads free a stage
            for (; u < u1; ++u, next(p)) {
                if (!mbar_wait(&sh.empty[st], lap)) {
                    ok = false;
                    break;
                }
                mbar_expect_tx(&sh.full[st], STAGE);
                tma_load_2d(ring + st * STAGE, &map_w, p.kb * 128, p.row * 128, &sh.full[st]);
                tma_load_2d(ring + st * STAGE + 128 * 128, &map_x, p.kb * 128, p.tok * NT, &sh.full[st]);
                if (++st == STAGES) st = 0, lap ^= 1u;
            }
            if (!ok) {  // the copies in flight have to land before the block's shared memory goes away
                for (long long v = max(u0, u - STAGES); v < u; ++v) {
                    const int n = (int)(v - u0);
                    mbar_wait(&sh.full[n % STAGES], (uint32_t)(n / STAGES) & 1u);
                }
                sh.failed = 1;
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---- tensor core: one thread, one wait and one commit a block (each costs it a hundred cycles or two) ----
        if (elect_one()) {
            const uint64_t da = sw128_desc(smem_u32(ring)), db = sw128_desc(smem_u32(ring) + 128 * 128);
            int st = 0;
            uint32_t lap = 0;
            for (long long u = u0; u < u1; ++u) {
                if (!mbar_wait(&sh.full[st], lap)) {
                    sh.failed = 1;
                    break;
                }
                tc5_fence_after();  // (the accumulator's reads: before the arrivals that let the stage be filled again)
                const uint64_t at = (uint64_t)(st * (STAGE >> 4));
#pragma unroll
                for (int j = 0; j < 4; ++j) umma_f8(tmem + st * NT, da + at + 2 * j, db + at + 2 * j, f8_idesc(128, NT), j > 0);
                umma_commit1(&sh.done[st]);
                if (++st == STAGES) st = 0, lap ^= 1u;
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        // ---- promotion: thread = row of the weight (TMEM lane); COLS tokens ----
        pdl_wait();  // the tokens' scales
        const int pw = warp - 4, quarter = warp & 3, col0 = (pw >> 2) * COLS;
        const uint32_t tbase = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)col0;
        float acc[COLS];
        bool ok = true;
        long long u = u0;
        int st = 0;
        uint32_t lap = 0;
        constexpr int AHEAD = 4;
        static_assert(COLS <= 32, "a lane's token");
        // (a wait that ran out is not waited for again, but the run is walked to its end: the other warps of the
        // block count on this one at the named barriers, and the tiles' counters have to come out even)
        while (u < u1) {
            const long long tile = u / a.kb_n;
            const int kb_a = (int)(u - tile * a.kb_n);
            const int kb_b = (int)min((long long)a.kb_n, kb_a + (u1 - u));
            const int row0 = (int)(tile / tok_tiles) * 128, tok0 = (int)(tile % tok_tiles) * NT;
            const float* swp = a.sw + (size_t)(row0 >> 7) * a.kb_n;
            // scales are fetched AHEAD blocks before their use: a block passes in less than a load from L2 takes
            float nx[AHEAD], nw[AHEAD];
            auto fetch = [&](int kb, float& x, float& w) {
                w = 0.0f, x = 0.0f;
                if (kb >= kb_b) return;
                w = swp[kb];
                if (lane < COLS && tok0 + col0 + lane < a.tokens) x = a.sx[(size_t)(tok0 + col0 + lane) * a.kb_n + kb];
            };
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) fetch(kb_a + i, nx[i], nw[i]);
#pragma unroll
            for (int i = 0; i < COLS; ++i) acc[i] = 0.0f;
            for (int kb0 = kb_a; kb0 < kb_b; kb0 += AHEAD)
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    const int kb = kb0 + i;
                    if (kb >= kb_b) break;
                    float* sxs = sh.sx[pw][i & 1];
                    if (lane < COLS) sxs[lane] = nx[i] * nw[i];
                    __syncwarp();
                    fetch(kb + AHEAD, nx[i], nw[i]);
                    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&sh.done[st], lap));
                    tc5_fence_after();
                    uint32_t v[2][16];  // a chunk is read while the one before it is added up
                    tmem_load16(tbase + st * NT, v[0]);
#pragma unroll
                    for (int c = 0; c < COLS / 16; ++c) {
                        tmem_wait16(v[c & 1]);
                        if (c + 1 < COLS / 16) tmem_load16(tbase + st * NT + (c + 1) * 16, v[(c + 1) & 1]);
#pragma unroll
                        for (int q = 0; q < 16; q += 4) {
                            const float4 f = *reinterpret_cast<const float4*>(sxs + c * 16 + q);
                            acc[c * 16 + q] = fmaf(__uint_as_float(v[c & 1][q]), f.x, acc[c * 16 + q]);
                            acc[c * 16 + q + 1] = fmaf(__uint_as_float(v[c & 1][q + 1]), f.y, acc[c * 16 + q + 1]);
                            acc[c * 16 + q + 2] = fmaf(__uint_as_float(v[c & 1][q + 2]), f.z, acc[c * 16 + q + 2]);
                            acc[c * 16 + q + 3] = fmaf(__uint_as_float(v[c & 1][q + 3]), f.w, acc[c * 16 + q + 3]);
                        }
                    }
                    tc5_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_one(&sh.empty[st]);
                    if (++st == STAGES) st = 0, lap ^= 1u;
                }
            u += kb_b - kb_a;
            const int row = row0 + quarter * 32 + lane;
            if (kb_a == 0 && kb_b == a.kb_n) {
                if (row < a.rows)
#pragma unroll
                    for (int i = 0; i < COLS; ++i)
                        if (tok0 + col0 + i < a.tokens)
                            store_as(a.out, a.out_type, (size_t)(tok0 + col0 + i) * a.out_stride + row, acc[i]);
                continue;
            }
            // A piece of a tile: into the workspace; the CTA whose piece is the last to arrive adds them all up.
            auto slot = [&](int cta, long long first) {  // slot 0: the piece the CTA's run begins with
                return a.part + (((size_t)cta * 2 + (first / a.kb_n == tile ? 0 : 1)) * NT) * 128;
            };
            float* mine = slot(blockIdx.x, u0);
#pragma unroll
            for (int i = 0; i < COLS; ++i)
                if (tok0 + col0 + i < a.tokens) __stcg(mine + (size_t)(col0 + i) * 128 + quarter * 32 + lane, acc[i]);
            // If the other pieces are all there, this one needs no publication (usual for the tile a run ends in: the next
            // run began with the tile's other end): its threads read what they wrote themselves.
            const unsigned mine_kb = (unsigned)(kb_b - kb_a);
            if (tid == 128) {
                unsigned now;
                asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(now) : "l"(a.done + tile) : "memory");
                sh.last = now + mine_kb == (unsigned)a.kb_n;
            }
            asm volatile("bar.sync 1, %0;" ::"n"(PW * 32) : "memory");
            const bool alone = sh.last;
            if (alone && tid == 128) a.done[tile] = 0;  // ready for the next launch
            int is_last = alone;
            if (!alone) {
                __threadfence();
                asm volatile("bar.sync 1, %0;" ::"n"(PW * 32) : "memory");
                if (tid == 128) {
                    const unsigned before = atomicAdd(&a.done[tile], mine_kb);
                    sh.last = before + mine_kb == (unsigned)a.kb_n;
                    if (sh.last) a.done[tile] = 0;
                    __threadfence();
                }
                asm volatile("bar.sync 1, %0;" ::"n"(PW * 32) : "memory");
                is_last = sh.last;
            }
            if (is_last) {
                const long long t0 = tile * a.kb_n, t1 = t0 + a.kb_n;
                // the run of CTA c is [units * c / grid, units * (c + 1) / grid)
                int c = (int)(t0 * gridDim.x / units);
                while (units * (c + 1) / gridDim.x <= t0) ++c;
                while (c > 0 && units * c / gridDim.x > t0) --c;
#pragma unroll
                for (int i = 0; i < COLS; ++i) acc[i] = 0.0f;
                for (; units * c / gridDim.x < t1; ++c) {
                    const float* p = slot(c, units * c / gridDim.x);
#pragma unroll
                    for (int i = 0; i < COLS; ++i)
                        if (tok0 + col0 + i < a.tokens) acc[i] += __ldcg(p + (size_t)(col0 + i) * 128 + quarter * 32 + lane);
                    if (c + 1 >= (int)gridDim.x) break;
                }
                if (row < a.rows)
#pragma unroll
                    for (int i = 0; i < COLS; ++i)
                        if (tok0 + col0 + i < a.tokens)
                            store_as(a.out, a.out_type, (size_t)(tok0 + col0 + i) * a.out_stride + row, acc[i]);
            }
            asm volatile("bar.sync 1, %0;" ::"n"(PW * 32) : "memory");  // sh.last may be written again
        }
        if (!ok && lane == 0) sh.failed = 1;
    }
    tc5_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc5_fence_after();
        tmem_free(tmem, TMEM_COLS);
    }
    if (tid == 0 && sh.failed) set_err(a.err, DEV_ERR_TMA_TIMEOUT);
}

// ----------------------------------------------------------- many tokens ----
// What bounds it is the promotion: a block (128 x 256 x 128) takes 0.60 us, 0.59 with a quarter of its multiplications, and
// 0.43 without the promotion.  What of the promotion costs that is not known: it reads the block's 128 KB from tensor
// memory, from the barrier on and to the end before the next block's barrier, and its threads (96 registers at 640
// threads) spill 400 to 976 bytes.  4096 x 8192 -> 28672 in 1.02 ms, 1.9 PFLOP/s, in a burst, 1.2 ms at the power limit.
// Measured and not kept: pairs of CTAs on one tile (a third less to load: 1.06 ms),
// accumulators handed over by halves (1.05), two multiply-adds an instruction (1.09), one arrival a warp (1.05).
constexpr int MANY_M = 128, MANY_N = 256, MANY_STAGES = 4;
constexpr int MANY_STAGE = (MANY_M + MANY_N) * 128;
constexpr int MANY_THREADS = 128 + 512;  // producer, tensor core, two idle warps (a warp reads the TMEM lanes of its rank of 4), promotion

struct ManySmem {
    uint64_t full[MANY_STAGES], empty[MANY_STAGES];
    uint64_t acc_full[2], acc_empty[2];
    uint32_t tmem;
    int failed;
    uint32_t turn[16][32][16];  // a promoting warp's 32 tokens x 64 bytes, on their way to stores along the rows
};

template <class T>
__global__ void __launch_bounds__(MANY_THREADS, 1)
fp8_many_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const F8Args a) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    ManySmem& sh = *reinterpret_cast<ManySmem*>(ring + MANY_STAGES * MANY_STAGE);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int m_tiles = (a.tokens + MANY_M - 1) / MANY_M, n_tiles = (a.rows + MANY_N - 1) / MANY_N;
    const int tiles = m_tiles * n_tiles;
    // tiles in bands of up to 16 token tiles: the CTAs at work share few row and token tiles of both operands in L2
    auto tile_at = [&](int t, int& m, int& n) {
        constexpr int BAND = 16;
        const int band = t / (BAND * n_tiles), in = t - band * BAND * n_tiles;
        const int h = min(BAND, m_tiles - band * BAND);
        m = band * BAND + in % h;
        n = in / h;
    };

    if (tid == 0) {
        for (int i = 0; i < MANY_STAGES; ++i) {
            mbar_init(&sh.full[i], 1);
            mbar_init(&sh.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.acc_full[i], 1);
            mbar_init(&sh.acc_empty[i], 512);
        }
        sh.failed = 0;
        fence_mbar_init();
        tma_prefetch_map(&map_w);
        tma_prefetch_map(&map_x);
    }
    if (warp == 1) tmem_alloc(&sh.tmem, 512);
    tc5_fence_before();
    __syncthreads();
    tc5_fence_after();
    const uint32_t tmem = sh.tmem;
    pdl_wait();

    if (warp == 0) {
        if (elect_one()) {
            bool ok = true;
            int n = 0;
            for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
                int mt, nt;
                tile_at(t, mt, nt);
                for (int kb = 0; kb < a.kb_n; ++kb, ++n) {
                    const int st = n % MANY_STAGES;
                    if (n >= MANY_STAGES && !mbar_wait(&sh.empty[st], (uint32_t)(n / MANY_STAGES - 1) & 1u)) {
                        ok = false;
                        break;
                    }
                    mbar_expect_tx(&sh.full[st], MANY_STAGE);
                    tma_load_2d(ring + st * MANY_STAGE, &map_x, kb * 128, mt * MANY_M, &sh.full[st]);
                    tma_load_2d(ring + st * MANY_STAGE + MANY_M * 128, &map_w, kb * 128, nt * MANY_N, &sh.full[st]);
                }
            }
            if (!ok) {
                for (int v = max(0, n - MANY_STAGES); v < n; ++v)
                    mbar_wait(&sh.full[v % MANY_STAGES], (uint32_t)(v / MANY_STAGES) & 1u);
                sh.failed = 1;
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (elect_one()) {
            const uint64_t da = sw128_desc(smem_u32(ring)), db = sw128_desc(smem_u32(ring) + MANY_M * 128);
            bool ok = true;
            int st = 0;
            uint32_t lap = 0, n = 0;
            for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x)
                for (int kb = 0; kb < a.kb_n; ++kb, ++n) {
                    const uint32_t buf = n & 1;
                    ok = mbar_wait(&sh.acc_empty[buf], ((n >> 1) & 1u) ^ 1u) && mbar_wait(&sh.full[st], lap);  // (the first lap's wait passes)
                    if (!ok) break;
                    tc5_fence_after();
                    const uint64_t at = (uint64_t)(st * (MANY_STAGE >> 4));
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        umma_f8(tmem + buf * MANY_N, da + at + 2 * j, db + at + 2 * j, f8_idesc(MANY_M, MANY_N), j > 0);
                    umma_commit1(&sh.empty[st]);
                    umma_commit1(&sh.acc_full[buf]);
                    if (++st == MANY_STAGES) st = 0, lap ^= 1u;
                }
            if (!ok) sh.failed = 1;
        }
        __syncwarp();
    } else if (warp >= 4) {
        // thread = token (TMEM lane), 64 rows of the weight (of one row of scale blocks)
        constexpr int COLS = 64;
        const int quarter = warp & 3, col0 = ((warp - 4) >> 2) * COLS;
        const uint32_t tbase = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)col0;
        const bool wide = ((reinterpret_cast<uintptr_t>(a.out) | (size_t)a.out_stride * sizeof(T)) & 15) == 0;
        bool ok = true;
        int n = 0;
        for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
            int mt, nt;
            tile_at(t, mt, nt);
            const int tok = mt * MANY_M + quarter * 32 + lane, row0 = nt * MANY_N + col0;
            const float* sxp = a.sx + (size_t)min(tok, a.tokens - 1) * a.kb_n;
            const float* swp = a.sw + (size_t)(min(row0, a.rows - 1) >> 7) * a.kb_n;
            float acc[COLS];
#pragma unroll
            for (int i = 0; i < COLS; ++i) acc[i] = 0.0f;
            float nx = sxp[0], nw = swp[0];
            for (int kb = 0; kb < a.kb_n; ++kb, ++n) {
                const int buf = n & 1;
                const float f = nx * nw;
                if (kb + 1 < a.kb_n) {
                    nx = sxp[kb + 1];
                    nw = swp[kb + 1];
                }
                ok = __all_sync(0xffffffffu, mbar_wait(&sh.acc_full[buf], (uint32_t)(n >> 1) & 1u));
                if (!ok) break;
                tc5_fence_after();
                uint32_t v[2][16];  // a chunk is read while the one before it is added up
                tmem_load16(tbase + buf * MANY_N, v[0]);
#pragma unroll
                for (int c = 0; c < COLS / 16; ++c) {
                    tmem_wait16(v[c & 1]);
                    if (c + 1 < COLS / 16) tmem_load16(tbase + buf * MANY_N + (c + 1) * 16, v[(c + 1) & 1]);
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[c * 16 + i] = fmaf(__uint_as_float(v[c & 1][i]), f, acc[c * 16 + i]);
                }
                tc5_fence_before();
                mbar_arrive_one(&sh.acc_empty[buf]);
            }
            if (!ok) break;
            if (wide && row0 + COLS <= a.rows) {
                T* o = static_cast<T*>(a.out) + (size_t)tok * a.out_stride + row0;
                constexpr int V = 16 / (int)sizeof(T);
                if (tok < a.tokens)
#pragma unroll
                    for (int i = 0; i < COLS; i += V) {
                        alignas(16) T p[V];
#pragma unroll
                        for (int j = 0; j < V; ++j) p[j] = narrow<T>(acc[i + j]);
                        *reinterpret_cast<uint4*>(o + i) = *reinterpret_cast<const uint4*>(p);
                    }
            } else {
                // the lanes turn from tokens to columns, so that a store covers 64 bytes of a row (one element in each of
                // 32 rows otherwise: 351 x 320 -> 13241 bf16 80 us against 28)
                constexpr int PACK = 4 / (int)sizeof(T), C = 16 * PACK;
                uint32_t(*turn)[16] = sh.turn[warp - 4];
                const int col = lane % C, tok0 = mt * MANY_M + quarter * 32;
#pragma unroll
                for (int c0 = 0; c0 < COLS; c0 += C) {
#pragma unroll
                    for (int w = 0; w < 16; ++w) {
                        alignas(4) T p[PACK];
#pragma unroll
                        for (int j = 0; j < PACK; ++j) p[j] = narrow<T>(acc[c0 + w * PACK + j]);
                        turn[lane][w ^ (lane & 15)] = *reinterpret_cast<const uint32_t*>(p);
                    }
                    __syncwarp();
                    for (int r0 = 0; r0 < 32; r0 += 32 / C) {
                        const int r = r0 + lane / C;
                        const uint32_t word = turn[r][(col / PACK) ^ (r & 15)];
                        if (tok0 + r < a.tokens && row0 + c0 + col < a.rows)
                            static_cast<T*>(a.out)[(size_t)(tok0 + r) * a.out_stride + row0 + c0 + col] =
                                reinterpret_cast<const T*>(&word)[col % PACK];
                    }
                    __syncwarp();
                }
            }
        }
        if (!ok && lane == 0) sh.failed = 1;
    }
    tc5_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc5_fence_after();
        tmem_free(tmem, 512);
    }
    if (tid == 0 && sh.failed) set_err(a.err, DEV_ERR_TMA_TIMEOUT);
}

// ------------------------------------------------------------------ host ----
// [rows][cols] bytes, box of 128 columns; what lies past the ends reads as zero (an e4m3 zero).
cudaError_t encode_bytes(CUtensorMap* map, const void* base, size_t rows, size_t cols, size_t pitch, int box_rows) {
    return encode_tile_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, rows, cols, pitch, box_rows, 128, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int NT>
cudaError_t launch_few(const Fp8Product& p, const F8Args& a, int grid, cudaStream_t st) {
    CUtensorMap mw, mx;
    cudaError_t e = encode_bytes(&mw, p.w, p.rows, p.cols, p.cols, 128);
    if (e == cudaSuccess) e = encode_bytes(&mx, p.codes, p.tokens, p.cols, p.code_pitch, NT);
    if (e != cudaSuccess) return e;
    const size_t smem = 1024 + (size_t)few_stages(NT) * few_stage_bytes(NT) + sizeof(FewSmem<NT>);
    static_assert(1024 + few_stages(NT) * few_stage_bytes(NT) + sizeof(FewSmem<NT>) <= 227 * 1024, "shared memory");
    if ((e = set_max_dyn_smem((const void*)fp8_few_kernel<NT>, 227 * 1024)) != cudaSuccess) return e;
    return launch_chained(fp8_few_kernel<NT>, dim3(grid), dim3(few_threads(NT)), smem, st, mw, mx, a);
}

template <class T>
cudaError_t launch_many(const Fp8Product& p, const F8Args& a, int grid, cudaStream_t st) {
    CUtensorMap mw, mx;
    cudaError_t e = encode_bytes(&mw, p.w, p.rows, p.cols, p.cols, MANY_N);
    if (e == cudaSuccess) e = encode_bytes(&mx, p.codes, p.tokens, p.cols, p.code_pitch, MANY_M);
    if (e != cudaSuccess) return e;
    constexpr size_t smem = 1024 + (size_t)MANY_STAGES * MANY_STAGE + sizeof(ManySmem);
    static_assert(smem <= 227 * 1024, "shared memory");
    if ((e = set_max_dyn_smem((const void*)fp8_many_kernel<T>, 227 * 1024)) != cudaSuccess) return e;
    return launch_chained(fp8_many_kernel<T>, dim3(grid), dim3(MANY_THREADS), smem, st, mw, mx, a);
}

// How a product runs, from estimates in microseconds (fitted to 23 shapes of 1 to 1024 tokens): a k block of a few-token
// tile takes an SM 0.235 to 0.40 by its columns, or the memory the time of its 16 KB; joining pieces of tiles costs 3.5,
// 0.11 per column and 0.45 per piece of a tile; a k block of a 128 x 256 tile of the other kernel takes 0.60.  Measured,
// quantisation included, whole tiles | tiles spread over the grid | the other kernel:
//   1 x 3840 -> 15360    16 columns 14.7 | 19.4 | 20.8
//   16 x 28672 -> 8192   16 columns 51.5 | 49.9 | 105
//   64 x 2880 -> 2880    16 columns 10.7 | 16.7, 32 columns 11.3 | 16.3, 64 columns 13.1 | 19.7, 16.5
//   64 x 8192 -> 28672   64 columns 59.8 | 55.9 | 49.7
//   128 x 28672 -> 8192  32 columns 122 | 155, 64 columns 96.8 | 95.9 | 134
//   250 x 2880 -> 2880   32 columns 20.6 | 22.7, 64 columns 14.6 | 21.4 | 20.7
//   512 x 8192 -> 8192   64 columns 107 | 104 | 45.5
// (128 columns were never the fastest: 171 | 108 us at 128 x 28672 -> 8192, 20.3 | 29.3 at 250 x 2880 -> 2880.)
struct Way {
    int nt;  // columns of the few-token kernel's accumulators, 0: the other kernel
    bool whole;
    int grid;
    double us;
};
Way way_of(size_t tokens, size_t rows, size_t cols, int sm_count) {
    const double kb = (double)((cols + 127) / 128), sms = sm_count, row_tiles = (double)((rows + 127) / 128);
    const double memory = row_tiles * kb * 0.00264;
    Way best{};
    auto take = [&](const Way& w) {
        if (best.grid == 0 || w.us < best.us) best = w;
    };
    for (int nt = 16; nt <= 64; nt *= 2) {
        const double tiles = (double)((tokens + nt - 1) / nt) * row_tiles, units = tiles * kb;
        const double unit = nt == 16 ? 0.235 : (nt == 32 ? 0.27 : 0.40);
        take(Way{nt, true, (int)std::min(tiles, sms), std::max(memory, std::ceil(tiles / sms) * kb * unit)});
        take(Way{nt, false, (int)std::min(units, sms), std::max(memory, std::ceil(units / sms) * unit) + 3.5 + 0.11 * nt + 0.45 * sms / tiles});
        if ((size_t)nt >= tokens) break;
    }
    const double tiles = (double)((tokens + MANY_M - 1) / MANY_M) * (double)((rows + MANY_N - 1) / MANY_N);
    take(Way{0, true, (int)std::min(tiles, sms), std::max(memory, std::ceil(tiles / sms) * kb * 0.60)});
    return best;
}

}  // namespace

cudaError_t launch_fp8_quantize(const void* x, int type, size_t tokens, size_t cols, size_t x_stride, uint8_t* codes,
                                size_t code_pitch, float* scales, int sm_count, cudaStream_t st) {
    if (tokens == 0 || cols == 0) return cudaSuccess;
    const int kb_n = (int)((cols + 127) / 128);
    const size_t z = type == LQ_T_F32 ? 4 : 2;
    const bool vec = cols % 8 == 0 && (((uintptr_t)x | x_stride * z) & 15) == 0;
    const int wide = cols % 8 == 0 && (((uintptr_t)codes | code_pitch) & 7) == 0;
    const size_t most = std::max<size_t>(1, (size_t)(1 << 29) / kb_n);  // tokens whose blocks are counted in 32 bits
    for (size_t t0 = 0; t0 < tokens; t0 += most) {
        const int units = (int)(std::min(most, tokens - t0) * kb_n);
        const void* xt = (const uint8_t*)x + t0 * x_stride * z;
        uint8_t* ct = codes + t0 * code_pitch;
        float* sc = scales + t0 * kb_n;
        auto go = [&](auto* tag, auto vtag, auto qtag) {
            using T = std::remove_pointer_t<decltype(tag)>;
            constexpr int Q = decltype(qtag)::value;
            const int grid = std::min((units + 16 * Q - 1) / (16 * Q), sm_count * 32);
            return launch_chained(fp8_quantize_kernel<T, decltype(vtag)::value, Q>, dim3(grid), dim3(256), 0, st, (const T*)xt,
                                  (long long)x_stride, units, kb_n, (int)cols, ct, (long long)code_pitch, sc, wide, Divisor::make((uint32_t)kb_n));
        };
        auto by_type = [&](auto vtag, auto qtag) {
            if (type == LQ_T_F32) return go((float*)nullptr, vtag, qtag);
            if (type == LQ_T_BF16) return go((__nv_bfloat16*)nullptr, vtag, qtag);
            return go((__half*)nullptr, vtag, qtag);
        };
        using One = std::integral_constant<int, 1>;
        using Two = std::integral_constant<int, 2>;
        cudaError_t e;
        if (!vec) e = by_type(std::false_type{}, One{});
        else if (units >= sm_count * 64) e = by_type(std::true_type{}, Two{});
        else e = by_type(std::true_type{}, One{});
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

// Partial tiles and counters of the few-token kernel.
size_t fp8_part_bytes(size_t tokens, size_t rows, size_t cols, int sm_count) {
    const Way w = way_of(tokens, rows, cols, sm_count);
    return w.whole ? 0 : (size_t)w.grid * 2 * w.nt * 128 * 4;
}
size_t fp8_tile_count(size_t tokens, size_t rows, size_t cols, int sm_count) {
    const Way w = way_of(tokens, rows, cols, sm_count);
    return w.whole ? 0 : ((rows + 127) / 128) * ((tokens + w.nt - 1) / w.nt);
}
cudaError_t launch_fp8_matmul(const Fp8Product& p, bool chained, int sm_count, int* err, cudaStream_t st) {
    const int kb_n = (int)((p.cols + 127) / 128);
    F8Args a{};
    a.sx = p.scales, a.sw = p.w_scales, a.out = p.out, a.out_stride = (long long)p.out_stride, a.out_type = p.out_type;
    a.tokens = (int)p.tokens, a.rows = (int)p.rows, a.kb_n = kb_n;
    a.part = p.part, a.done = p.done, a.err = err;
    const Way w = way_of(p.tokens, p.rows, p.cols, sm_count);
    const int grid = w.grid;
    a.whole = w.whole;
    a.chained = chained;
    switch (w.nt) {
        case 16: return launch_few<16>(p, a, grid, st);
        case 32: return launch_few<32>(p, a, grid, st);
        case 64: return launch_few<64>(p, a, grid, st);
    }
    if (p.out_type == LQ_T_F32) return launch_many<float>(p, a, grid, st);
    if (p.out_type == LQ_T_BF16) return launch_many<__nv_bfloat16>(p, a, grid, st);
    return launch_many<__half>(p, a, grid, st);
}

}  // namespace lq
