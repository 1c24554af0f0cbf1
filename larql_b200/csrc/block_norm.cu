// The norms around a block of a decoder layer, fused with its gate and residual scale (lq_dev_block_norm):
//
//   z  = y / rms(y) * (off + post_w)            (z = y without the post norm)
//   h' = h_scale * h + y_scale * gate * z       (h' = h_scale * h without a block output)
//   n  = h' / rms(h') * (off + pre_w)           rms(v) = sqrt(mean(v^2) + eps)
//
// run_ffn's norm -> FFN -> residual add (crates/larql-compute/src/forward/layer.rs:61-127) with the post-FFN
// norm, the learned weights and the residual multiplier of layers that have them.
//
// What bounds it is reading h, y, gate and writing h', n once (one token: the two reductions' latency).  Everything is
// kept in f32 between the loads and the stores, n is taken from the unrounded h'.  A row's squares are summed in f32,
// pairwise over the threads; when that sum leaves f32's range the row is summed again at 2^-80 of its size
// (f64 sums, which need no branch, cost 36 us of 159 at 4096 x 8192 bf16: the conversions run at a few lanes a cycle).
// Underflow needs no branch: what a square loses is below 2^-149 and eps is at least 2^-126.
// rms is at least sqrt(eps) >= 2^-63; rows with an rms above 2^100 are scaled down before 1 / rms is taken of them, so that
// it is a normal f32 far from the type's end and one multiply per element replaces a division.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/larql_cuda.h"
#include "kernels.h"
#include "tc5.cuh"

#include <type_traits>

namespace lq {

namespace {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// VEC consecutive elements: one 16-byte access, or one element where an address or width rules that out.
template <class T, int VEC>
struct alignas(VEC * sizeof(T)) Pack {
    T v[VEC];
};

// VEC weights as f32: of the activation's type (SAME: one access), or of any type, element by element.
template <class T, int VEC, bool SAME>
__device__ __forceinline__ void load_w(const void* w, int type, size_t at, float (&out)[VEC]) {
    if (SAME) {
        const Pack<T, VEC> p = *reinterpret_cast<const Pack<T, VEC>*>(static_cast<const T*>(w) + at);
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = to_f32(p.v[i]);
    } else if (type == LQ_T_F32) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = static_cast<const float*>(w)[at + i];
    } else if (type == LQ_T_BF16) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = to_f32(static_cast<const __nv_bfloat16*>(w)[at + i]);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = to_f32(static_cast<const __half*>(w)[at + i]);
    }
}

// The sum over the threads of a row, one warp (WARP) or the whole block.
template <bool WARP>
__device__ __forceinline__ float row_sum(float s, float* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (WARP) return s;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockDim.x >> 5;
    __syncthreads();  // the previous result has been read
    if (lane == 0) red[warp] = s;
    __syncthreads();
    s = lane < n ? red[lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}

// Sum of N squares, pairwise.
template <int N>
__device__ __forceinline__ float square_sum(const float (&v)[N], float scale) {
    float q[N];
#pragma unroll
    for (int i = 0; i < N; ++i) q[i] = (v[i] * scale) * (v[i] * scale);
#pragma unroll
    for (int n = N / 2; n > 0; n >>= 1)
#pragma unroll
        for (int i = 0; i < n; ++i) q[i] += q[i + n];
    return q[0];
}
// inverse_rms for a row whose squares' sum left f32's range: its mean square lies between 2^112 (cols <= 2^14) and 2^256.  Such a
// row is measured at 2^-80 of its size; above an rms of 2^100 it also goes on at 2^-64 (`shrink`, for the caller to apply to
// its elements), or 1 / rms and its products with small weights would be subnormal.  An infinity gives 0 (finite / inf, and
// inf * 0 = NaN where it stands), a NaN NaN.
template <bool WARP, int N>
__device__ __forceinline__ float inverse_rms_beyond(const float (&v)[N], float inv_cols, float eps, float* red, float& shrink) {
    const float t = row_sum<WARP>(square_sum(v, 0x1p-80f), red);
    const float inv = 1.0f / sqrtf(fmaf(t, inv_cols, eps * 0x1p-80f * 0x1p-80f));  // of the row at 2^-80, at least 2^-48
    shrink = inv < 0x1p-20f ? 0x1p-64f : 1.0f;
    return inv * (inv < 0x1p-20f ? 0x1p-16f : 0x1p-80f);
}
// 1 / rms of the row whose elements the threads hold N each (zero past the end; scaled down with it where they are too large).
template <bool WARP, int N>
__device__ __forceinline__ float inverse_rms(float (&v)[N], float inv_cols, float eps, float* red) {
    const float s = row_sum<WARP>(square_sum(v, 1.0f), red);
    if (s <= 1e38f) return 1.0f / sqrtf(s * inv_cols + eps);
    float shrink;
    const float inv = inverse_rms_beyond<WARP>(v, inv_cols, eps, red, shrink);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] *= shrink;
    return inv;
}

// One row per warp (WARP: blockDim = 32 x rows) or per block; a thread holds NV packs of VEC elements.  AHEAD: weights are
// loaded before the reduction their use waits for (1 x 2885 f32 6.3 -> 5.4 us, 300 x 8192 bf16 14.5 -> 13.1); with many rows
// to an SM, or blocks of 1024 threads, the registers that takes cost more (1000 x 529 bf16 5.9 -> 6.7, 4096 x 1024 9.7 ->
// 10.5, 1 x 16384 6.0 -> 6.9).
template <class T, int VEC, int NV, bool WARP, bool SAME, bool AHEAD, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) block_norm_kernel(const BlockNorm a) {
    __shared__ float red[32];
    const int tid = threadIdx.x, step = blockDim.x;
    const int n_pack = a.cols / VEC;
    const float inv_cols = 1.0f / (float)a.cols, eps = (float)a.eps;
    using P = Pack<T, VEC>;
    const int rows_per = WARP ? blockDim.y : 1;
    pdl_wait();
    // (unsigned: a step past the last row may leave int's range)
    for (unsigned row = blockIdx.x * rows_per + (WARP ? threadIdx.y : 0); row < (unsigned)a.rows; row += gridDim.x * rows_per) {
        P h[NV], g[NV];
        float v[NV * VEC];  // y, then z, then h'
        const T* hp = static_cast<const T*>(a.h) + (size_t)row * a.h_stride;
        const T* yp = static_cast<const T*>(a.y) + (a.y ? (size_t)row * a.y_stride : 0);
        const T* gp = static_cast<const T*>(a.gate) + (a.gate ? (size_t)(row / (unsigned)a.gate_group) * a.gate_stride : 0);
        const bool gate_vec = a.gate && a.gate_cols != 1;
        float gs = a.y_scale;
        if (a.gate && a.gate_cols == 1) gs *= to_f32(gp[0]);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int p = tid + i * step;
            P y = {};
            if (p < n_pack) {
                if (a.y) y = *reinterpret_cast<const P*>(yp + (size_t)p * VEC);
                h[i] = *reinterpret_cast<const P*>(hp + (size_t)p * VEC);
                if (gate_vec) g[i] = *reinterpret_cast<const P*>(gp + (size_t)p * VEC);
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[i * VEC + j] = to_f32(y.v[j]);
        }
        float ahead[AHEAD ? NV * VEC : 1];  // (SAME: converted after the reduction)
        P raw[AHEAD && SAME ? NV : 1];
        auto fetch = [&](const void* w) {
            if (!AHEAD || !w) return;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int p = tid + i * step;
                if (p >= n_pack) continue;
                if constexpr (AHEAD && SAME) {
                    raw[i] = *reinterpret_cast<const P*>(static_cast<const T*>(w) + (size_t)p * VEC);
                } else if constexpr (AHEAD) {
                    float e[VEC];
                    load_w<T, VEC, false>(w, a.w_type, (size_t)p * VEC, e);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) ahead[i * VEC + j] = e[j];
                }
            }
        };
        auto weights = [&](const void* w, int i, float (&out)[VEC]) {
            if constexpr (AHEAD) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    if constexpr (SAME) out[j] = to_f32(raw[i].v[j]);
                    else out[j] = ahead[i * VEC + j];
                }
            } else if (w) {
                load_w<T, VEC, SAME>(w, a.w_type, (size_t)(tid + i * step) * VEC, out);
            }
        };
        float inv = 1.0f;
        if (a.post_norm) {
            fetch(a.post_w);
            inv = inverse_rms<WARP>(v, inv_cols, eps, red);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int p = tid + i * step;
            if (p < n_pack) {
                if (a.post_norm) {
                    float w[VEC];
                    weights(a.post_w, i, w);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) v[i * VEC + j] *= a.post_w ? inv * (a.w_offset + w[j]) : inv;
                }
                P o;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    float x = a.h_scale * to_f32(h[i].v[j]);
                    if (a.y) x = fmaf(gate_vec ? gs * to_f32(g[i].v[j]) : gs, v[i * VEC + j], x);
                    v[i * VEC + j] = x;
                    o.v[j] = from_f32<T>(x);
                }
                if (a.h_out) *reinterpret_cast<P*>(static_cast<T*>(a.h_out) + (size_t)row * a.h_out_stride + (size_t)p * VEC) = o;
            }
        }
        if (a.n_out) {
            fetch(a.pre_w);
            inv = inverse_rms<WARP>(v, inv_cols, eps, red);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int p = tid + i * step;
                if (p < n_pack) {
                    float w[VEC];
                    weights(a.pre_w, i, w);
                    P o;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) o.v[j] = from_f32<T>(v[i * VEC + j] * (a.pre_w ? inv * (a.w_offset + w[j]) : inv));
                    *reinterpret_cast<P*>(static_cast<T*>(a.n_out) + (size_t)row * a.n_out_stride + (size_t)p * VEC) = o;
                }
            }
        }
    }
}

// Two f32 in one register pair, worked on by one instruction (each lane of it correctly rounded).
using F2 = unsigned long long;
__device__ __forceinline__ F2 pair(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 halves(F2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
// A pack's elements in pairs, and back.
template <class T, int VEC>
__device__ __forceinline__ void pairs_of(const Pack<T, VEC>& p, F2 (&out)[VEC / 2]) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
        if constexpr (sizeof(T) == 4) {
            out[i] = pair(p.v[2 * i], p.v[2 * i + 1]);
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            const uint32_t w = reinterpret_cast<const uint32_t*>(&p)[i];
            out[i] = pair(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
        } else {
            const float2 f = __half22float2(reinterpret_cast<const __half2*>(&p)[i]);
            out[i] = pair(f.x, f.y);
        }
    }
}
template <class T>
__device__ __forceinline__ void put_pair(T* at, F2 v) {
    const float2 f = halves(v);
    if constexpr (sizeof(T) == 4) at[0] = f.x, at[1] = f.y;
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) *reinterpret_cast<__nv_bfloat162*>(at) = __floats2bfloat162_rn(f.x, f.y);
    else *reinterpret_cast<__half2*>(at) = __floats2half2_rn(f.x, f.y);
}
// inverse_rms of elements held in pairs, by the whole block.
template <int N>
__device__ __forceinline__ float inverse_rms_pairs(F2 (&v)[N], float inv_cols, float eps, float* red) {
    F2 q[N];
#pragma unroll
    for (int i = 0; i < N; ++i) q[i] = mul2(v[i], v[i]);
#pragma unroll
    for (int n = N / 2; n > 0; n >>= 1)
#pragma unroll
        for (int i = 0; i < n; ++i) q[i] = add2(q[i], q[i + n]);
    const float2 f = halves(q[0]);
    const float s = row_sum<false>(f.x + f.y, red);
    if (s <= 1e38f) return 1.0f / sqrtf(s * inv_cols + eps);
    float e[2 * N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float2 h = halves(v[i]);
        e[2 * i] = h.x, e[2 * i + 1] = h.y;
    }
    float shrink;
    const float inv = inverse_rms_beyond<false>(e, inv_cols, eps, red, shrink);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = mul2(v[i], pair(shrink, shrink));
    return inv;
}

// Many long rows: a block walks its rows with the next one's operands on their way into shared memory (bulk copies), so
// that the memory is never idle during a row's two reductions.  4096 x 8192 bf16 with a full gate: 60 us (5.6 TB/s) against 98
// with loads into registers.
template <class T, int VEC, int NV, bool SAME, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) block_norm_stream_kernel(const BlockNorm a, int gate_rows) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float red[32];
    __shared__ uint64_t full[2];
    const int tid = threadIdx.x, step = blockDim.x;
    const int n_pack = a.cols / VEC;
    const float inv_cols = 1.0f / (float)a.cols, eps = (float)a.eps;
    using P = Pack<T, VEC>;
    const uint32_t row_bytes = (uint32_t)a.cols * sizeof(T), stage = row_bytes * (gate_rows ? 3 : 2);
    unsigned issued = 0;  // (thread 0)
    auto issue = [&](int s, int row) {  // h, y and the row's own gate row, behind one another
        ++issued;
        uint8_t* dst = smem + (size_t)s * stage;
        mbar_expect_tx(&full[s], stage);
        tma_bulk_g2s(dst, static_cast<const T*>(a.h) + (size_t)row * a.h_stride, row_bytes, &full[s]);
        tma_bulk_g2s(dst + row_bytes, static_cast<const T*>(a.y) + (size_t)row * a.y_stride, row_bytes, &full[s]);
        if (gate_rows) tma_bulk_g2s(dst + 2 * row_bytes, static_cast<const T*>(a.gate) + (size_t)row * a.gate_stride, row_bytes, &full[s]);
    };
    if (tid == 0) {
        mbar_init(&full[0], 1);
        mbar_init(&full[1], 1);
        fence_mbar_init();
    }
    pdl_wait();
    if (tid == 0) {
        issue(0, blockIdx.x);  // (the grid is no larger than the rows)
        if (blockIdx.x + gridDim.x < (unsigned)a.rows) issue(1, blockIdx.x + gridDim.x);
    }
    __syncthreads();
    bool ok = true;
    int s = 0;
    uint32_t phase = 0;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        if (ok) ok = mbar_wait(&full[s], phase);
        const T* hs = reinterpret_cast<const T*>(smem + (size_t)s * stage);
        const T* ys = hs + a.cols;
        const T* gp = gate_rows ? ys + a.cols : static_cast<const T*>(a.gate) + (a.gate ? (size_t)(row / a.gate_group) * a.gate_stride : 0);
        const bool gate_vec = a.gate && a.gate_cols != 1;
        float gs = a.y_scale;
        if (a.gate && a.gate_cols == 1) gs *= to_f32(gp[0]);
        constexpr int H = VEC / 2;
        F2 v[NV * H];  // y, then z, then h'
        const F2 gs2 = pair(gs, gs), hs2 = pair(a.h_scale, a.h_scale), off2 = pair(a.w_offset, a.w_offset);
        // weights of the activation's type are on their way during the reduction before their use
        P raw[NV];
        auto fetch = [&](const void* w) {
            if (!SAME || !w) return;
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (tid + i * step < n_pack) raw[i] = *reinterpret_cast<const P*>(static_cast<const T*>(w) + (size_t)(tid + i * step) * VEC);
        };
        auto weights = [&](const void* w, int i, float inv, F2 (&out)[H]) {  // inv * (offset + weight)
            const F2 inv2 = pair(inv, inv);
            const int p = tid + i * step;
            if (SAME) {
                pairs_of<T, VEC>(raw[i], out);
            } else {
                float e[VEC];
                load_w<T, VEC, false>(w, a.w_type, (size_t)p * VEC, e);
#pragma unroll
                for (int j = 0; j < H; ++j) out[j] = pair(e[2 * j], e[2 * j + 1]);
            }
#pragma unroll
            for (int j = 0; j < H; ++j) out[j] = mul2(inv2, add2(off2, out[j]));
        };
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int p = tid + i * step;
            F2 y[H] = {};
            if (p < n_pack) pairs_of<T, VEC>(*reinterpret_cast<const P*>(ys + p * VEC), y);
#pragma unroll
            for (int j = 0; j < H; ++j) v[i * H + j] = y[j];
        }
        float inv = 1.0f;
        if (a.post_norm) {
            fetch(a.post_w);
            inv = inverse_rms_pairs(v, inv_cols, eps, red);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int p = tid + i * step;
            if (p < n_pack) {
                if (a.post_norm) {
                    F2 w[H];
                    if (a.post_w) {
                        weights(a.post_w, i, inv, w);
                    } else {
#pragma unroll
                        for (int j = 0; j < H; ++j) w[j] = pair(inv, inv);
                    }
#pragma unroll
                    for (int j = 0; j < H; ++j) v[i * H + j] = mul2(v[i * H + j], w[j]);
                }
                F2 h[H], g[H];
                pairs_of<T, VEC>(*reinterpret_cast<const P*>(hs + p * VEC), h);
                if (gate_vec) {
                    pairs_of<T, VEC>(*reinterpret_cast<const P*>(gp + p * VEC), g);
#pragma unroll
                    for (int j = 0; j < H; ++j) g[j] = mul2(gs2, g[j]);
                } else {
#pragma unroll
                    for (int j = 0; j < H; ++j) g[j] = gs2;
                }
                P o;
#pragma unroll
                for (int j = 0; j < H; ++j) {
                    v[i * H + j] = fma2(g[j], v[i * H + j], mul2(hs2, h[j]));
                    put_pair(o.v + 2 * j, v[i * H + j]);
                }
                if (a.h_out) *reinterpret_cast<P*>(static_cast<T*>(a.h_out) + (size_t)row * a.h_out_stride + (size_t)p * VEC) = o;
            }
        }
        if (a.n_out) {
            fetch(a.pre_w);
            inv = inverse_rms_pairs(v, inv_cols, eps, red);
        } else {
            __syncthreads();
        }
        // (everyone has read the stage: the reduction above was a barrier)
        if (tid == 0 && ok && row + 2ll * gridDim.x < a.rows) issue(s, (int)(row + 2ll * gridDim.x));
        if (a.n_out) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int p = tid + i * step;
                if (p < n_pack) {
                    P o;
                    F2 w[H];
                    if (a.pre_w) {
                        weights(a.pre_w, i, inv, w);
                    } else {
#pragma unroll
                        for (int j = 0; j < H; ++j) w[j] = pair(inv, inv);
                    }
#pragma unroll
                    for (int j = 0; j < H; ++j) put_pair(o.v + 2 * j, mul2(v[i * H + j], w[j]));
                    *reinterpret_cast<P*>(static_cast<T*>(a.n_out) + (size_t)row * a.n_out_stride + (size_t)p * VEC) = o;
                }
            }
        }
        s ^= 1;
        if (s == 0) phase ^= 1;
    }
    if (!ok) {  // (whichever thread's wait ran out)
        set_err(a.err, DEV_ERR_TMA_TIMEOUT);
        // the copies in flight have to land before the block's shared memory goes away
        for (unsigned n = issued > 2 ? issued - 2 : 0; n < issued; ++n) mbar_wait(&full[n & 1], (n >> 1) & 1u);
    }
}

template <class T, int VEC, int NV, bool SAME, int THREADS>
cudaError_t launch_stream(const BlockNorm& a, int threads, int gate_rows, size_t smem, int sm_count, cudaStream_t st) {
    auto* fn = block_norm_stream_kernel<T, VEC, NV, SAME, THREADS>;
    cudaError_t e = set_max_dyn_smem((const void*)fn, 224 * 1024 * THREADS / 1024);
    if (e != cudaSuccess) return e;
    return launch_chained(fn, dim3(std::min(a.rows, sm_count * (1024 / THREADS))), dim3(threads), smem, st, a, gate_rows);
}

template <class T, int VEC, int NV, bool SAME>
cudaError_t launch_norm(const BlockNorm& a, int sm_count, cudaStream_t st) {
    const int n_pack = a.cols / VEC;
    if (n_pack <= 32 * NV) {
        const int grid = (int)std::min<long long>(((long long)a.rows + 7) / 8, (long long)sm_count * 32);
        return launch_chained(block_norm_kernel<T, VEC, NV, true, SAME, false, 256>, dim3(grid), dim3(32, 8), 0, st, a);
    }
    const int threads = ((n_pack + NV - 1) / NV + 31) / 32 * 32;
    if constexpr (VEC > 1) {
        // Streaming pays from two rows per resident block on, for rows long enough to hide a copy's latency; its outputs may
        // be the rows of h or y (a row is written after it was read) but not lie in rows that are read later.
        const int gate_rows = a.gate && a.gate_cols != 1 && a.gate_group == 1;
        const int resident = threads <= 256 ? 4 : (threads <= 512 ? 2 : 1);
        const size_t smem = 2 * (size_t)a.cols * sizeof(T) * (gate_rows ? 3 : 2);
        if (a.y && threads > 128 && a.rows >= 2 * resident * sm_count && smem <= (size_t)(224 * 1024 / resident)) {
            if (resident == 4) return launch_stream<T, VEC, NV, SAME, 256>(a, threads, gate_rows, smem, sm_count, st);
            if (resident == 2) return launch_stream<T, VEC, NV, SAME, 512>(a, threads, gate_rows, smem, sm_count, st);
            return launch_stream<T, VEC, NV, SAME, 1024>(a, threads, gate_rows, smem, sm_count, st);
        }
    }
    const int grid = (int)std::min<long long>(a.rows, (long long)sm_count * 32);
    auto go = [&](auto ahead) {
        constexpr bool A = decltype(ahead)::value;
        if (threads <= 256) return launch_chained(block_norm_kernel<T, VEC, NV, false, SAME, A, 256>, dim3(grid), dim3(threads), 0, st, a);
        return launch_chained(block_norm_kernel<T, VEC, NV, false, SAME, A, 512>, dim3(grid), dim3(threads), 0, st, a);
    };
    if (threads > 512) return launch_chained(block_norm_kernel<T, VEC, NV, false, SAME, false, 1024>, dim3(grid), dim3(threads), 0, st, a);
    return a.rows <= 4 * sm_count ? go(std::true_type{}) : go(std::false_type{});
}

template <class T>
cudaError_t launch_norm_t(const BlockNorm& a, int type, int sm_count, cudaStream_t st) {
    constexpr int VEC = 16 / (int)sizeof(T);
    // 16-byte accesses need every row of every operand to start on a multiple of 16 bytes; weights of the activation's type
    // are read the same way, others element by element.
    const size_t z = sizeof(T);
    auto fits = [&](const void* p, long long stride) { return !p || (((uintptr_t)p | (size_t)stride * z) & 15) == 0; };
    const bool vec = a.cols % VEC == 0 && fits(a.h, a.h_stride) && fits(a.y, a.y_stride) &&
                     fits(a.h_out, a.h_out_stride) && fits(a.n_out, a.n_out_stride) &&
                     (a.gate_cols == 1 || fits(a.gate, a.gate_stride));
    const bool same = a.w_type == type && fits(a.post_w, 0) && fits(a.pre_w, 0);
    if (!vec) return a.cols <= 8192 ? launch_norm<T, 1, 8, false>(a, sm_count, st) : launch_norm<T, 1, 16, false>(a, sm_count, st);
    // 16 elements a thread hold fewer threads to a row (two rows of 8192 share an SM); 8 where the registers of 16 f32
    // elements of three operands do not fit, and for few rows, whose latency more threads cut
    constexpr int WIDE = 16 / VEC, NARROW = 8 / VEC;
    const bool narrow = a.cols <= 8192 && (sizeof(T) == 4 || a.rows <= sm_count);
    if (narrow) return same ? launch_norm<T, VEC, NARROW, true>(a, sm_count, st) : launch_norm<T, VEC, NARROW, false>(a, sm_count, st);
    return same ? launch_norm<T, VEC, WIDE, true>(a, sm_count, st) : launch_norm<T, VEC, WIDE, false>(a, sm_count, st);
}

}  // namespace

cudaError_t launch_block_norm(const BlockNorm& a, int type, int sm_count, cudaStream_t st) {
    if (a.rows <= 0) return cudaSuccess;
    switch (type) {
        case LQ_T_F32: return launch_norm_t<float>(a, type, sm_count, st);
        case LQ_T_BF16: return launch_norm_t<__nv_bfloat16>(a, type, sm_count, st);
        case LQ_T_F16: return launch_norm_t<__half>(a, type, sm_count, st);
    }
    return cudaErrorInvalidValue;
}

}  // namespace lq
