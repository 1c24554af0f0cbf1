// The norms around a block of a decoder layer, fused with its gate and residual scale (lq_dev_block_norm):
//
//   z  = y / rms(y) * (off + post_w)            (z = y without the post norm)
//   h' = h_scale * h + y_scale * gate * z       (h' = h_scale * h without a block output)
//   n  = h' / rms(h') * (off + pre_w)           rms(v) = sqrt(mean(v^2) + eps)
//
// run_ffn's norm -> FFN -> residual add (crates/larql-compute/src/forward/layer.rs:61-127) with the post-FFN
// norm, the learned weights and the residual multiplier of layers that have them.
//
// Everything is kept in f32 between the loads and the stores (n is taken from the unrounded h'), the squares are
// summed in f64: v^2 of a bf16 or f32 activation can leave f32's range, and the sum costs nothing beside the loads.
// rms is at least sqrt(eps) >= 2^-63, so 1 / rms is a normal f32 and one multiply per element replaces a division.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/larql_cuda.h"
#include "kernels.h"

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

// Weights come in any of the three types, whatever the activation's: VEC of them as f32.
template <int VEC>
__device__ __forceinline__ void load_w(const void* w, int type, size_t at, float (&out)[VEC]) {
    if (type == LQ_T_F32) {
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

// Sum over the threads of a row: one warp (WARP) or the whole block.
template <bool WARP>
__device__ __forceinline__ double row_sum(double s, double* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (WARP) return s;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockDim.x >> 5;
    __syncthreads();  // the previous sum has been read
    if (lane == 0) red[warp] = s;
    __syncthreads();
    s = lane < n ? red[lane] : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}

// One row per warp (WARP: blockDim = 32 x rows) or per block; a thread holds NV packs of VEC elements.
template <class T, int VEC, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024) block_norm_kernel(const BlockNorm a) {
    __shared__ double red[32];
    const int tid = threadIdx.x, step = blockDim.x;
    const int n_pack = a.cols / VEC;
    const double inv_cols = 1.0 / (double)a.cols;
    using P = Pack<T, VEC>;
    const int rows_per = WARP ? blockDim.y : 1;
    for (int row = blockIdx.x * rows_per + (WARP ? threadIdx.y : 0); row < a.rows; row += gridDim.x * rows_per) {
        P h[NV], y[NV], g[NV];
        const T* hp = static_cast<const T*>(a.h) + (size_t)row * a.h_stride;
        const T* yp = static_cast<const T*>(a.y) + (a.y ? (size_t)row * a.y_stride : 0);
        const T* gp = static_cast<const T*>(a.gate) + (a.gate ? (size_t)(row / a.gate_group) * a.gate_stride : 0);
        const bool gate_vec = a.gate && a.gate_cols != 1;
        float gs = a.y_scale;
        if (a.gate && a.gate_cols == 1) gs *= to_f32(gp[0]);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int p = tid + i * step;
            if (p < n_pack) {
                if (a.y) y[i] = *reinterpret_cast<const P*>(yp + (size_t)p * VEC);
                h[i] = *reinterpret_cast<const P*>(hp + (size_t)p * VEC);
                if (gate_vec) g[i] = *reinterpret_cast<const P*>(gp + (size_t)p * VEC);
            }
        }
        float v[NV * VEC];
        float inv = 1.0f;
        if (a.post_norm) {
            double s = 0.0;
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (tid + i * step < n_pack)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const double d = (double)to_f32(y[i].v[j]);
                        s = fma(d, d, s);
                    }
            s = row_sum<WARP>(s, red);
            inv = (float)(1.0 / sqrt(s * inv_cols + a.eps));
        }
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int p = tid + i * step;
            if (p < n_pack) {
                float w[VEC];
                if (a.post_norm && a.post_w) load_w<VEC>(a.post_w, a.w_type, (size_t)p * VEC, w);
                P o;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    float x = a.h_scale * to_f32(h[i].v[j]);
                    if (a.y) {
                        float z = to_f32(y[i].v[j]);
                        if (a.post_norm) {
                            z *= inv;
                            if (a.post_w) z *= a.w_offset + w[j];
                        }
                        x = fmaf(gate_vec ? gs * to_f32(g[i].v[j]) : gs, z, x);
                    }
                    v[i * VEC + j] = x;
                    o.v[j] = from_f32<T>(x);
                    s = fma((double)x, (double)x, s);
                }
                if (a.h_out) *reinterpret_cast<P*>(static_cast<T*>(a.h_out) + (size_t)row * a.h_out_stride + (size_t)p * VEC) = o;
            }
        }
        if (a.n_out) {
            s = row_sum<WARP>(s, red);
            inv = (float)(1.0 / sqrt(s * inv_cols + a.eps));
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int p = tid + i * step;
                if (p < n_pack) {
                    float w[VEC];
                    if (a.pre_w) load_w<VEC>(a.pre_w, a.w_type, (size_t)p * VEC, w);
                    P o;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        float x = v[i * VEC + j] * inv;
                        if (a.pre_w) x *= a.w_offset + w[j];
                        o.v[j] = from_f32<T>(x);
                    }
                    *reinterpret_cast<P*>(static_cast<T*>(a.n_out) + (size_t)row * a.n_out_stride + (size_t)p * VEC) = o;
                }
            }
        }
    }
}

template <class T, int VEC, int NV>
cudaError_t launch_norm(const BlockNorm& a, int sm_count, cudaStream_t st) {
    const int n_pack = a.cols / VEC;
    if (n_pack <= 32 * NV) {
        const int grid = (int)min((long long)(a.rows + 7) / 8, (long long)sm_count * 32);
        block_norm_kernel<T, VEC, NV, true><<<grid, dim3(32, 8), 0, st>>>(a);
    } else {
        const int threads = ((n_pack + NV - 1) / NV + 31) / 32 * 32;
        const int grid = (int)min((long long)a.rows, (long long)sm_count * 32);
        block_norm_kernel<T, VEC, NV, false><<<grid, threads, 0, st>>>(a);
    }
    return cudaGetLastError();
}

template <class T>
cudaError_t launch_norm_t(const BlockNorm& a, int sm_count, cudaStream_t st) {
    constexpr int VEC = 16 / (int)sizeof(T);
    // 16-byte accesses need every row of every operand to start on one, weights included (a pack of VEC weights)
    const size_t z = sizeof(T), wz = a.w_type == LQ_T_F32 ? 4 : 2;
    auto fits = [&](const void* p, long long stride) { return !p || (((uintptr_t)p | (size_t)stride * z) & 15) == 0; };
    const bool vec = a.cols % VEC == 0 && fits(a.h, a.h_stride) && fits(a.y, a.y_stride) &&
                     fits(a.h_out, a.h_out_stride) && fits(a.n_out, a.n_out_stride) &&
                     (a.gate_cols == 1 || fits(a.gate, a.gate_stride)) &&
                     (((uintptr_t)a.post_w | (uintptr_t)a.pre_w) & (wz - 1)) == 0;
    if (vec) return launch_norm<T, VEC, 16 / VEC>(a, sm_count, st);
    return launch_norm<T, 1, 16>(a, sm_count, st);
}

}  // namespace

cudaError_t launch_block_norm(const BlockNorm& a, int type, int sm_count, cudaStream_t st) {
    if (a.rows <= 0) return cudaSuccess;
    switch (type) {
        case LQ_T_F32: return launch_norm_t<float>(a, sm_count, st);
        case LQ_T_BF16: return launch_norm_t<__nv_bfloat16>(a, sm_count, st);
        case LQ_T_F16: return launch_norm_t<__half>(a, sm_count, st);
    }
    return cudaErrorInvalidValue;
}

}  // namespace lq
