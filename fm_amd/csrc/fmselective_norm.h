// Kernels of the root-mean-square norm with the residual's addition: forward (output in the inputs' type, or e4m3
// with one scale a row) and backward.
//
// Both are bound by memory: every stream is moved once. In bf16 at (8192, 4096) forward with a residual takes 45 us
// (268 MB, 5.9 TB/s with what the last-level cache keeps), backward with the stream's gradient 51 us (268 MB, 5.3 TB/s);
// the output in 8 bits at (4096, 5120) 32 us (147 MB, 4.6 TB/s). A row stays in registers between the sum of squares and
// its use: TPR threads a row (a wave for short rows, a block for long ones), CH chunks of 16 bytes a thread.
// What the norm sees is the sum as it is stored, rounded to the stream's type: the backward pass, which has
// only the stored stream, is then the gradient of exactly what forward computed.
#pragma once

#include "fmselective_device.h"

namespace fmselective {

constexpr float kE4m3Max = 448.0f;
// A row whose largest value is below this is quantised to zeros with scale 0 (its scale's reciprocal would leave
// the range of float32)
constexpr float kE4m3Least = 0x1p-100f;

// E values of the weight from element i (dense, any alignment)
template <typename T>
__device__ __forceinline__ void load_weight(const void* w, int64_t i, int64_t D, bool narrow, float (&f)[Elem<T>::E]) {
    constexpr int E = Elem<T>::E;
    if (narrow) {
        load_values<T, E>(reinterpret_cast<const T*>(w), i, D, f);
    } else {
        load_values<float, E>(reinterpret_cast<const float*>(w), i, D, f);
    }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) v += __shfl_xor(v, s);
    return v;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)v, s);
        v = o > v ? o : v;
    }
    return v;
}
// over the TPR threads of a row; `shared` holds a word a wave, and may be used again after the next barrier
template <int TPR>
__device__ __forceinline__ float row_total(float v, float* shared) {
    v = wave_sum(v);
    if constexpr (TPR > 64) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) shared[wave] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < TPR / 64; ++w) v += shared[w];
    }
    return v;
}
template <int TPR>
__device__ __forceinline__ uint32_t row_top(uint32_t v, uint32_t* shared) {
    v = wave_max(v);
    if constexpr (TPR > 64) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) shared[wave] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int w = 0; w < TPR / 64; ++w) v = shared[w] > v ? shared[w] : v;
    }
    return v;
}

// E values to e4m3, rounded to nearest even
template <int E>
__device__ __forceinline__ void store_e4m3(uint8_t* __restrict__ row, int64_t t0, int64_t D, const float (&f)[E]) {
    uint32_t words[E / 4];
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i], f[4 * i + 1], 0, false);
        words[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2], f[4 * i + 3], w, true);
    }
    if (t0 + E <= D) {
        typedef uint32_t loose __attribute__((ext_vector_type(E / 4), aligned(1)));
        loose v;
        if constexpr (E == 8) { v.x = words[0]; v.y = words[1]; }
        else v = words[0];
        *reinterpret_cast<loose*>(row + t0) = v;
    } else {
#pragma unroll
        for (int k = 0; k < E; ++k)
            if (t0 + k < D) row[t0 + k] = (uint8_t)(words[k / 4] >> (8 * (k & 3)));
    }
}

template <typename T, int TPR, int CH, bool QUANT>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void norm_forward_kernel(const T* __restrict__ inputs,
                                                                             const T* __restrict__ residual,
                                                                             const void* __restrict__ weight,
                                                                             T* __restrict__ residual_out, void* __restrict__ out,
                                                                             float* __restrict__ scales, float* __restrict__ inv_rms,
                                                                             int64_t rows, int32_t D, float eps, unsigned flags) {
    constexpr int E = Elem<T>::E, RPB = TPR == 64 ? 4 : 1;
    __shared__ float shared[2][TPR / 64];
    const int i = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
    if (RPB > 1 && row >= rows) return;
    const T* x = inputs + row * D;
    float h[CH][E], w[CH][E], sum = 0.0f;
    fmscan::u32x4 raw[CH], res[CH];
#pragma unroll
    for (int j = 0; j < CH; ++j) raw[j] = fmscan::load_chunk<T, false, true>(x, ((int64_t)j * TPR + i) * E, D, 0u);
    if (residual) {
#pragma unroll
        for (int j = 0; j < CH; ++j) res[j] = fmscan::load_chunk<T, false, true>(residual + row * D, ((int64_t)j * TPR + i) * E, D, 0u);
    }
#pragma unroll
    for (int j = 0; j < CH; ++j) load_weight<T>(weight, ((int64_t)j * TPR + i) * E, D, flags & FMSELECTIVE_NARROW_WEIGHT, w[j]);
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        Elem<T>::unpack(raw[j], h[j]);
        if (residual) {
            float r[E];
            Elem<T>::unpack(res[j], r);
#pragma unroll
            for (int k = 0; k < E; ++k) h[j][k] += r[k];
            const fmscan::u32x4 packed = Elem<T>::pack(h[j]);
            fmscan::store_chunk<T, false>(residual_out + row * D, ((int64_t)j * TPR + i) * E, D, packed);
            Elem<T>::unpack(packed, h[j]);
        }
#pragma unroll
        for (int k = 0; k < E; ++k) sum = __builtin_fmaf(h[j][k], h[j][k], sum);
    }
    sum = row_total<TPR>(sum, shared[0]);
    const float mean = sum / (float)D + eps;
    const float inv = mean == 0.0f ? 0.0f : rsqrtf(mean);  // (a row of zeros without eps is zeros; the mean may be subnormal)
    if (inv_rms && i == 0) inv_rms[row] = inv;
#pragma unroll
    for (int j = 0; j < CH; ++j)
#pragma unroll
        for (int k = 0; k < E; ++k) h[j][k] = h[j][k] * inv * w[j][k];
    if constexpr (!QUANT) {
#pragma unroll
        for (int j = 0; j < CH; ++j) store_values<T, E>((T*)out + row * D, ((int64_t)j * TPR + i) * E, D, h[j]);
    } else {
        uint32_t top = 0;  // of the magnitudes' bits: a NaN is above every number and is kept
#pragma unroll
        for (int j = 0; j < CH; ++j)
#pragma unroll
            for (int k = 0; k < E; ++k) {
                const uint32_t m = f2u(h[j][k]) & 0x7fffffffu;
                top = m > top ? m : top;
            }
        const float amax = u2f(row_top<TPR>(top, reinterpret_cast<uint32_t*>(shared[1])));
        const bool nothing = amax < kE4m3Least;
        const float up = nothing ? 0.0f : kE4m3Max / amax;
        if (i == 0) scales[row] = nothing ? 0.0f : amax / kE4m3Max;
#pragma unroll
        for (int j = 0; j < CH; ++j) {
#pragma unroll
            for (int k = 0; k < E; ++k) h[j][k] *= up;
            store_e4m3<E>((uint8_t*)out + row * D, ((int64_t)j * TPR + i) * E, D, h[j]);
        }
    }
}

// dr = dresidual + (dy w - x mean(dy w x)) / rms with x = r / rms;  dweight = sum over the rows of dy x.
// A block (a wave, for short rows) takes every slots-th row and keeps its part of the weight's gradient in registers;
// each block leaves one part.
template <typename T, int TPR, int CH>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void norm_backward_kernel(const T* __restrict__ out_grad,
                                                                              const T* __restrict__ residual_grad,
                                                                              const T* __restrict__ stream_in,
                                                                              const void* __restrict__ weight,
                                                                              const float* __restrict__ inv_rms,
                                                                              T* __restrict__ grad, float* __restrict__ weight_part,
                                                                              int64_t rows, int32_t D, unsigned flags) {
    constexpr int E = Elem<T>::E, RPB = TPR == 64 ? 4 : 1;
    __shared__ float shared[2][TPR / 64];
    const int i = threadIdx.x % TPR;
    const int64_t slot = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR, slots = (int64_t)gridDim.x * RPB;
    float w[CH][E], dw[CH][E];
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        load_weight<T>(weight, ((int64_t)j * TPR + i) * E, D, flags & FMSELECTIVE_NARROW_WEIGHT, w[j]);
#pragma unroll
        for (int k = 0; k < E; ++k) dw[j][k] = 0.0f;
    }
    int turn = 0;
    for (int64_t row = slot; row < rows; row += slots, turn ^= 1) {
        fmscan::u32x4 gy[CH], xr[CH], gr[CH];
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            const int64_t at = ((int64_t)j * TPR + i) * E;
            gy[j] = fmscan::load_chunk<T, false, true>(out_grad + row * D, at, D, 0u);
            xr[j] = fmscan::load_chunk<T, false, true>(stream_in + row * D, at, D, 0u);
            if (residual_grad) gr[j] = fmscan::load_chunk<T, false, true>(residual_grad + row * D, at, D, 0u);
        }
        const float inv = inv_rms[row];
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            float y[E], x[E];
            Elem<T>::unpack(gy[j], y);
            Elem<T>::unpack(xr[j], x);
#pragma unroll
            for (int k = 0; k < E; ++k) {
                x[k] *= inv;
                sum = __builtin_fmaf(y[k] * w[j][k], x[k], sum);
                dw[j][k] = __builtin_fmaf(y[k], x[k], dw[j][k]);
            }
        }
        const float mean = row_total<TPR>(sum, shared[turn]) / (float)D;
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            float y[E], x[E], g[E];
            Elem<T>::unpack(gy[j], y);
            Elem<T>::unpack(xr[j], x);
            if (residual_grad) Elem<T>::unpack(gr[j], g);
#pragma unroll
            for (int k = 0; k < E; ++k) {
                const float v = inv * __builtin_fmaf(-(x[k] * inv), mean, y[k] * w[j][k]);
                g[k] = residual_grad ? g[k] + v : v;
            }
            store_values<T, E>(grad + row * D, ((int64_t)j * TPR + i) * E, D, g);
        }
    }
    float* part = weight_part + (int64_t)blockIdx.x * D;
    if constexpr (RPB > 1) {  // the block's waves hold parts of the same columns
        __shared__ float held[RPB - 1][CH][E][64];
        const int wave = threadIdx.x >> 6;
        if (wave) {
#pragma unroll
            for (int j = 0; j < CH; ++j)
#pragma unroll
                for (int k = 0; k < E; ++k) held[wave - 1][j][k][i] = dw[j][k];
        }
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int w = 0; w < RPB - 1; ++w)
#pragma unroll
            for (int j = 0; j < CH; ++j)
#pragma unroll
                for (int k = 0; k < E; ++k) dw[j][k] += held[w][j][k][i];
    }
#pragma unroll
    for (int j = 0; j < CH; ++j) store_values<float, E>(part, ((int64_t)j * TPR + i) * E, D, dw[j]);
}

}  // namespace fmselective
