// Device-side pieces shared by the kernels of the selective layer (convolution, scan, norm): parameters of two
// widths, rows with an end inside a chunk, activations in float32, and column sums of partial gradients.
// Contract of the calls: include/fmselective.h.
#pragma once

#include "../../include/fmselective.h"
#include "fmscan_device.h"

namespace fmselective {

using fmscan::Elem;
using fmscan::f2u;
using fmscan::u2f;
using fmscan::u32x4;

constexpr float kLog2E = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// One value of a parameter: float32, or the inputs' element type where `narrow`
template <typename T>
__device__ __forceinline__ float param(const void* p, int64_t i, bool narrow) {
    return narrow ? Elem<T>::widen(reinterpret_cast<const T*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
}
template <typename T>
__device__ __forceinline__ void put(void* p, int64_t i, bool narrow, float v) {
    if (narrow) reinterpret_cast<T*>(p)[i] = (T)v;
    else reinterpret_cast<float*>(p)[i] = v;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float sigmoid(float x) {
    return __builtin_amdgcn_rcpf(1.0f + exp2_fast(-kLog2E * x));
}
// d/dx x sigmoid(x), from x and sigmoid(x)
__device__ __forceinline__ float silu_slope(float x, float s) { return s * __builtin_fmaf(x, 1.0f - s, 1.0f); }

// The steps that count of batch element b
__device__ __forceinline__ int64_t row_length(const int32_t* __restrict__ lengths, int64_t b, int64_t L) {
    if (!lengths) return L;
    const int64_t n = lengths[b];
    return n < 0 ? 0 : (n > L ? L : n);
}

// C consecutive values from t0 of a row of which `len` count, the others as zeros (not read)
template <typename T, int C>
__device__ __forceinline__ void load_values(const T* __restrict__ row, int64_t t0, int64_t len, float (&f)[C]) {
    constexpr int E = Elem<T>::E;
    static_assert(C % E == 0, "whole chunks");
#pragma unroll
    for (int i = 0; i < C / E; ++i) {
        float part[E];
        Elem<T>::unpack(fmscan::load_chunk<T, false, false>(row, t0 + i * E, len, 0u), part);
#pragma unroll
        for (int k = 0; k < E; ++k) f[i * E + k] = part[k];
    }
}
template <typename T, int C>
__device__ __forceinline__ void store_values(T* __restrict__ row, int64_t t0, int64_t L, const float (&f)[C]) {
    constexpr int E = Elem<T>::E;
#pragma unroll
    for (int i = 0; i < C / E; ++i) {
        float part[E];
#pragma unroll
        for (int k = 0; k < E; ++k) part[k] = f[i * E + k];
        fmscan::store_chunk<T, false>(row, t0 + i * E, L, Elem<T>::pack(part));
    }
}

// Sums by DPP, a lane's source outside its row being zero
template <int CTRL, int ROW_MASK = 0xf>
__device__ __forceinline__ float dpp_or_zero(float v) {
    return u2f((uint32_t)__builtin_amdgcn_update_dpp(0, (int)f2u(v), CTRL, ROW_MASK, 0xf, ROW_MASK == 0xf));
}
// Lane 15 of each row of 16: the sum over the row
__device__ __forceinline__ float row_sum(float v) {
    v += dpp_or_zero<0x111>(v);  // row_shr 1, 2, 4, 8
    v += dpp_or_zero<0x112>(v);
    v += dpp_or_zero<0x114>(v);
    v += dpp_or_zero<0x118>(v);
    return v;
}
// Lane 63: the sum over the wave
__device__ __forceinline__ float wave_sum_high(float v) {
    v = row_sum(v);
    v += dpp_or_zero<0x142, 0xa>(v);  // row_bcast 15 into rows 1 and 3
    v += dpp_or_zero<0x143, 0xc>(v);  // row_bcast 31 into rows 2 and 3
    return v;
}

// The slot of row b of a single-token call, or -1: the row is skipped (see fmselective.h). Called by the whole
// block, for one b: an earlier row with the same slot is looked for by all its threads.
__device__ __forceinline__ int64_t slot_of_row(const void* __restrict__ slots, bool wide, int32_t b, int64_t S) {
    if (!slots) return b;
    auto at = [&](int32_t i) {
        return wide ? reinterpret_cast<const int64_t*>(slots)[i] : (int64_t)reinterpret_cast<const int32_t*>(slots)[i];
    };
    const int64_t slot = at(b);
    bool taken = slot < 0 || slot >= S;
    for (int32_t i = threadIdx.x; i < b; i += blockDim.x) taken |= at(i) == slot;
    return __syncthreads_or(taken) ? -1 : slot;
}

// ---- column sums -----------------------------------------------------------------------------------------
// out[c] = sum over i < n of src[i * cols + c], rounded once to the type of `out`. The partial sums that the
// blocks of a backward kernel leave are added in a fixed order: the same inputs give the same bits.
struct ColumnSum {
    const float* src;
    void* out;
    int64_t n, cols;
    int32_t narrow;
    uint32_t first_block;  // of this section in the launch
};
constexpr int kSumSections = 3;
struct ColumnSums {
    ColumnSum part[kSumSections];
};
constexpr int kSumWaves = 16;

template <typename T>
__device__ __forceinline__ void column_sums(const ColumnSums& s, uint32_t block) {
    int which = 0;
#pragma unroll
    for (int i = 1; i < kSumSections; ++i)
        if (s.part[i].src && block >= s.part[i].first_block) which = i;
    const ColumnSum& p = s.part[which];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = (int64_t)(block - p.first_block) * 64 + lane;
    float sum = 0.0f;
    if (c < p.cols) {
#pragma unroll 8
        for (int64_t i = wave; i < p.n; i += kSumWaves) sum += p.src[i * p.cols + c];
    }
    __shared__ float shared[kSumWaves][64];
    shared[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && c < p.cols) {
#pragma unroll
        for (int w = 1; w < kSumWaves; ++w) sum += shared[w][lane];
        put<T>(p.out, c, p.narrow != 0, sum);
    }
}
template <typename T>
__global__ __launch_bounds__(64 * kSumWaves) void column_sums_kernel(ColumnSums s) {
    column_sums<T>(s, blockIdx.x);
}

}  // namespace fmselective
