// Kernels of the short depthwise convolution along time: forward, backward, one token.
//
// A row is read once and written once, W <= 4 multiply-adds an element: forward and the single token's call are bound by
// memory. Backward does 33 vector instructions an element (bf16, silu) beside 6 bytes and comes to the limit of both at once.
#pragma once

#include "fmselective_device.h"

#include <type_traits>

namespace fmselective {

// W - 1 values before chunk position t0 of a row: the row's own where t0 > 0 (a chunk has at least 4 elements and
// chunks start at multiples of that, so t0 >= 4), else the carried state's, else zeros.
template <typename T, int W>
__device__ __forceinline__ void values_before(const T* __restrict__ row, int64_t t0, int64_t len,
                                              const T* __restrict__ state, float (&f)[W - 1]) {
    if (t0 > 0) {
        if (t0 > len) {  // nothing of this chunk counts
#pragma unroll
            for (int i = 0; i < W - 1; ++i) f[i] = 0.0f;
        } else if constexpr (sizeof(T) == 4) {
            const u32x4 v = fmscan::load16<T, false, false>(row + t0 - 4);
#pragma unroll
            for (int i = 0; i < W - 1; ++i) f[i] = u2f(v[i + 5 - W]);
        } else {
            typedef uint32_t u32x2_at2 __attribute__((ext_vector_type(2), aligned(2)));
            const u32x2_at2 v = *reinterpret_cast<const u32x2_at2*>(row + t0 - 4);
            u32x4 wide = {v.x, v.y, 0u, 0u};
            float four[8];
            Elem<T>::unpack(wide, four);
#pragma unroll
            for (int i = 0; i < W - 1; ++i) f[i] = four[i + 5 - W];
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < W - 1; ++i) f[i] = state ? Elem<T>::widen(state[i]) : 0.0f;
}

template <typename T, int W>
__device__ __forceinline__ void conv_taps(const void* weight, const void* bias, int64_t d, unsigned flags,
                                          float (&w)[W], float& b) {
#pragma unroll
    for (int j = 0; j < W; ++j) w[j] = param<T>(weight, d * W + j, flags & FMSELECTIVE_NARROW_WEIGHT);
    b = bias ? param<T>(bias, d, flags & FMSELECTIVE_NARROW_BIAS) : 0.0f;
}

struct ConvRows {
    int64_t batch_stride, channel_stride, L;
    int32_t rows, D;
    uint32_t units;           // of 64 * CH chunks a row has, a wave each (long rows)
    uint32_t rows_per_block;  // (short rows)
    uint32_t chunks;          // of a row
    uint32_t magic;           // ceil(2^16 / chunks) (short rows)
};

// A chunk's outputs from its inputs and the W - 1 values before it
template <typename T, int W>
__device__ __forceinline__ void conv_chunk(const float (&f)[Elem<T>::E], const float (&before)[W - 1], const float (&w)[W], float bias,
                                           bool silu, float (&y)[Elem<T>::E]) {
    auto at = [&](int i) { return i < 0 ? before[i + W - 1] : f[i]; };
#pragma unroll
    for (int k = 0; k < Elem<T>::E; ++k) {
        float v = bias;
#pragma unroll
        for (int j = 0; j < W; ++j) v = __builtin_fmaf(w[j], at(k - (W - 1) + j), v);
        y[k] = v;
    }
    if (silu) {
#pragma unroll
        for (int k = 0; k < Elem<T>::E; ++k) y[k] *= sigmoid(y[k]);
    }
}

template <typename T, int W>
__device__ __forceinline__ void conv_final_state(const T* __restrict__ x, const T* __restrict__ state, int64_t len, T* __restrict__ to) {
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
        const int64_t p = len - (W - 1) + i;
        to[i] = p >= 0 ? x[p] : (state ? state[p + W - 1] : (T)0.0f);
    }
}

// Rows of at most 64 chunks of 16 bytes: a chunk a thread, as many whole rows a block as it has threads for. The W - 1
// values before a chunk are a second, 8-byte load that the L1 answers. Bound by memory: 57 us at (64, 4096, 256) in bf16,
// 4.7 TB/s; rows off the 16-byte grid 65 us at (64, 4096, 255), 80 at (256, 4096, 65). A wave for every row, as below,
// takes 146, 160 and 540 us there.
template <typename T, int W>
__global__ __launch_bounds__(256) void conv_forward_short_kernel(const T* __restrict__ inputs, const void* __restrict__ weight,
                                                                 const void* __restrict__ bias, const T* __restrict__ initial,
                                                                 const int32_t* __restrict__ lengths, T* __restrict__ out,
                                                                 T* __restrict__ final_state, ConvRows g, unsigned flags) {
    constexpr int E = Elem<T>::E;
    const uint32_t r = (threadIdx.x * g.magic) >> 16;
    const uint32_t row = blockIdx.x * g.rows_per_block + r, chunk = threadIdx.x - r * g.chunks;
    if (r >= g.rows_per_block || row >= (uint32_t)g.rows) return;
    const uint32_t b = row / (uint32_t)g.D, d = row - b * g.D;
    const int64_t len = row_length(lengths, b, g.L), t0 = (int64_t)chunk * E;
    const T* x = inputs + b * g.batch_stride + d * g.channel_stride;
    const T* state = initial ? initial + (int64_t)row * (W - 1) : nullptr;
    float w[W], bv, f[E], before[W - 1], y[E];
    load_values<T, E>(x, t0, len, f);
    values_before<T, W>(x, t0, len, state, before);
    conv_taps<T, W>(weight, bias, d, flags, w, bv);
    conv_chunk<T, W>(f, before, w, bv, flags & FMSELECTIVE_SILU, y);
#pragma unroll
    for (int k = 0; k < E; ++k) y[k] = t0 + k < len ? y[k] : 0.0f;
    store_values<T, E>(out + (int64_t)row * g.L, t0, g.L, y);
    if (final_state && chunk == 0) conv_final_state<T, W>(x, state, len, final_state + (int64_t)row * (W - 1));
}

// Long rows: a wave takes CH * 64 chunks of a row, all its loads in flight at once; a lane's values before its chunk come
// from the lane below, lane 0's from lane 63 of the chunks before, and from memory once a wave. Bound by memory:
// 44 us at (8, 4096, 2048) in bf16, 6.1 TB/s with what the last-level cache keeps of 134 MB of inputs.
template <typename T, int W, int CH>
__global__ __launch_bounds__(256) void conv_forward_kernel(const T* __restrict__ inputs, const void* __restrict__ weight,
                                                           const void* __restrict__ bias, const T* __restrict__ initial,
                                                           const int32_t* __restrict__ lengths, T* __restrict__ out,
                                                           T* __restrict__ final_state, ConvRows g, unsigned flags) {
    constexpr int E = Elem<T>::E;
    const int lane = threadIdx.x & 63;
    const uint32_t at = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const uint32_t row = at / g.units, unit = at - row * g.units;
    if (row >= (uint32_t)g.rows) return;
    const uint32_t b = row / (uint32_t)g.D, d = row - b * g.D;
    const int64_t len = row_length(lengths, b, g.L), start = (int64_t)unit * (CH * 64 * E);
    const T* x = inputs + b * g.batch_stride + d * g.channel_stride;
    const T* state = initial ? initial + (int64_t)row * (W - 1) : nullptr;
    T* y_row = out + (int64_t)row * g.L;
    const bool full = start + CH * 64 * E <= len;
    u32x4 raw[CH];
    if (full) {
#pragma unroll
        for (int j = 0; j < CH; ++j) raw[j] = fmscan::load16<T, true, false>(x + start + (j * 64 + lane) * E);
    } else {
#pragma unroll
        for (int j = 0; j < CH; ++j) raw[j] = fmscan::load_chunk<T, false, false>(x, start + (j * 64 + lane) * E, len, 0u);
    }
    float w[W], bv, first[W - 1];
#pragma unroll
    for (int i = 0; i < W - 1; ++i) first[i] = 0.0f;
    if (lane == 0) values_before<T, W>(x, start, len, state, first);
    conv_taps<T, W>(weight, bias, d, flags, w, bv);
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        float f[E], before[W - 1], y[E];
        Elem<T>::unpack(raw[j], f);
#pragma unroll
        for (int i = 0; i < W - 1; ++i) {
            before[i] = fmscan::dpp<fmscan::kWaveShr1>(first[i], f[E - (W - 1) + i]);  // lane 0 keeps `first`
            first[i] = fmscan::lane63(f[E - (W - 1) + i]);
        }
        conv_chunk<T, W>(f, before, w, bv, flags & FMSELECTIVE_SILU, y);
        const int64_t t0 = start + (j * 64 + lane) * E;
        if (full) {
            fmscan::store16<T, false>(y_row + t0, Elem<T>::pack(y));
        } else {
#pragma unroll
            for (int k = 0; k < E; ++k) y[k] = t0 + k < len ? y[k] : 0.0f;
            store_values<T, E>(y_row, t0, g.L, y);
        }
    }
    if (final_state && unit == 0 && lane == 0) conv_final_state<T, W>(x, state, len, final_state + (int64_t)row * (W - 1));
}

struct ConvBack {
    int64_t batch_stride, channel_stride, grad_batch_stride, grad_channel_stride, L;
    int32_t rows, B, D;
    int32_t chunks;       // of a row
    int32_t parts;        // of the parameters' gradients, each (D, W) and (D)
    // short rows
    int32_t row_lanes_magic, rows_per_wave, groups, each;  // ceil(2^16 / chunks); groups of rows_per_wave channels; batch elements a wave
    // long rows
    int32_t tiles, segments, seg_tiles;  // tiles of 64 chunks
};

// The steps of a chunk from t0 that lie before `end`
template <int E>
__device__ __forceinline__ int steps_before(int64_t t0, int64_t end) {
    const int64_t n = end - t0;
    return n < 0 ? 0 : (n > E ? E : (int)n);
}

// The 16 bytes from element t0 of a row of which `len` elements count, the others as zeros (not read). At the row's end one
// load of its last 16 bytes, shifted, instead of loads one by one, which wait for each other: backward at
// (16, 4096, 1021) in bf16 133 -> 111 us, (64, 4096, 255) 144 -> 110. (Rows of whole chunks pay 2 us of 75 for it; forward
// gains nothing, and the scan and the norm lose more registers by it than the loads cost.)
template <typename T>
__device__ __forceinline__ u32x4 load_part(const T* __restrict__ row, int64_t t0, int64_t len) {
    constexpr int E = Elem<T>::E;
    if (len < E) {  // a row shorter than a chunk
        uint64_t half[2] = {0, 0};
        using Bits = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;
#pragma unroll 1
        for (int64_t k = t0; k < len; ++k) {
            const uint64_t v = (uint64_t)reinterpret_cast<const Bits*>(row)[k] << (8 * sizeof(T) * (k & (E / 2 - 1)));
            if (k < E / 2) half[0] |= v;
            else half[1] |= v;
        }
        return u32x4{(uint32_t)half[0], (uint32_t)(half[0] >> 32), (uint32_t)half[1], (uint32_t)(half[1] >> 32)};
    }
    const int64_t from = t0 + E <= len ? t0 : len - E;
    u32x4 v = fmscan::load16<T, false, false>(row + from);
    if (t0 > from) {  // the first t0 - from elements belong to the chunk before
        const int s = t0 - from < E ? (int)(t0 - from) : E;
        const int words = E == 8 ? s >> 1 : s;
        if (words & 2) v = u32x4{v.z, v.w, 0u, 0u};
        if (words & 1) v = u32x4{v.y, v.z, v.w, 0u};
        if (E == 8 && (s & 1))
            v = u32x4{v.x >> 16 | v.y << 16, v.y >> 16 | v.z << 16, v.z >> 16 | v.w << 16, v.w >> 16};
        if (s == E) v = u32x4{0u, 0u, 0u, 0u};
    }
    return v;
}

// What backward does with a lane's chunk, of which `left` steps count. dpre[k]: the gradient of the sum before the
// activation, computed once an element; the H from beyond the chunk come from the next lane, or are `behind` where `last`.
// dw and db: the parameters' gradients of this lane so far. `whole`: the same in all lanes, all their steps count.
template <typename T, int W>
__device__ __forceinline__ void conv_chunk_back(const float (&f)[Elem<T>::E], const float (&gy)[Elem<T>::E], const float (&before)[W - 1],
                                                const float (&w)[W], float bias, bool silu, int left, bool whole, bool last,
                                                const float (&behind)[W - 1], float (&dpre)[Elem<T>::E + W - 1], float (&dw)[W],
                                                float& db, float (&dx)[Elem<T>::E]) {
    constexpr int E = Elem<T>::E, H = W - 1;
    auto at = [&](int p) { return p < 0 ? before[p + H] : f[p]; };
#pragma unroll
    for (int k = 0; k < E; ++k) dpre[k] = gy[k];
    if (silu) {
        float pre[E];
#pragma unroll
        for (int k = 0; k < E; ++k) {
            pre[k] = bias;
#pragma unroll
            for (int j = 0; j < W; ++j) pre[k] = __builtin_fmaf(w[j], at(k - H + j), pre[k]);
        }
#pragma unroll
        for (int k = 0; k < E; ++k) dpre[k] = gy[k] * silu_slope(pre[k], sigmoid(pre[k]));
    }
    if (whole) {
#pragma unroll
        for (int k = 0; k < E; ++k)
#pragma unroll
            for (int j = 0; j < W; ++j) dw[j] = __builtin_fmaf(dpre[k], at(k - H + j), dw[j]);
    } else {  // (a step that does not count adds nothing, whatever stands before it)
#pragma unroll
        for (int k = 0; k < E; ++k) {
            const bool in = k < left;
            dpre[k] = in ? dpre[k] : 0.0f;
#pragma unroll
            for (int j = 0; j < W; ++j) dw[j] = __builtin_fmaf(dpre[k], in ? at(k - H + j) : 0.0f, dw[j]);
        }
    }
#pragma unroll
    for (int k = 0; k < E; ++k) db += dpre[k];
#pragma unroll
    for (int k = 0; k < H; ++k) {
        const float next = fmscan::dpp<fmscan::kWaveShl1>(0.0f, dpre[k]);
        dpre[E + k] = last ? behind[k] : next;
    }
#pragma unroll
    for (int k = 0; k < E; ++k) {
        dx[k] = 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) dx[k] = __builtin_fmaf(w[j], dpre[k + H - j], dx[k]);
    }
    if (!whole) {
#pragma unroll
        for (int k = 0; k < E; ++k) dx[k] = k < left ? dx[k] : 0.0f;
    }
}

// The final state's gradient, where it reaches a chunk from t0 of a row of `len` steps
template <typename T, int H>
__device__ __forceinline__ void add_final_grad(const T* fg, int64_t t0, int64_t len, float (&dx)[Elem<T>::E]) {
    const int64_t first = len - H - t0;  // the state's oldest value stands here in the chunk
    if (first >= Elem<T>::E || len <= t0) return;
#pragma unroll
    for (int k = 0; k < Elem<T>::E; ++k)
        if (k >= first && t0 + k < len) dx[k] += Elem<T>::widen(fg[k - first]);
}
// The initial state's gradient, from the first steps' dpre
template <typename T, int W>
__device__ __forceinline__ void put_initial_grad(const float* dpre, const float (&w)[W], const T* fg, int64_t len, T* to) {
    constexpr int H = W - 1;
#pragma unroll
    for (int i = 0; i < H; ++i) {
        float v = 0.0f;
        if (len > 0) {
#pragma unroll
            for (int j = 0; j <= i; ++j) v = __builtin_fmaf(w[j], dpre[i - j], v);
        }
        if (fg && i >= len) v += Elem<T>::widen(fg[i - len]);
        to[i] = (T)v;
    }
}

// Rows of at most 64 chunks: a chunk a lane, as many channels side by side in a wave as it has lanes for. A wave keeps its
// channels and walks over batch elements, the next one's chunks in flight, so that the parameters' gradients are summed
// in registers and over the lanes once for all of them. In bf16 80 us at (256, 4096, 64), 5.0 TB/s, and 125 us at
// (256, 4096, 65), where a wave for every row, its lanes a power of two, takes 210 and 495.
template <typename T, int W>
__global__ __launch_bounds__(256) void conv_backward_short_kernel(const T* __restrict__ inputs, const T* __restrict__ out_grad,
                                                                  const void* __restrict__ weight, const void* __restrict__ bias,
                                                                  const T* __restrict__ initial, const T* __restrict__ final_grad,
                                                                  const int32_t* __restrict__ lengths, T* __restrict__ inputs_grad,
                                                                  T* __restrict__ initial_grad, float* __restrict__ weight_part,
                                                                  float* __restrict__ bias_part, ConvBack g, unsigned flags) {
    constexpr int E = Elem<T>::E, H = W - 1;
    const int lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const int32_t part = wave / (uint32_t)g.groups, group = wave - part * g.groups;
    if (part >= g.parts) return;
    const int r = (lane * g.row_lanes_magic) >> 16, c = lane - r * g.chunks;
    const int32_t want = group * g.rows_per_wave + r;
    const bool live = r < g.rows_per_wave && want < g.D;
    const int32_t d = live ? want : g.D - 1;  // (a lane without a row loads and stores nothing)
    const int64_t t0 = (int64_t)c * E, mine = live ? g.L : 0;
    const bool silu = flags & FMSELECTIVE_SILU, last = c == g.chunks - 1;
    const float zeros[H] = {};
    float w[W], bv, dw[W] = {}, db = 0.0f, dpre[E + H];
    conv_taps<T, W>(weight, bias, d, flags, w, bv);
    const int32_t b0 = part * g.each, b1 = b0 + g.each < g.B ? b0 + g.each : g.B;
    const T* x = inputs + d * g.channel_stride;
    const T* dy = out_grad + d * g.grad_channel_stride;
    u32x4 next_x, next_dy;
    int64_t next_len;
    auto fetch = [&](int32_t b) {
        next_len = row_length(lengths, b, g.L);
        next_x = load_part<T>(x + b * g.batch_stride, t0, live ? next_len : 0);
        next_dy = load_part<T>(dy + b * g.grad_batch_stride, t0, live ? next_len : 0);
    };
    fetch(b0);
    for (int32_t b = b0; b < b1; ++b) {
        const int64_t len = next_len, row = (int64_t)b * g.D + d;
        float f[E], gy[E], before[H], dx[E];
        Elem<T>::unpack(next_x, f);
        Elem<T>::unpack(next_dy, gy);
        if (b + 1 < b1) fetch(b + 1);
#pragma unroll
        for (int k = 0; k < H; ++k) {
            const float below = fmscan::dpp<fmscan::kWaveShr1>(0.0f, f[E - H + k]);
            before[k] = c == 0 ? (initial && live ? Elem<T>::widen(initial[row * H + k]) : 0.0f) : below;
        }
        const int left = live ? steps_before<E>(t0, len) : 0;
        conv_chunk_back<T, W>(f, gy, before, w, bv, silu, left, __all(left == E || !live), last, zeros, dpre, dw, db, dx);
        if (final_grad && live) add_final_grad<T, H>(final_grad + row * H, t0, len, dx);
        store_values<T, E>(inputs_grad + row * g.L, t0, mine, dx);
        if (initial_grad && live && c == 0)
            put_initial_grad<T, W>(dpre, w, final_grad ? final_grad + row * H : nullptr, len, initial_grad + row * H);
    }
    // the first lane of a row's chunks: the sum over them
    auto over_chunks = [&](float v) {
        for (int s = 1; s < g.chunks; s *= 2) {
            const float other = __shfl_down(v, s);
            v += c + s < g.chunks ? other : 0.0f;
        }
        return v;
    };
    const int64_t at = (int64_t)part * g.D + d;
#pragma unroll
    for (int j = 0; j < W; ++j) {
        const float v = over_chunks(dw[j]);
        if (live && c == 0) weight_part[at * W + j] = v;
    }
    db = over_chunks(db);
    if (live && c == 0) bias_part[at] = db;
}

// Long rows: a wave walks a row, or a segment of one, from its end to its start, a tile of 64 chunks after the other, up to
// four in flight. What the last lane needs from behind a tile is kept from the tile before. The gradients of weight and bias
// are summed over the whole walk in registers and across the lanes once. In bf16 72 us at (8, 4096, 2048), 5.6 TB/s; rows of
// two tiles 88 us at (16, 4096, 1024).
template <typename T, int W>
__global__ __launch_bounds__(256) void conv_backward_kernel(const T* __restrict__ inputs, const T* __restrict__ out_grad,
                                                            const void* __restrict__ weight, const void* __restrict__ bias,
                                                            const T* __restrict__ initial, const T* __restrict__ final_grad,
                                                            const int32_t* __restrict__ lengths, T* __restrict__ inputs_grad,
                                                            T* __restrict__ initial_grad, float* __restrict__ weight_part,
                                                            float* __restrict__ bias_part, ConvBack g, unsigned flags) {
    constexpr int E = Elem<T>::E, H = W - 1, kTile = 64 * E;
    const int lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const int32_t row = wave / (uint32_t)g.segments, seg = wave - row * g.segments;
    if (row >= g.rows) return;
    const int32_t b = row / g.D, d = row - b * g.D;
    const int64_t len = row_length(lengths, b, g.L);
    const bool silu = flags & FMSELECTIVE_SILU;
    const T* x = inputs + b * g.batch_stride + d * g.channel_stride;
    const T* dy = out_grad + b * g.grad_batch_stride + d * g.grad_channel_stride;
    const T* state = initial ? initial + (int64_t)row * H : nullptr;
    const T* fg = final_grad ? final_grad + (int64_t)row * H : nullptr;
    T* dx_row = inputs_grad + (int64_t)row * g.L;
    float w[W], bv;
    conv_taps<T, W>(weight, bias, d, flags, w, bv);

    const int32_t lo = seg * g.seg_tiles;
    const int32_t hi = lo + g.seg_tiles < g.tiles ? lo + g.seg_tiles : g.tiles;
    float carry[H];  // dpre of the H positions behind the tile at work
    {
        const int64_t end = (int64_t)hi * kTile;
#pragma unroll
        for (int i = 0; i < H; ++i) {
            carry[i] = 0.0f;
            if (end + i < len) {  // the segment behind is another wave's: its first positions again
                float pre = bv;
#pragma unroll
                for (int j = 0; j < W; ++j) pre = __builtin_fmaf(w[j], Elem<T>::widen(x[end + i - H + j]), pre);
                const float g0 = Elem<T>::widen(dy[end + i]);
                carry[i] = silu ? g0 * silu_slope(pre, sigmoid(pre)) : g0;
            }
        }
    }
    float dw[W] = {}, db = 0.0f, dpre[E + H] = {};
    int32_t i = hi - 1;
    // FULL: the tiles lie wholly inside the row, and the final state's gradient does not reach them
    auto walk = [&](auto count_tag, auto full_tag) {
        constexpr int CH = decltype(count_tag)::value;
        constexpr bool FULL = decltype(full_tag)::value;
        u32x4 raw_x[CH], raw_dy[CH];
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            const int64_t t0 = (int64_t)(i - j) * kTile + lane * E;
            if (FULL || (int64_t)(i - j + 1) * kTile <= len) {
                raw_x[j] = fmscan::load16<T, false, false>(x + t0);
                raw_dy[j] = fmscan::load16<T, true, false>(dy + t0);
            } else {
                raw_x[j] = load_part<T>(x, t0, len);
                raw_dy[j] = load_part<T>(dy, t0, len);
            }
        }
        float first[H];  // lane 0's values before the lowest of these tiles
#pragma unroll
        for (int k = 0; k < H; ++k) first[k] = 0.0f;
        if (lane == 0) values_before<T, W>(x, (int64_t)(i - (CH - 1)) * kTile, len, state, first);
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            const int64_t end = (int64_t)(i - j + 1) * kTile, t0 = end - kTile + lane * E;
            const bool whole = FULL || end <= len;
            float f[E], gy[E], before[H], dx[E];
            Elem<T>::unpack(raw_x[j], f);
            Elem<T>::unpack(raw_dy[j], gy);
            float below[E] = {};
            if (j + 1 < CH) Elem<T>::unpack(raw_x[j + 1 < CH ? j + 1 : j], below);
#pragma unroll
            for (int k = 0; k < H; ++k)  // lane 0's come from lane 63 of the tile below, which is here but for the last
                before[k] = fmscan::dpp<fmscan::kWaveShr1>(j + 1 < CH ? fmscan::lane63(below[E - H + k]) : first[k], f[E - H + k]);
            conv_chunk_back<T, W>(f, gy, before, w, bv, silu, whole ? E : steps_before<E>(t0, len), whole, lane == 63, carry, dpre,
                                  dw, db, dx);
#pragma unroll
            for (int k = 0; k < H; ++k) carry[k] = fmscan::lane_value(dpre[k], 0);
            if (!FULL && fg && end + H > len) add_final_grad<T, H>(fg, t0, len, dx);
            if (FULL || end <= g.L) fmscan::store16<T, false>(dx_row + t0, Elem<T>::pack(dx));
            else store_values<T, E>(dx_row, t0, g.L, dx);
        }
        i -= CH;
    };
    while (i >= lo) {
        const bool full = (int64_t)(i + 1) * kTile + (fg ? H : 0) <= len;
        if (full && i - lo >= 3) walk(std::integral_constant<int, 4>{}, std::true_type{});
        else if (i - lo == 1 || (full && i > lo)) walk(std::integral_constant<int, 2>{}, std::false_type{});
        else walk(std::integral_constant<int, 1>{}, std::false_type{});
    }
    if (initial_grad && seg == 0 && lane == 0) put_initial_grad<T, W>(dpre, w, fg, len, initial_grad + (int64_t)row * H);
    const int64_t at = (int64_t)seg * g.rows + row;
#pragma unroll
    for (int j = 0; j < W; ++j) dw[j] = wave_sum_high(dw[j]);
    db = wave_sum_high(db);
    if (lane == 63) {
#pragma unroll
        for (int j = 0; j < W; ++j) weight_part[at * W + j] = dw[j];
        bias_part[at] = db;
    }
}

// 4 M consecutive values as M accesses at the alignment of an element, those from `count` on untouched
template <typename T, int M>
__device__ __forceinline__ void load_fours(const T* p, int count, T (&f)[4 * M]) {
    typedef T four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    if (count >= 4 * M) {
#pragma unroll
        for (int i = 0; i < M; ++i) {
            const four v = reinterpret_cast<const four*>(p)[i];
#pragma unroll
            for (int k = 0; k < 4; ++k) f[4 * i + k] = v[k];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4 * M; ++i) f[i] = i < count ? p[i] : (T)0.0f;
    }
}
template <typename T, int M>
__device__ __forceinline__ void store_fours(T* p, int count, const T (&f)[4 * M]) {
    typedef T four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    if (count >= 4 * M) {
#pragma unroll
        for (int i = 0; i < M; ++i) {
            four v;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = f[4 * i + k];
            reinterpret_cast<four*>(p)[i] = v;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4 * M; ++i)
            if (i < count) p[i] = f[i];
    }
}
template <typename T, int M>
__device__ __forceinline__ void load_param_fours(const void* p, int64_t at, bool narrow, int count, float (&f)[4 * M]) {
    if (narrow) {
        T v[4 * M];
        load_fours<T, M>(reinterpret_cast<const T*>(p) + at, count, v);
#pragma unroll
        for (int i = 0; i < 4 * M; ++i) f[i] = Elem<T>::widen(v[i]);
    } else {
        load_fours<float, M>(reinterpret_cast<const float*>(p) + at, count, f);
    }
}

// One token: four channels of a row a thread, whose states are 4 (W - 1) values in a row. The state moves by one place
// and takes the new input. 6.3 us at 256 rows of 4096 channels in f16 (9.4 with a channel a thread), 2.4 at one row of 2048:
// bound by the launch and the chain slot, state, store.
template <typename T, int W>
__global__ __launch_bounds__(256) void conv_step_kernel(const T* __restrict__ inputs, int64_t batch_stride, const T* state,
                                                        T* state_out, const void* __restrict__ weight,
                                                        const void* __restrict__ bias, const void* __restrict__ slots,
                                                        T* __restrict__ out, int32_t D, uint32_t tiles, int64_t S,
                                                        unsigned flags) {
    const uint32_t b = tiles == 1 ? blockIdx.x : blockIdx.x / tiles;
    const int32_t d = ((blockIdx.x - b * tiles) * blockDim.x + threadIdx.x) * 4;
    const int n = D - d;  // channels left, this thread's among them
    T x[4];
    float w[4 * W], v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (n > 0) {
        load_fours<T, 1>(inputs + b * batch_stride + d, n, x);
        load_param_fours<T, W>(weight, (int64_t)d * W, flags & FMSELECTIVE_NARROW_WEIGHT, n < 4 ? n * W : 4 * W, w);
        if (bias) load_param_fours<T, 1>(bias, d, flags & FMSELECTIVE_NARROW_BIAS, n, v);
    }
    const int64_t slot = slot_of_row(slots, flags & FMSELECTIVE_SLOTS_64, (int32_t)b, S);
    if (n <= 0) return;
    T y[4] = {(T)0.0f, (T)0.0f, (T)0.0f, (T)0.0f};
    if (slot >= 0) {
        const int64_t at = (slot * D + d) * (W - 1);
        const int held = n < 4 ? n * (W - 1) : 4 * (W - 1);
        T old[4 * (W - 1)], moved[4 * (W - 1)];
        load_fours<T, W - 1>(state + at, held, old);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const T value = j < W - 1 ? old[i * (W - 1) + (j < W - 1 ? j : 0)] : x[i];
                v[i] = __builtin_fmaf(w[i * W + j], Elem<T>::widen(value), v[i]);
                if (j) moved[i * (W - 1) + (j ? j - 1 : 0)] = value;
            }
            if (flags & FMSELECTIVE_SILU) v[i] *= sigmoid(v[i]);
            y[i] = (T)v[i];
        }
        store_fours<T, W - 1>(state_out + at, held, moved);
    }
    store_fours<T, 1>(out + (int64_t)b * D + d, n, y);
}

}  // namespace fmselective
