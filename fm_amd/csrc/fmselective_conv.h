// Kernels of the short depthwise convolution along time: forward, backward, one token.
//
// All three are bound by memory: a row is read once and written once, W <= 4 multiply-adds an element.
#pragma once

#include "fmselective_device.h"

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
// values before a chunk are a second, 8-byte load that the L1 answers.
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
// from the lane below, lane 0's from lane 63 of the chunks before, and from memory once a wave.
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
    int32_t rows, D;
    int32_t lanes_log2;   // lanes a row takes in a wave
    int32_t tiles;        // of 64 chunks, where lanes_log2 is 6; else 1
    int32_t segments, seg_tiles;
};

// d pre of one position: the gradient of the sum under the activation
__device__ __forceinline__ float conv_dpre(float pre, float dy, bool silu) {
    return silu ? dy * silu_slope(pre, sigmoid(pre)) : dy;
}

// A wave walks a row (or a segment of a long one) from its end to its start, one chunk a lane: the gradient of
// the sum before the activation is computed once an element, the W - 1 of them that a lane needs from beyond its
// chunk come from the next lane, and the last lane's from the tile before (lane 0's, kept). The gradients of
// weight and bias are summed over the whole walk in registers and across the lanes once. Rows of fewer than
// 64 chunks share a wave, 2^lanes_log2 lanes each.
// Tiles that lie wholly inside the row are loaded four at a time, by loads without a condition; the others come first
// in the walk.
template <typename T, int W>
__global__ __launch_bounds__(256) void conv_backward_kernel(const T* __restrict__ inputs, const T* __restrict__ out_grad,
                                                            const void* __restrict__ weight, const void* __restrict__ bias,
                                                            const T* __restrict__ initial, const T* __restrict__ final_grad,
                                                            const int32_t* __restrict__ lengths, T* __restrict__ inputs_grad,
                                                            T* __restrict__ initial_grad, float* __restrict__ weight_part,
                                                            float* __restrict__ bias_part, ConvBack g, unsigned flags) {
    constexpr int E = Elem<T>::E, H = W - 1;
    const int lane = threadIdx.x & 63;
    const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lanes = 1 << g.lanes_log2, c = lane & (lanes - 1);
    const int64_t slot = (wave << (6 - g.lanes_log2)) + (lane >> g.lanes_log2);  // row, or segment of a row
    const int64_t want_row = g.segments == 1 ? slot : slot / g.segments;
    const int32_t seg = g.segments == 1 ? 0 : (int32_t)(slot - want_row * g.segments);
    const bool live = want_row < g.rows;
    const int32_t row = live ? (int32_t)want_row : g.rows - 1;
    const int32_t b = row / g.D, d = row - b * g.D;
    const int64_t L = live ? g.L : 0;  // a lane without a row loads and stores nothing
    const int64_t len = live ? row_length(lengths, b, g.L) : 0;
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
    const int64_t tile = (int64_t)lanes * E;
    float carry[H];  // d pre of the H positions behind the tile at work
    {
        const int64_t end = hi * tile;
#pragma unroll
        for (int i = 0; i < H; ++i) {
            carry[i] = 0.0f;
            if (end + i < len) {  // the segment behind is another wave's: its first positions again
                float pre = bv;
#pragma unroll
                for (int j = 0; j < W; ++j) pre = __builtin_fmaf(w[j], Elem<T>::widen(x[end + i - H + j]), pre);
                carry[i] = conv_dpre(pre, Elem<T>::widen(dy[end + i]), silu);
            }
        }
    }
    float dw[W], db = 0.0f;
#pragma unroll
    for (int j = 0; j < W; ++j) dw[j] = 0.0f;
    float dpre[E + H];
#pragma unroll
    for (int k = 0; k < E + H; ++k) dpre[k] = 0.0f;

    // `first`: the values before the row's first lane's chunk, in that lane; FULL: every step of the tile counts and none
    // is in the final state's gradient
    auto work = [&](auto full_tag, int32_t i, const u32x4& raw_x, const u32x4& raw_dy, const float (&first)[H]) {
        constexpr bool FULL = decltype(full_tag)::value;
        const int64_t t0 = i * tile + (int64_t)c * E;
        float f[E], gy[E], before[H], dx[E];
        Elem<T>::unpack(raw_x, f);
        Elem<T>::unpack(raw_dy, gy);
#pragma unroll
        for (int k = 0; k < H; ++k) {
            const float below = fmscan::dpp<fmscan::kWaveShr1>(0.0f, f[E - H + k]);
            before[k] = c == 0 ? first[k] : below;
        }
        auto at = [&](int p) { return p < 0 ? before[p + H] : f[p]; };
        if (silu) {
            float pre[E];
#pragma unroll
            for (int k = 0; k < E; ++k) {
                pre[k] = bv;
#pragma unroll
                for (int j = 0; j < W; ++j) pre[k] = __builtin_fmaf(w[j], at(k - H + j), pre[k]);
            }
#pragma unroll
            for (int k = 0; k < E; ++k) dpre[k] = conv_dpre(pre[k], gy[k], true);
        } else {
#pragma unroll
            for (int k = 0; k < E; ++k) dpre[k] = gy[k];
        }
#pragma unroll
        for (int k = 0; k < E; ++k) {
            const bool in = FULL || t0 + k < len;
            if (!FULL) dpre[k] = in ? dpre[k] : 0.0f;
            // (a position that does not count adds nothing, whatever stands before it)
#pragma unroll
            for (int j = 0; j < W; ++j) dw[j] = __builtin_fmaf(dpre[k], in ? at(k - H + j) : 0.0f, dw[j]);
            db += dpre[k];
        }
#pragma unroll
        for (int k = 0; k < H; ++k) {
            const float next = fmscan::dpp<fmscan::kWaveShl1>(0.0f, dpre[k]);
            dpre[E + k] = c == lanes - 1 ? carry[k] : next;
            carry[k] = fmscan::lane_value(dpre[k], 0);  // read by rows that fill the wave alone
        }
#pragma unroll
        for (int k = 0; k < E; ++k) {
            float v = 0.0f;
#pragma unroll
            for (int j = 0; j < W; ++j) v = __builtin_fmaf(w[j], dpre[k + H - j], v);
            if (!FULL) {
                const int64_t p = t0 + k - (len - H);  // place in the final state
                if (fg && p >= 0 && p < H && t0 + k < len) v += Elem<T>::widen(fg[p]);
            }
            dx[k] = FULL || t0 + k < len ? v : 0.0f;
        }
        if constexpr (FULL) fmscan::store16<T, false>(dx_row + t0, Elem<T>::pack(dx));
        else store_values<T, E>(dx_row, t0, L, dx);
    };
    auto fetch_first = [&](int32_t i, float (&first)[H]) {
#pragma unroll
        for (int k = 0; k < H; ++k) first[k] = 0.0f;
        if (c == 0) values_before<T, W>(x, i * tile, len, state, first);
    };
    int32_t i = hi - 1;
    // the final state's gradient reaches H positions back, so a tile is full only with H more steps behind it;
    // rows that share a wave have one tile, of their own lengths
    for (; i >= lo && (g.lanes_log2 < 6 || (i + 1) * tile + (fg ? H : 0) > len); --i) {
        const int64_t t0 = i * tile + (int64_t)c * E;
        float first[H];
        fetch_first(i, first);
        work(std::false_type{}, i, fmscan::load_chunk<T, false, false>(x, t0, len, 0u),
             fmscan::load_chunk<T, false, false>(dy, t0, len, 0u), first);
    }
    auto walk = [&](auto count_tag) {
        constexpr int CH = decltype(count_tag)::value;
        u32x4 raw_x[CH], raw_dy[CH];
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            raw_x[j] = fmscan::load16<T, false, false>(x + (i - j) * tile + lane * E);
            raw_dy[j] = fmscan::load16<T, true, false>(dy + (i - j) * tile + lane * E);
        }
        float first[H];
        fetch_first(i - (CH - 1), first);
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            float before[H];
            if (j + 1 < CH) {  // lane 63 of the tile before, which is here
                float f[E];
                Elem<T>::unpack(raw_x[j + 1 < CH ? j + 1 : j], f);
#pragma unroll
                for (int k = 0; k < H; ++k) before[k] = fmscan::lane63(f[E - H + k]);
            } else {
#pragma unroll
                for (int k = 0; k < H; ++k) before[k] = first[k];
            }
            work(std::true_type{}, i - j, raw_x[j], raw_dy[j], before);
        }
        i -= CH;
    };
    while (i - lo >= 3) walk(std::integral_constant<int, 4>{});
    while (i >= lo) walk(std::integral_constant<int, 1>{});
    if (initial_grad && live && seg == 0 && c == 0) {
#pragma unroll
        for (int i = 0; i < H; ++i) {
            float v = 0.0f;
            if (len > 0) {
#pragma unroll
                for (int j = 0; j <= i; ++j) v = __builtin_fmaf(w[j], dpre[i - j], v);
            }
            if (fg && i >= len) v += Elem<T>::widen(fg[i - len]);
            initial_grad[(int64_t)row * H + i] = (T)v;
        }
    }
    const int64_t at = (int64_t)seg * g.rows + row;
    if (lanes == 64) {  // (live: a wave without a row has none to write)
#pragma unroll
        for (int j = 0; j < W; ++j) dw[j] = wave_sum_high(dw[j]);
        db = wave_sum_high(db);
        if (live && lane == 63) {
#pragma unroll
            for (int j = 0; j < W; ++j) weight_part[at * W + j] = dw[j];
            bias_part[at] = db;
        }
        return;
    }
    auto over_lanes = [&](float v) {
        for (int s = lanes >> 1; s > 0; s >>= 1) v += __shfl_xor(v, s);
        return v;
    };
#pragma unroll
    for (int j = 0; j < W; ++j) {
        const float v = over_lanes(dw[j]);
        if (live && c == 0) weight_part[at * W + j] = v;
    }
    db = over_lanes(db);
    if (live && c == 0) bias_part[at] = db;
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
// and takes the new input.
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
