// Kernels of the selective scan: forward, backward, one token.
//
//   dt = softplus(delta + delta_bias),  h[n] <- exp(dt A[n]) h[n] + dt u write[n],  y = sum_n read[n] h[n] + skip u
//
// The decay differs for every channel, state and step, so there is no matrix product in it: per (b, d, n, t) one
// exponential and four multiply-adds forward, about twenty operations backward, against at most 14 bytes per
// (b, d, t). With 16 states the kernels are bound by vector float32 arithmetic, not by memory.
//
// Layout. Time runs along the lanes: a lane holds 8 consecutive steps of a channel, 16 lanes (one DPP row) a tile
// of 128 steps, so a wave works on 4 channels at a time and every tensor moves as 16-byte accesses along time.
// For one state of a channel a lane composes its 8 steps (its total decay is one exponential of the steps' sum),
// the row scans the pairs (decay, value) by DPP, and a second walk over the 8 steps with the true entering state
// gives the states. A block's waves share the tile of write and read, kept in LDS as float32 and fetched one
// tile ahead; the state that leaves a tile waits in LDS for the next one.
#pragma once

#include "fmselective_device.h"

namespace fmselective {

constexpr int kSteps = 8;         // consecutive steps a lane holds
constexpr int kMark = 128;        // steps between the states that forward saves for backward
constexpr int kScanWaves = 4;

// log(1 + e^x) to float32 accuracy also where e^x is small: with w = 1 + e rounded, log(w) e / (w - 1)
// (the rounding of w cancels in the quotient; a classical device, due to Kahan)
__device__ __forceinline__ float softplus(float x) {
    const float e = exp2_fast(-kLog2E * __builtin_fabsf(x));
    const float w = 1.0f + e, d = w - 1.0f;
    const float l = d == 0.0f ? e : kLn2 * __builtin_amdgcn_logf(w) * (e * __builtin_amdgcn_rcpf(d));
    return fmaxf(x, 0.0f) + l;
}

// What the kernels need of include/fmselective.h's fmselective_scan
struct Scan {
    const void *tokens, *delta, *gate, *write, *read, *skip, *delta_bias;
    const float *A, *initial;
    const int32_t* lengths;
    int64_t tokens_b, tokens_d, delta_b, delta_d, gate_b, gate_d, write_b, write_g, write_n, read_b, read_g, read_n;
    int64_t L;
    int32_t D, N, G, per_group, blocks_per_group, marks;  // marks: ceil(L / kMark)
    uint32_t flags;
};

// Two rows' worth of (decay, value) pairs, composed over the lanes of a row of 16 (and, with LPC = 64, over the
// rows): on exit a lane holds the composition of its own and all earlier lanes' pairs. Two pairs at a time: the
// instructions of one fill the two wait states that the other needs between a write and a DPP read.
#define FMSELECTIVE_LEVEL(CTRL)                                          \
    "v_fmac_f32_dpp %1, %1, %0 " CTRL "\n\t"                             \
    "v_fmac_f32_dpp %3, %3, %2 " CTRL "\n\t"                             \
    "v_mul_f32_dpp %0, %0, %0 " CTRL "\n\t"                              \
    "v_mul_f32_dpp %2, %2, %2 " CTRL "\n\t"
template <int LPC>
__device__ __forceinline__ void scan_up(float& a0, float& b0, float& a1, float& b1) {
    if constexpr (LPC == 16)
        asm("s_nop 1\n\t"
            FMSELECTIVE_LEVEL("row_shr:1 row_mask:0xf bank_mask:0xf")
            FMSELECTIVE_LEVEL("row_shr:2 row_mask:0xf bank_mask:0xf")
            FMSELECTIVE_LEVEL("row_shr:4 row_mask:0xf bank_mask:0xf")
            FMSELECTIVE_LEVEL("row_shr:8 row_mask:0xf bank_mask:0xf")
            "s_nop 1"
            : "+v"(a0), "+v"(b0), "+v"(a1), "+v"(b1));
    else
        asm("s_nop 1\n\t"
            FMSELECTIVE_LEVEL("row_shr:1 row_mask:0xf bank_mask:0xf")
            FMSELECTIVE_LEVEL("row_shr:2 row_mask:0xf bank_mask:0xf")
            FMSELECTIVE_LEVEL("row_shr:4 row_mask:0xf bank_mask:0xf")
            FMSELECTIVE_LEVEL("row_shr:8 row_mask:0xf bank_mask:0xf")
            FMSELECTIVE_LEVEL("row_bcast:15 row_mask:0xa bank_mask:0xf")
            FMSELECTIVE_LEVEL("row_bcast:31 row_mask:0xc bank_mask:0xf")
            "s_nop 1"
            : "+v"(a0), "+v"(b0), "+v"(a1), "+v"(b1));
}
// The same towards lower lanes, inside rows of 16
__device__ __forceinline__ void scan_down(float& a0, float& b0, float& a1, float& b1) {
    asm("s_nop 1\n\t"
        FMSELECTIVE_LEVEL("row_shl:1 row_mask:0xf bank_mask:0xf")
        FMSELECTIVE_LEVEL("row_shl:2 row_mask:0xf bank_mask:0xf")
        FMSELECTIVE_LEVEL("row_shl:4 row_mask:0xf bank_mask:0xf")
        FMSELECTIVE_LEVEL("row_shl:8 row_mask:0xf bank_mask:0xf")
        "s_nop 1"
        : "+v"(a0), "+v"(b0), "+v"(a1), "+v"(b1));
}
#undef FMSELECTIVE_LEVEL

constexpr int kRowShr1 = 0x111;  // lane i <- lane i-1 inside its row of 16

template <int CTRL>
__device__ __forceinline__ float dpp_or_zero(float v) {
    return u2f((uint32_t)__builtin_amdgcn_update_dpp(0, (int)f2u(v), CTRL, 0xf, 0xf, true));
}
// Lane 15 of each row of 16: the sum over the row
__device__ __forceinline__ float row_sum(float v) {
    v += dpp_or_zero<0x111>(v);
    v += dpp_or_zero<0x112>(v);
    v += dpp_or_zero<0x114>(v);
    v += dpp_or_zero<0x118>(v);
    return v;
}

// 8 steps of a row as they lie in memory
template <typename T>
struct Raw {
    u32x4 v[kSteps / Elem<T>::E];
};
template <typename T>
__device__ __forceinline__ Raw<T> load_raw(const T* __restrict__ row, int64_t t0, int64_t len) {
    Raw<T> r;
#pragma unroll
    for (int i = 0; i < kSteps / Elem<T>::E; ++i)
        r.v[i] = fmscan::load_chunk<T, false, false>(row, t0 + i * Elem<T>::E, len, 0u);
    return r;
}
template <typename T>
__device__ __forceinline__ void widen_raw(const Raw<T>& r, float (&f)[kSteps]) {
    constexpr int E = Elem<T>::E;
#pragma unroll
    for (int i = 0; i < kSteps / E; ++i) {
        float part[E];
        Elem<T>::unpack(r.v[i], part);
#pragma unroll
        for (int k = 0; k < E; ++k) f[i * E + k] = part[k];
    }
}

// The shared tile of write and read: for each of NC states, LPC chunks of 8 steps, the chunks' first and second
// halves in planes of their own so that the lanes of a row read whole lines of banks.
template <int LPC, int WAVES>
struct SharedTile {
    static constexpr int kStates = 64 * WAVES / LPC;  // states in LDS at a time: one chunk of each operand a thread
    float v[2][kStates][2][LPC][4];                   // write / read, state, half, chunk, step
    __device__ __forceinline__ void put(int which, const float (&f)[kSteps]) {
        const int n = threadIdx.x / LPC, c = threadIdx.x % LPC;
        *reinterpret_cast<float4*>(v[which][n][0][c]) = make_float4(f[0], f[1], f[2], f[3]);
        *reinterpret_cast<float4*>(v[which][n][1][c]) = make_float4(f[4], f[5], f[6], f[7]);
    }
    __device__ __forceinline__ void get(int which, int n, int c, float (&f)[kSteps]) const {
        const float4 a = *reinterpret_cast<const float4*>(v[which][n][0][c]);
        const float4 b = *reinterpret_cast<const float4*>(v[which][n][1][c]);
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
        f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    }
};

// states of a channel in LDS: an even number, the one beyond N with no decay and no value
__host__ __device__ __forceinline__ int padded_states(int N) { return (N + 1) & ~1; }
// and the stride between channels, in entries: odd, so that channels do not share banks
__host__ __device__ __forceinline__ int state_stride(int N) { return padded_states(N) | 1; }

template <int LPC, int WAVES>
constexpr size_t scan_tiles_bytes() { return 2 * sizeof(SharedTile<LPC, WAVES>); }
template <int LPC, int WAVES>
size_t scan_forward_lds(int N) { return scan_tiles_bytes<LPC, WAVES>() + (size_t)WAVES * (64 / LPC) * state_stride(N) * sizeof(float2); }

template <typename T, int LPC, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void selective_forward_kernel(Scan p, T* __restrict__ out, float* __restrict__ final_state,
                                                                       float* __restrict__ marks) {
    using Tile = SharedTile<LPC, WAVES>;
    constexpr int NC = Tile::kStates, kTile = LPC * kSteps, CW = 64 / LPC;
    extern __shared__ char lds[];
    Tile* tiles = reinterpret_cast<Tile*>(lds);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & (LPC - 1), ch = lane / LPC;
    const int stride = state_stride(p.N);
    float2* held = reinterpret_cast<float2*>(lds + scan_tiles_bytes<LPC, WAVES>()) + wave * CW * stride;  // (A log2 e, state)

    const uint32_t bg = blockIdx.x / (uint32_t)p.blocks_per_group, block = blockIdx.x - bg * p.blocks_per_group;
    const uint32_t b = bg / (uint32_t)p.G, g = bg - b * p.G;
    const int32_t first = (int32_t)(block * WAVES + wave) * CW;  // the wave's first channel in the group
    const int32_t local = first + ch;
    const bool valid = local < p.per_group;
    const int32_t d = (int32_t)g * p.per_group + (valid ? local : p.per_group - 1);
    const int64_t row = (int64_t)b * p.D + d;
    const int64_t len = row_length(p.lengths, b, p.L), mine = valid ? len : 0;  // (no steps for a channel beyond the group)
    const T* u_row = (const T*)p.tokens + b * p.tokens_b + d * p.tokens_d;
    const T* delta_row = (const T*)p.delta + b * p.delta_b + d * p.delta_d;
    const T* gate_row = p.gate ? (const T*)p.gate + b * p.gate_b + d * p.gate_d : nullptr;
    const T* write_rows = (const T*)p.write + b * p.write_b + g * p.write_g;
    const T* read_rows = (const T*)p.read + b * p.read_b + g * p.read_g;
    const float skip = p.skip ? param<T>(p.skip, d, p.flags & FMSELECTIVE_NARROW_SKIP) : 0.0f;
    const float bias = p.delta_bias ? param<T>(p.delta_bias, d, p.flags & FMSELECTIVE_NARROW_BIAS) : 0.0f;

    // decay rates and entering states of the wave's channels
    const int padded = padded_states(p.N);
    auto each_state = [&](auto&& f) {  // f(entry in `held`, its channel's row or -1, n) over the wave's lanes
        for (int i = lane; i < CW * padded; i += 64) {
            const int k = i / padded, n = i - k * padded;
            const bool real = n < p.N && first + k < p.per_group;
            f(held[k * stride + n], real ? (int64_t)b * p.D + (int64_t)g * p.per_group + first + k : (int64_t)-1, n);
        }
    };
    each_state([&](float2& e, int64_t r, int n) {
        e.x = r < 0 ? 0.0f : p.A[(r - (int64_t)b * p.D) * p.N + n] * kLog2E;
        e.y = r < 0 || !p.initial ? 0.0f : p.initial[r * p.N + n];
    });

    const int chunks = (p.N + NC - 1) / NC;
    const int32_t n_tiles = (int32_t)((len + kTile - 1) / kTile);
    const int32_t total = n_tiles * chunks;
    Raw<T> next_w, next_r, next_u, next_delta, next_gate = {};
    auto fetch_shared = [&](int32_t it) {
        const int32_t tile = it / chunks;
        const int n = (it - tile * chunks) * NC + threadIdx.x / LPC;
        const int64_t t0 = (int64_t)tile * kTile + (threadIdx.x % LPC) * kSteps, end = n < p.N ? len : 0;
        next_w = load_raw<T>(write_rows + n * p.write_n, t0, end);
        next_r = load_raw<T>(read_rows + n * p.read_n, t0, end);
    };
    auto fetch_rows = [&](int32_t tile) {
        const int64_t t0 = (int64_t)tile * kTile + c * kSteps;
        next_u = load_raw<T>(u_row, t0, mine);
        next_delta = load_raw<T>(delta_row, t0, mine);
        if (gate_row) next_gate = load_raw<T>(gate_row, t0, mine);
    };
    auto put_shared = [&](Tile& t) {
        float f[kSteps];
        widen_raw(next_w, f);
        t.put(0, f);
        widen_raw(next_r, f);
        t.put(1, f);
    };
    if (total) {
        fetch_shared(0);
        fetch_rows(0);
        put_shared(tiles[0]);
    }
    __syncthreads();

    float dt[kSteps], dtu[kSteps], y[kSteps], total_dt = 0.0f;
    Raw<T> gate_now = {};
    int32_t it = 0;
    for (int32_t tile = 0; tile < n_tiles; ++tile) {
        const int64_t t0 = (int64_t)tile * kTile + c * kSteps;
        {
            float u[kSteps];
            widen_raw(next_u, u);
            widen_raw(next_delta, dt);
            gate_now = next_gate;
            total_dt = 0.0f;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                float v = dt[k] + bias;
                if (p.flags & FMSELECTIVE_SOFTPLUS) v = softplus(v);
                dt[k] = t0 + k < mine ? v : 0.0f;  // a step of length zero leaves the state as it is
                dtu[k] = dt[k] * u[k];
                y[k] = skip * u[k];
                total_dt += dt[k];
            }
            if (tile + 1 < n_tiles) fetch_rows(tile + 1);
        }
        for (int chunk = 0; chunk < chunks; ++chunk, ++it) {
            if (it + 1 < total) fetch_shared(it + 1);
            const Tile& now = tiles[it & 1];
            const int n0 = chunk * NC, n_end = padded - n0 < NC ? padded - n0 : NC;
            for (int nl = 0; nl < n_end; nl += 2) {
                float a[2][kSteps], v[2][kSteps], P[2], S[2], enter[2];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const float2 e = held[ch * stride + n0 + nl + q];
                    enter[q] = e.y;
                    now.get(0, nl + q, c, v[q]);
#pragma unroll
                    for (int k = 0; k < kSteps; ++k) {
                        a[q][k] = exp2_fast(dt[k] * e.x);
                        v[q][k] *= dtu[k];
                    }
                    S[q] = v[q][0];
#pragma unroll
                    for (int k = 1; k < kSteps; ++k) S[q] = __builtin_fmaf(a[q][k], S[q], v[q][k]);
                    P[q] = exp2_fast(total_dt * e.x);
                }
                scan_up<LPC>(P[0], S[0], P[1], S[1]);
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    constexpr int kShift = LPC == 16 ? kRowShr1 : fmscan::kWaveShr1;
                    float h = __builtin_fmaf(fmscan::dpp<kShift>(1.0f, P[q]), enter[q], fmscan::dpp<kShift>(0.0f, S[q]));
                    const int n = n0 + nl + q;
                    if (c == LPC - 1) held[ch * stride + n].y = __builtin_fmaf(P[q], enter[q], S[q]);
                    if (marks && (c & 15) == 0) {
                        const int32_t mark = tile * (LPC / 16) + c / 16;
                        if (valid && n < p.N && mark < p.marks) marks[(row * p.marks + mark) * p.N + n] = h;
                    }
                    float r[kSteps];
                    now.get(1, nl + q, c, r);
#pragma unroll
                    for (int k = 0; k < kSteps; ++k) {
                        h = __builtin_fmaf(a[q][k], h, v[q][k]);
                        y[k] = __builtin_fmaf(r[k], h, y[k]);
                    }
                }
            }
            if (it + 1 < total) put_shared(tiles[(it + 1) & 1]);
            __syncthreads();
        }
        if (gate_row) {
            float z[kSteps];
            widen_raw(gate_now, z);
#pragma unroll
            for (int k = 0; k < kSteps; ++k) y[k] *= z[k] * sigmoid(z[k]);
        }
#pragma unroll
        for (int k = 0; k < kSteps; ++k) y[k] = t0 + k < mine ? y[k] : 0.0f;
        if (valid) store_values<T, kSteps>(out + row * p.L, t0, p.L, y);
    }
#pragma unroll
    for (int k = 0; k < kSteps; ++k) y[k] = 0.0f;
    if (valid)
        for (int64_t t0 = (int64_t)n_tiles * kTile + c * kSteps; t0 < p.L; t0 += kTile) store_values<T, kSteps>(out + row * p.L, t0, p.L, y);
    if (final_state)
        each_state([&](float2& e, int64_t r, int n) {
            if (r >= 0) final_state[r * p.N + n] = e.y;
        });
}

// Adds the values of the four rows of a wave and deals the sums out: of v[0..7] and v[8..15], row 0 gets the sums
// of v[0..3], row 1 v[4..7], row 2 v[8..11], row 3 v[12..15]. Each swap exchanges halves of two registers, so one
// addition settles both: 24 instructions for 16 sums.
__device__ __forceinline__ float4 sum_rows(const float (&v)[16]) {
    float w[8], x[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const auto s = __builtin_amdgcn_permlane32_swap(f2u(v[i]), f2u(v[i + 8]), false, false);
        w[i] = u2f(s[0]) + u2f(s[1]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const auto s = __builtin_amdgcn_permlane16_swap(f2u(w[i]), f2u(w[i + 4]), false, false);
        x[i] = u2f(s[0]) + u2f(s[1]);
    }
    return make_float4(x[0], x[1], x[2], x[3]);
}

struct ScanGrads {
    const void *out_grad;
    int64_t out_b, out_d;
    const float *final_grad, *marks;
    void *tokens, *delta, *gate;         // (B, D, L) dense
    float *initial;                      // (B, D, N)
    float *A_part, *skip_part, *bias_part;  // (B, D, N), (B, D), (B, D)
    float *shared_part;                  // [block][n][mark][256]: sums of write's and read's gradients over the block's channels
};

template <int WAVES>
size_t scan_backward_lds(int N) {
    return scan_tiles_bytes<16, WAVES>() + sizeof(float4) * 2 * WAVES * 2 * 64 + (size_t)WAVES * 4 * state_stride(N) * sizeof(float4);
}

// Backward. The tiles are walked from the last to the first. In a tile the states are made again from the state that
// forward saved before it, the gradient of the state runs against time through the same decays, and
//   dh[t] = g[t] read[t] + a[t+1] dh[t+1]     g = out_grad * silu(gate)
//   dtokens = dt sum_n dh write + skip g      dA = sum_t dt p      p = dh a h[t-1]
//   ddt = u sum_n dh write + sum_n A p        dwrite = sum_d dh dt u      dread = sum_d g h
// The sums over n stay in registers, those over time are added up in LDS, one float a state and channel. The sums
// over the channels are made in the wave (its 4 channels, sum_rows), over the block's waves in LDS and over
// the blocks by a second kernel, always in the same order.
template <typename T, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void selective_backward_kernel(Scan p, ScanGrads o) {
    constexpr int LPC = 16, kTile = LPC * kSteps, CW = 4;
    using Tile = SharedTile<LPC, WAVES>;
    constexpr int NC = Tile::kStates;
    extern __shared__ char lds[];
    Tile* tiles = reinterpret_cast<Tile*>(lds);
    float4* sums = reinterpret_cast<float4*>(lds + scan_tiles_bytes<LPC, WAVES>());  // [parity][wave][state of the pair][lane]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, ch = lane >> 4;
    const int stride = state_stride(p.N);
    // per channel and state: A log2 e, the gradient that arrives from later steps, the sum for dA, the state before the tile
    float4* held = sums + 2 * WAVES * 2 * 64 + wave * CW * stride;

    const uint32_t bg = blockIdx.x / (uint32_t)p.blocks_per_group, block = blockIdx.x - bg * p.blocks_per_group;
    const uint32_t b = bg / (uint32_t)p.G, g = bg - b * p.G;
    const int32_t first = (int32_t)(block * WAVES + wave) * CW, local = first + ch;
    const bool valid = local < p.per_group;
    const int32_t d = (int32_t)g * p.per_group + (valid ? local : p.per_group - 1);
    const int64_t row = (int64_t)b * p.D + d;
    const int64_t len = row_length(p.lengths, b, p.L), mine = valid ? len : 0;
    const T* u_row = (const T*)p.tokens + b * p.tokens_b + d * p.tokens_d;
    const T* delta_row = (const T*)p.delta + b * p.delta_b + d * p.delta_d;
    const T* gate_row = p.gate ? (const T*)p.gate + b * p.gate_b + d * p.gate_d : nullptr;
    const T* dy_row = (const T*)o.out_grad + b * o.out_b + d * o.out_d;
    const T* write_rows = (const T*)p.write + b * p.write_b + g * p.write_g;
    const T* read_rows = (const T*)p.read + b * p.read_b + g * p.read_g;
    const float skip = p.skip ? param<T>(p.skip, d, p.flags & FMSELECTIVE_NARROW_SKIP) : 0.0f;
    const float bias = p.delta_bias ? param<T>(p.delta_bias, d, p.flags & FMSELECTIVE_NARROW_BIAS) : 0.0f;

    const int padded = padded_states(p.N);
    auto each_state = [&](auto&& f) {
        for (int i = lane; i < CW * padded; i += 64) {
            const int k = i / padded, n = i - k * padded;
            const bool real = n < p.N && first + k < p.per_group;
            f(held[k * stride + n], real ? (int64_t)b * p.D + (int64_t)g * p.per_group + first + k : (int64_t)-1, n);
        }
    };
    each_state([&](float4& e, int64_t r, int n) {
        e.x = r < 0 ? 0.0f : p.A[(r - (int64_t)b * p.D) * p.N + n] * kLog2E;
        e.y = r < 0 || !o.final_grad ? 0.0f : o.final_grad[r * p.N + n];
        e.z = 0.0f;
        e.w = 0.0f;
    });

    const int chunks = (p.N + NC - 1) / NC;
    const int32_t n_tiles = (int32_t)((len + kTile - 1) / kTile);
    const int32_t total = n_tiles * chunks;
    Raw<T> next_w, next_r;
    auto fetch_shared = [&](int32_t it) {
        const int32_t back = it / chunks;
        const int n = (it - back * chunks) * NC + threadIdx.x / LPC;
        const int64_t t0 = (int64_t)(n_tiles - 1 - back) * kTile + (threadIdx.x % LPC) * kSteps, end = n < p.N ? len : 0;
        next_w = load_raw<T>(write_rows + n * p.write_n, t0, end);
        next_r = load_raw<T>(read_rows + n * p.read_n, t0, end);
    };
    auto put_shared = [&](Tile& t) {
        float f[kSteps];
        widen_raw(next_w, f);
        t.put(0, f);
        widen_raw(next_r, f);
        t.put(1, f);
    };
    if (total) {
        fetch_shared(0);
        put_shared(tiles[0]);
    }
    __syncthreads();

    float skip_sum = 0.0f, bias_sum = 0.0f;
    int32_t it = 0, pairs = 0;
    float* part = o.shared_part + (int64_t)blockIdx.x * p.N * p.marks * 256;
    for (int32_t tile = n_tiles - 1; tile >= 0; --tile) {
        const int64_t t0 = (int64_t)tile * kTile + c * kSteps;
        float dt[kSteps], dtu[kSteps], gy[kSteps], sum_w[kSteps], sum_a[kSteps], y[kSteps], total_dt = 0.0f;
        {
            float u[kSteps], z[kSteps];
            load_values<T, kSteps>(u_row, t0, mine, u);
            load_values<T, kSteps>(delta_row, t0, mine, dt);
            load_values<T, kSteps>(dy_row, t0, mine, gy);
            if (gate_row) load_values<T, kSteps>(gate_row, t0, mine, z);
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                float v = dt[k] + bias;
                if (p.flags & FMSELECTIVE_SOFTPLUS) v = softplus(v);
                dt[k] = t0 + k < mine ? v : 0.0f;
                dtu[k] = dt[k] * u[k];
                total_dt += dt[k];
                if (gate_row) gy[k] *= z[k] * sigmoid(z[k]);
                sum_w[k] = sum_a[k] = y[k] = 0.0f;
            }
        }
        each_state([&](float4& e, int64_t r, int n) { e.w = r < 0 ? 0.0f : o.marks[(r * p.marks + tile) * p.N + n]; });
        __builtin_amdgcn_wave_barrier();  // what the wave's lanes have written its lanes read: LDS answers in order
        for (int chunk = 0; chunk < chunks; ++chunk, ++it) {
            if (it + 1 < total) fetch_shared(it + 1);
            const Tile& now = tiles[it & 1];
            const int n0 = chunk * NC, n_end = padded - n0 < NC ? padded - n0 : NC;
            for (int nl = 0; nl < n_end; nl += 2, ++pairs) {
                float a[2][kSteps], h[2][kSteps], m[2][kSteps], dh[2][kSteps], P[2], S[2], Q[2], R[2];
                float4 e[2];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    e[q] = held[ch * stride + n0 + nl + q];
                    now.get(0, nl + q, c, h[q]);
#pragma unroll
                    for (int k = 0; k < kSteps; ++k) {
                        a[q][k] = exp2_fast(dt[k] * e[q].x);
                        h[q][k] *= dtu[k];
                    }
                    S[q] = h[q][0];
#pragma unroll
                    for (int k = 1; k < kSteps; ++k) S[q] = __builtin_fmaf(a[q][k], S[q], h[q][k]);
                    P[q] = exp2_fast(total_dt * e[q].x);
                    Q[q] = P[q];
                    now.get(1, nl + q, c, dh[q]);
#pragma unroll
                    for (int k = 0; k < kSteps; ++k) dh[q][k] *= gy[k];
                    R[q] = dh[q][kSteps - 1];
#pragma unroll
                    for (int k = kSteps - 2; k >= 0; --k) R[q] = __builtin_fmaf(a[q][k + 1], R[q], dh[q][k]);
                    R[q] *= a[q][0];
                }
                scan_up<16>(P[0], S[0], P[1], S[1]);
                scan_down(Q[0], R[0], Q[1], R[1]);
                float4 rows[2];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    float s = __builtin_fmaf(fmscan::dpp<kRowShr1>(1.0f, P[q]), e[q].w, fmscan::dpp<kRowShr1>(0.0f, S[q]));
#pragma unroll
                    for (int k = 0; k < kSteps; ++k) {
                        m[q][k] = a[q][k] * s;
                        s = h[q][k] = m[q][k] + h[q][k];
                    }
                    if (gate_row) {
                        float r[kSteps];
                        now.get(1, nl + q, c, r);
#pragma unroll
                        for (int k = 0; k < kSteps; ++k) y[k] = __builtin_fmaf(r[k], h[q][k], y[k]);
                    }
                    float t = __builtin_fmaf(fmscan::dpp<fmscan::kRowShl1>(1.0f, Q[q]), e[q].y,
                                             fmscan::dpp<fmscan::kRowShl1>(0.0f, R[q]));
                    float& arriving = held[ch * stride + n0 + nl + q].y;
                    if (c == 0) arriving = __builtin_fmaf(Q[q], e[q].y, R[q]);
#pragma unroll
                    for (int k = kSteps - 1; k >= 0; --k) {
                        dh[q][k] += t;
                        t = a[q][k] * dh[q][k];
                    }
                    float w[kSteps], v[16], in_time = 0.0f;
                    now.get(0, nl + q, c, w);
#pragma unroll
                    for (int k = 0; k < kSteps; ++k) {
                        sum_w[k] = __builtin_fmaf(dh[q][k], w[k], sum_w[k]);
                        v[k] = dh[q][k] * dtu[k];
                        v[8 + k] = gy[k] * h[q][k];
                        const float pk = dh[q][k] * m[q][k];
                        sum_a[k] = __builtin_fmaf(e[q].x, pk, sum_a[k]);
                        in_time = __builtin_fmaf(dt[k], pk, in_time);
                    }
                    in_time = row_sum(in_time);
                    if (c == 15) held[ch * stride + n0 + nl + q].z = e[q].z + in_time;
                    rows[q] = sum_rows(v);
                }
                float4* mine_sums = sums + (pairs & 1) * WAVES * 2 * 64;
                mine_sums[(wave * 2 + 0) * 64 + lane] = rows[0];
                mine_sums[(wave * 2 + 1) * 64 + lane] = rows[1];
                __syncthreads();
                // two states' 64 float4 each, over the waves: the first two waves of the block add one each
                if (wave < 2) {
                    const int n = n0 + nl + wave;
                    float4 s = mine_sums[wave * 64 + lane];
#pragma unroll
                    for (int w = 1; w < WAVES; ++w) {
                        const float4 v = mine_sums[(w * 2 + wave) * 64 + lane];
                        s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
                    }
                    if (n < p.N) reinterpret_cast<float4*>(part + ((int64_t)n * p.marks + tile) * 256)[lane] = s;
                }
            }
            if (it + 1 < total) put_shared(tiles[(it + 1) & 1]);
            __syncthreads();
        }
        {
            float u[kSteps], dd[kSteps], x[kSteps], z[kSteps];
            load_values<T, kSteps>(u_row, t0, mine, u);
            load_values<T, kSteps>(delta_row, t0, mine, x);
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                float v = __builtin_fmaf(u[k], sum_w[k], kLn2 * sum_a[k]);
                if (p.flags & FMSELECTIVE_SOFTPLUS) v *= sigmoid(x[k] + bias);
                const bool in = t0 + k < mine;
                dd[k] = in ? v : 0.0f;
                bias_sum += dd[k];
                skip_sum = __builtin_fmaf(gy[k], u[k], skip_sum);
                x[k] = in ? __builtin_fmaf(dt[k], sum_w[k], skip * gy[k]) : 0.0f;
                y[k] = __builtin_fmaf(skip, u[k], y[k]);
            }
            if (valid) {
                store_values<T, kSteps>((T*)o.tokens + row * p.L, t0, p.L, x);
                store_values<T, kSteps>((T*)o.delta + row * p.L, t0, p.L, dd);
            }
            if (gate_row) {
                load_values<T, kSteps>(dy_row, t0, mine, dd);
                load_values<T, kSteps>(gate_row, t0, mine, z);
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    const float v = dd[k] * y[k] * silu_slope(z[k], sigmoid(z[k]));
                    dd[k] = t0 + k < mine ? v : 0.0f;
                }
                if (valid) store_values<T, kSteps>((T*)o.gate + row * p.L, t0, p.L, dd);
            }
        }
    }
    float zero[kSteps];
#pragma unroll
    for (int k = 0; k < kSteps; ++k) zero[k] = 0.0f;
    if (valid)
        for (int64_t t0 = (int64_t)n_tiles * kTile + c * kSteps; t0 < p.L; t0 += kTile) {
            store_values<T, kSteps>((T*)o.tokens + row * p.L, t0, p.L, zero);
            store_values<T, kSteps>((T*)o.delta + row * p.L, t0, p.L, zero);
            if (gate_row) store_values<T, kSteps>((T*)o.gate + row * p.L, t0, p.L, zero);
        }
    skip_sum = row_sum(skip_sum);
    bias_sum = row_sum(bias_sum);
    if (valid && c == 15) {
        if (o.skip_part) o.skip_part[row] = skip_sum;
        if (o.bias_part) o.bias_part[row] = bias_sum;
    }
    each_state([&](float4& e, int64_t r, int n) {
        if (r < 0) return;
        o.A_part[r * p.N + n] = e.z;
        if (o.initial) o.initial[r * p.N + n] = e.y;
    });
}

// The gradients of write and read: the blocks' sums added up in their order and rounded once. A wave a
// (b, g, n, mark), a float4 a lane, in the order that sum_rows left them.
template <typename T>
__global__ __launch_bounds__(256) void selective_shared_grads_kernel(const float* __restrict__ part, T* __restrict__ write_grad,
                                                                     T* __restrict__ read_grad, const int32_t* __restrict__ lengths,
                                                                     int64_t L, int64_t waves, int32_t N, int32_t G,
                                                                     int32_t marks, int32_t blocks) {
    const int lane = threadIdx.x & 63, part_of = lane >> 4, c = lane & 15;
    const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (wave >= waves) return;
    const int64_t line = wave / marks;  // (b, g, n)
    const int32_t mark = (int32_t)(wave - line * marks);
    const int64_t bg = line / N;
    const int32_t n = (int32_t)(line - bg * N);
    const int64_t len = row_length(lengths, bg / G, L);
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if ((int64_t)mark * kMark < len) {
        const float4* at = reinterpret_cast<const float4*>(part) + (((bg * blocks) * N + n) * marks + mark) * 64 + lane;
        const int64_t step = (int64_t)N * marks * 64;
#pragma unroll 4
        for (int32_t i = 0; i < blocks; ++i) {
            const float4 v = at[i * step];
            s[0] += v.x; s[1] += v.y; s[2] += v.z; s[3] += v.w;
        }
    }
    T* out = (part_of < 2 ? write_grad : read_grad) + line * L;
    const int64_t t0 = (int64_t)mark * kMark + c * kSteps + (part_of & 1) * 4;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (t0 + k < L) out[t0 + k] = t0 + k < len ? (T)s[k] : (T)0.0f;
}

struct Step {
    const void *tokens, *delta, *gate, *write, *read, *skip, *delta_bias, *slots;
    const float *A, *state;
    float* state_out;
    int64_t tokens_b, delta_b, gate_b, write_b, write_g, read_b, read_g, S;
    int32_t D, N, per_group;
    uint32_t tiles, flags;
};

// One token: four lanes a channel, each takes every fourth group of four states, 16 bytes at a time where N allows;
// a block takes 64 channels of a row.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void selective_step_kernel(Step p, T* __restrict__ out) {
    const uint32_t b = p.tiles == 1 ? blockIdx.x : blockIdx.x / p.tiles;
    const int64_t d = (int64_t)(blockIdx.x - b * p.tiles) * 64 + threadIdx.x / 4;
    const int part = threadIdx.x & 3;
    const int64_t slot = slot_of_row(p.slots, p.flags & FMSELECTIVE_SLOTS_64, (int32_t)b, p.S);
    if (d >= p.D) return;  // whole groups of four lanes
    if (slot < 0) {
        if (part == 0) out[(int64_t)b * p.D + d] = (T)0.0f;
        return;
    }
    const int32_t g = (int32_t)d / p.per_group;
    const float u = Elem<T>::widen(((const T*)p.tokens)[b * p.tokens_b + d]);
    float dt = Elem<T>::widen(((const T*)p.delta)[b * p.delta_b + d]);
    if (p.delta_bias) dt += param<T>(p.delta_bias, d, p.flags & FMSELECTIVE_NARROW_BIAS);
    if (p.flags & FMSELECTIVE_SOFTPLUS) dt = softplus(dt);
    const float dtu = dt * u;
    const T* write = (const T*)p.write + b * p.write_b + g * p.write_g;
    const T* read = (const T*)p.read + b * p.read_b + g * p.read_g;
    const float* A = p.A + d * p.N;
    const float* state = p.state + (slot * p.D + d) * p.N;
    float* state_out = p.state_out + (slot * p.D + d) * p.N;
    float y = 0.0f;
    for (int n0 = part * 4; n0 < p.N; n0 += 16) {
        float a[4], h[4];
        if constexpr (VEC) {  // N is a multiple of 4, the pools and A lie on 16 bytes
            *reinterpret_cast<float4*>(a) = *reinterpret_cast<const float4*>(A + n0);
            *reinterpret_cast<float4*>(h) = *reinterpret_cast<const float4*>(state + n0);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const bool in = n0 + k < p.N;
                a[k] = in ? A[n0 + k] : 0.0f;
                h[k] = in ? state[n0 + k] : 0.0f;
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (!VEC && n0 + k >= p.N) continue;
            h[k] = __builtin_fmaf(exp2_fast(dt * (a[k] * kLog2E)), h[k], dtu * Elem<T>::widen(write[n0 + k]));
            y = __builtin_fmaf(Elem<T>::widen(read[n0 + k]), h[k], y);
        }
        if constexpr (VEC) {
            *reinterpret_cast<float4*>(state_out + n0) = *reinterpret_cast<float4*>(h);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (n0 + k < p.N) state_out[n0 + k] = h[k];
        }
    }
    y += fmscan::dpp<0xb1>(0.0f, y);  // quad_perm 1,0,3,2
    y += fmscan::dpp<0x4e>(0.0f, y);  // quad_perm 2,3,0,1
    if (part) return;
    if (p.skip) y = __builtin_fmaf(param<T>(p.skip, d, p.flags & FMSELECTIVE_NARROW_SKIP), u, y);
    if (p.gate) {
        const float z = Elem<T>::widen(((const T*)p.gate)[b * p.gate_b + d]);
        y *= z * sigmoid(z);
    }
    out[(int64_t)b * p.D + d] = (T)y;
}

}  // namespace fmselective
