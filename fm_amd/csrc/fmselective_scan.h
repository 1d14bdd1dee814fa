// Kernels of the selective scan: forward, backward, one token.
//
//   dt = softplus(delta + delta_bias),  h[n] <- exp(dt A[n]) h[n] + dt u write[n],  y = sum_n read[n] h[n] + skip u
//
// The decay differs for every channel, state and step, so there is no matrix product in it: per (b, d, n, t) one
// exponential and four multiply-adds forward, about twenty operations backward, against at most 14 bytes per
// (b, d, t). With 16 states the kernels are bound by vector float32 arithmetic, not by memory.
//
// Layout. Time runs along the lanes: a lane holds 8 consecutive steps of a channel, 16 lanes (one DPP row) a tile
// of 128 steps, so a wave works on 4 channels at a time and every tensor moves as 16-byte accesses along time. (Forward
// also has tiles of 4 lanes, 32 steps of 16 channels, and of 64, 512 steps of one.)
// For one state of a channel a lane composes its 8 steps (its total decay is one exponential of the steps' sum),
// the row scans the pairs (decay, value) by DPP, and a second walk over the 8 steps with the true entering state
// gives the states; the state that enters the tile joins the scan in its first lane. A block's waves share the tile of
// write and read, kept in LDS as float32 and loaded while the tile before is worked on; the state that leaves a tile
// waits in LDS for the next one.
//
// Tried and not taken, at (8, 2048, 2048) with N = 16 in bf16: the exponents dt A as outer products of the matrix units
// (registers: forward 205 -> 220 to 300 us, backward 605 -> 830); two sets of channels a lane in backward (328 registers,
// 606 -> 748 us); more waves a SIMD by a bound on registers (spills, 591 -> 660 to 750); two states a turn in forward
// (142 registers, 196 -> 214 us; bounded to 128 it spills, 208); blocks of 8 waves in backward (618 + 27 against
// 591 + 49 us).
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

// A state's decay rate in base 2, finite where A is not or the product leaves float32: a step of length zero, such as the steps
// behind a row's end, then leaves every state as it is (0 times infinity would be NaN), and any other forgets it at once.
__device__ __forceinline__ float decay_rate(float A) {
    const float r = A * kLog2E;
    return r < -__FLT_MAX__ ? -__FLT_MAX__ : r;
}

// What the kernels need of include/fmselective.h's fmselective_scan
struct Scan {
    const void *tokens, *delta, *gate, *write, *read, *skip, *delta_bias;
    const float *A, *initial;
    const int32_t* lengths;
    int64_t tokens_b, tokens_d, delta_b, delta_d, gate_b, gate_d, write_b, write_g, write_n, read_b, read_g, read_n;
    int64_t L;
    int32_t D, N, G, per_group, blocks_per_group, marks;  // marks: ceil(L / kMark)
    int32_t segments, seg_tiles;  // a row's tiles are dealt to `segments` blocks, seg_tiles each
    int64_t rows;                 // B D
    float2* pairs;                // (segment, B D, N): what a segment does to a state (or a gradient) that enters it
    uint32_t flags;
};

// (decay, value) pairs composed over the lanes of a channel: on exit a lane holds the composition of its own and
// all earlier lanes' pairs. A register written by a VALU instruction may be read through DPP two wait states later
// at the earliest: the pair's other instruction is one, the s_nop the other.
#define FMSELECTIVE_LEVEL(A, B, CTRL)                     \
    "v_fmac_f32_dpp " B ", " B ", " A " " CTRL "\n\t"     \
    "v_mul_f32_dpp " A ", " A ", " A " " CTRL "\n\t"
#define FMSELECTIVE_LAST(A, B, CTRL) "v_fmac_f32_dpp " B ", " B ", " A " " CTRL "\n\t"
template <int LPC>
__device__ __forceinline__ void scan_up(float& a, float& b) {
    if constexpr (LPC == 4) {  // by quad permutations, which bring a lane no other channel's values
        const int c = threadIdx.x & 3;
        const float pb = fmscan::dpp<0x90>(0.0f, b), pa = fmscan::dpp<0x90>(0.0f, a);  // lanes 0, 0, 1, 2
        b = c ? __builtin_fmaf(pb, a, b) : b;
        a = c ? pa * a : a;
        const float qb = fmscan::dpp<0x44>(0.0f, b);  // lanes 0, 1, 0, 1
        b = c & 2 ? __builtin_fmaf(qb, a, b) : b;
    } else if constexpr (LPC == 16)
        asm("s_nop 1\n\t"
            FMSELECTIVE_LEVEL("%0", "%1", "row_shr:1 row_mask:0xf bank_mask:0xf") "s_nop 0\n\t"
            FMSELECTIVE_LEVEL("%0", "%1", "row_shr:2 row_mask:0xf bank_mask:0xf") "s_nop 0\n\t"
            FMSELECTIVE_LEVEL("%0", "%1", "row_shr:4 row_mask:0xf bank_mask:0xf") "s_nop 0\n\t"
            FMSELECTIVE_LAST("%0", "%1", "row_shr:8 row_mask:0xf bank_mask:0xf")
            "s_nop 1"
            : "+v"(a), "+v"(b));
    else
        asm("s_nop 1\n\t"
            FMSELECTIVE_LEVEL("%0", "%1", "row_shr:1 row_mask:0xf bank_mask:0xf") "s_nop 0\n\t"
            FMSELECTIVE_LEVEL("%0", "%1", "row_shr:2 row_mask:0xf bank_mask:0xf") "s_nop 0\n\t"
            FMSELECTIVE_LEVEL("%0", "%1", "row_shr:4 row_mask:0xf bank_mask:0xf") "s_nop 0\n\t"
            FMSELECTIVE_LEVEL("%0", "%1", "row_shr:8 row_mask:0xf bank_mask:0xf") "s_nop 0\n\t"
            FMSELECTIVE_LEVEL("%0", "%1", "row_bcast:15 row_mask:0xa bank_mask:0xf") "s_nop 0\n\t"
            FMSELECTIVE_LAST("%0", "%1", "row_bcast:31 row_mask:0xc bank_mask:0xf")
            "s_nop 1"
            : "+v"(a), "+v"(b));
}
__device__ __forceinline__ void scan_down(float& a, float& b) {
    asm("s_nop 1\n\t"
        FMSELECTIVE_LEVEL("%0", "%1", "row_shl:1 row_mask:0xf bank_mask:0xf") "s_nop 0\n\t"
        FMSELECTIVE_LEVEL("%0", "%1", "row_shl:2 row_mask:0xf bank_mask:0xf") "s_nop 0\n\t"
        FMSELECTIVE_LEVEL("%0", "%1", "row_shl:4 row_mask:0xf bank_mask:0xf") "s_nop 0\n\t"
        FMSELECTIVE_LAST("%0", "%1", "row_shl:8 row_mask:0xf bank_mask:0xf")
        "s_nop 1"
        : "+v"(a), "+v"(b));
}
// One pair towards higher lanes and one towards lower lanes, inside rows of 16: the two scans fill each other's
// wait states.
__device__ __forceinline__ void scan_both(float& up_a, float& up_b, float& down_a, float& down_b) {
    asm("s_nop 1\n\t"
        FMSELECTIVE_LEVEL("%0", "%1", "row_shr:1 row_mask:0xf bank_mask:0xf")
        FMSELECTIVE_LEVEL("%2", "%3", "row_shl:1 row_mask:0xf bank_mask:0xf")
        FMSELECTIVE_LEVEL("%0", "%1", "row_shr:2 row_mask:0xf bank_mask:0xf")
        FMSELECTIVE_LEVEL("%2", "%3", "row_shl:2 row_mask:0xf bank_mask:0xf")
        FMSELECTIVE_LEVEL("%0", "%1", "row_shr:4 row_mask:0xf bank_mask:0xf")
        FMSELECTIVE_LEVEL("%2", "%3", "row_shl:4 row_mask:0xf bank_mask:0xf")
        FMSELECTIVE_LAST("%0", "%1", "row_shr:8 row_mask:0xf bank_mask:0xf")
        FMSELECTIVE_LAST("%2", "%3", "row_shl:8 row_mask:0xf bank_mask:0xf")
        "s_nop 1"
        : "+v"(up_a), "+v"(up_b), "+v"(down_a), "+v"(down_b));
}
#undef FMSELECTIVE_LEVEL
#undef FMSELECTIVE_LAST

typedef float f32x4 __attribute__((ext_vector_type(4)));

// The value of the lane below of the same channel, in its first lane `first`
template <int LPC>
__device__ __forceinline__ float of_lane_below(float first, float v) {
    if constexpr (LPC == 4) {
        const float below = fmscan::dpp<0x90>(0.0f, v);  // (by all lanes: none reads an inactive one)
        return threadIdx.x & 3 ? below : first;
    } else return fmscan::dpp<LPC == 16 ? 0x111 : fmscan::kWaveShr1>(first, v);  // row_shr 1
}

constexpr int kRowShr1 = 0x111;  // lane i <- lane i-1 inside its row of 16

// 8 steps of a row as they lie in memory
template <typename T>
struct Raw {
    u32x4 v[kSteps / Elem<T>::E];
};
// (whole, the same in all lanes: all their steps count, and the loads need no condition)
template <typename T>
__device__ __forceinline__ Raw<T> load_raw(const T* __restrict__ row, int64_t t0, int64_t len, bool whole) {
    Raw<T> r;
    if (whole) {
#pragma unroll
        for (int i = 0; i < kSteps / Elem<T>::E; ++i) r.v[i] = fmscan::load16<T, false, false>(row + t0 + i * Elem<T>::E);
    } else {
#pragma unroll
        for (int i = 0; i < kSteps / Elem<T>::E; ++i)
            r.v[i] = fmscan::load_chunk<T, false, false>(row, t0 + i * Elem<T>::E, len, 0u);
    }
    return r;
}
template <typename T>
__device__ __forceinline__ void store_steps(T* __restrict__ row, int64_t t0, int64_t L, bool whole, const float (&f)[kSteps]) {
    constexpr int E = Elem<T>::E;
    if (!whole) return store_values<T, kSteps>(row, t0, L, f);
#pragma unroll
    for (int i = 0; i < kSteps / E; ++i) {
        float part[E];
#pragma unroll
        for (int k = 0; k < E; ++k) part[k] = f[i * E + k];
        fmscan::store16<T, false>(row + t0 + i * E, Elem<T>::pack(part));
    }
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
template <int LPC, int NC>
struct SharedTile {
    alignas(16) float v[2][NC][2][LPC][4];  // write / read, state, half, chunk, step
};
// Steps of a lane out of the tile: `at` points to the lane's four floats of a state of `write`
template <int LPC>
__device__ __forceinline__ void steps_at(const float* at, float (&f)[kSteps]) {
    const float4 a = *reinterpret_cast<const float4*>(at), b = *reinterpret_cast<const float4*>(at + 4 * LPC);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

// A thread's part of filling the tile: one or two chunks of 16-bit or 32-bit steps, loaded a tile ahead
template <typename T, int LPC, int NC, int WAVES>
struct TileLoader {
    static constexpr int kChunks = NC * LPC, kEach = 2 * kChunks / (64 * WAVES);
    static_assert(kEach >= 1 && 2 * kChunks % (64 * WAVES) == 0, "whole chunks a thread");
    Raw<T> raw[kEach];
    __device__ __forceinline__ void load(const T* write, int64_t write_n, const T* read, int64_t read_n, int n0, int N,
                                         int64_t tile_t0, int64_t len) {
        const bool whole = n0 + NC <= N && tile_t0 + LPC * kSteps <= len;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int i = threadIdx.x + j * 64 * WAVES, which = i / kChunks, n = n0 + (i / LPC) % NC, c = i % LPC;
            const T* rows = which ? read + n * read_n : write + n * write_n;
            raw[j] = load_raw<T>(rows, tile_t0 + c * kSteps, n < N ? len : 0, whole);
        }
    }
    __device__ __forceinline__ void put(SharedTile<LPC, NC>& t) const {
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int i = threadIdx.x + j * 64 * WAVES, which = i / kChunks, n = (i / LPC) % NC, c = i % LPC;
            float f[kSteps];
            widen_raw(raw[j], f);
            *reinterpret_cast<float4*>(t.v[which][n][0][c]) = make_float4(f[0], f[1], f[2], f[3]);
            *reinterpret_cast<float4*>(t.v[which][n][1][c]) = make_float4(f[4], f[5], f[6], f[7]);
        }
    }
};

// entries between the states of two channels in LDS: odd, so that channels do not share banks
__host__ __device__ __forceinline__ int state_stride(int N) { return N | 1; }

// Forward keeps two tiles of kStates states in LDS (one being filled), backward one
template <int LPC, int WAVES>
constexpr int tile_states() { return LPC == 64 ? WAVES : LPC == 16 ? 16 : 32; }
template <int LPC, int WAVES>
size_t scan_forward_lds(int N) {
    return 2 * sizeof(SharedTile<LPC, tile_states<LPC, WAVES>()>) + (size_t)WAVES * (64 / LPC) * state_stride(N) * sizeof(float2);
}

// Steps that count among the 8 from t0
__device__ __forceinline__ int steps_left(int64_t len, int64_t t0) {
    const int64_t n = len - t0;
    return n < 0 ? 0 : (n > kSteps ? kSteps : (int)n);
}

// The block's part of the problem
struct Place {
    uint32_t b, g, block;
    int32_t seg;
    int64_t line;  // of the block without its segment
};
__device__ __forceinline__ Place place_of(const Scan& p) {
    Place w;
    const uint32_t line = p.segments == 1 ? blockIdx.x : blockIdx.x / (uint32_t)p.segments;
    w.seg = (int32_t)(blockIdx.x - line * p.segments);
    const uint32_t bg = line / (uint32_t)p.blocks_per_group;
    w.block = line - bg * p.blocks_per_group;
    w.b = bg / (uint32_t)p.G;
    w.g = bg - w.b * p.G;
    w.line = line;
    return w;
}

// dt of a lane's steps from the raw delta
__device__ __forceinline__ void steps_of(float (&dt)[kSteps], float bias, uint32_t flags, bool ragged, int left) {
#pragma unroll
    for (int k = 0; k < kSteps; ++k) dt[k] += bias;
    if (flags & FMSELECTIVE_SOFTPLUS) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) dt[k] = softplus(dt[k]);
    }
    if (ragged) {  // a step of length zero leaves the state as it is
#pragma unroll
        for (int k = 0; k < kSteps; ++k) dt[k] = k < left ? dt[k] : 0.0f;
    }
}

// Forward over the tiles of a segment. Where rows are too few to fill the GPU they are cut into segments: a first
// launch (ENDS) finds what each segment but the last does to a state, without the outputs; the second composes
// the segments before its own, as many multiply-adds a state, and then runs as for a whole row.
// Bound by vector instructions: a state and step is 8 of them (two walks of 8 steps, the scan between them, the exponential
// at half rate) and 3 more are the steps' own softplus, gate and conversions. With N = 16 in bf16 196 us at (8, 2048, 2048),
// 2.7e12 states a second, the SIMDs busy for 90 % of it; 409 us at (1, 4096, 16384), 2.6e12.
template <typename T, int LPC, int WAVES, bool ENDS>
__global__ __launch_bounds__(64 * WAVES) void selective_forward_kernel(Scan p, T* __restrict__ out, float* __restrict__ final_state,
                                                                       float* __restrict__ marks) {
    static_assert(LPC == 64 || !ENDS, "only rows of 64 lanes are cut");
    constexpr int NC = tile_states<LPC, WAVES>(), kTile = LPC * kSteps, CW = 64 / LPC;
    using Tile = SharedTile<LPC, NC>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    Tile* tiles = reinterpret_cast<Tile*>(lds);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & (LPC - 1), ch = lane / LPC;

    const Place w = place_of(p);
    const uint32_t b = w.b, g = w.g;
    const int32_t local = (int32_t)(w.block * WAVES + wave) * CW + ch;  // the lane's channel in the group
    const bool valid = local < p.per_group;
    const int32_t d = (int32_t)g * p.per_group + (valid ? local : p.per_group - 1);
    const int64_t row = (int64_t)b * p.D + d;
    const int64_t len = row_length(p.lengths, b, p.L), mine = valid ? len : 0;  // (no steps for a channel beyond the group)
    const bool all_valid = __all(valid);
    const T* u_row = (const T*)p.tokens + b * p.tokens_b + d * p.tokens_d;
    const T* delta_row = (const T*)p.delta + b * p.delta_b + d * p.delta_d;
    const T* gate_row = p.gate ? (const T*)p.gate + b * p.gate_b + d * p.gate_d : nullptr;
    const T* write_rows = (const T*)p.write + b * p.write_b + g * p.write_g;
    const T* read_rows = (const T*)p.read + b * p.read_b + g * p.read_g;
    const float skip = p.skip ? param<T>(p.skip, d, p.flags & FMSELECTIVE_NARROW_SKIP) : 0.0f;
    const float bias = p.delta_bias ? param<T>(p.delta_bias, d, p.flags & FMSELECTIVE_NARROW_BIAS) : 0.0f;

    // the lane's channel's decay rates (A log2 e) and the states that enter the tile
    float2* held = reinterpret_cast<float2*>(lds + 2 * sizeof(Tile)) + (wave * CW + ch) * state_stride(p.N);
    for (int n = c; n < p.N; n += LPC) {
        float h = !ENDS && valid && p.initial ? p.initial[row * p.N + n] : 0.0f;
        if (!ENDS && valid) {
#pragma unroll 4
            for (int32_t j = 0; j < w.seg; ++j) {
                const float2 q = p.pairs[(j * p.rows + row) * p.N + n];
                h = __builtin_fmaf(q.x, h, q.y);
            }
        }
        held[n] = make_float2(decay_rate(p.A[(int64_t)d * p.N + n]), h);
    }

    const int chunks = (p.N + NC - 1) / NC;
    const int32_t row_tiles = (int32_t)((len + kTile - 1) / kTile), first_tile = w.seg * p.seg_tiles;
    const int32_t seg_end = first_tile + p.seg_tiles, n_tiles = row_tiles < seg_end ? row_tiles : seg_end;  // the last one, exclusive
    const int32_t total = n_tiles > first_tile ? (n_tiles - first_tile) * chunks : 0;
    float all_dt = 0.0f;
    TileLoader<T, LPC, NC, WAVES> loader;
    Raw<T> next_u, next_delta, next_gate = {};
    auto fetch_shared = [&](int32_t tile, int chunk) {
        loader.load(write_rows, p.write_n, read_rows, p.read_n, chunk * NC, p.N, (int64_t)tile * kTile, len);
    };
    auto fetch_rows = [&](int32_t tile) {
        const int64_t t0 = (int64_t)tile * kTile + c * kSteps;
        const bool whole = all_valid && (int64_t)(tile + 1) * kTile <= len;
        next_u = load_raw<T>(u_row, t0, mine, whole);
        next_delta = load_raw<T>(delta_row, t0, mine, whole);
        if (!ENDS && gate_row) next_gate = load_raw<T>(gate_row, t0, mine, whole);
    };
    if (total) {
        fetch_shared(first_tile, 0);
        fetch_rows(first_tile);
        loader.put(tiles[0]);
    }
    __syncthreads();

    float dt[kSteps], dtu[kSteps], y[kSteps], total_dt = 0.0f;
    Raw<T> gate_now = {};
    int32_t it = 0;
    for (int32_t tile = first_tile; tile < n_tiles; ++tile) {
        const int64_t t0 = (int64_t)tile * kTile + c * kSteps;
        const bool ragged = (int64_t)(tile + 1) * kTile > len;  // the row's last tile
        {
            float u[kSteps];
            widen_raw(next_u, u);
            widen_raw(next_delta, dt);
            gate_now = next_gate;
            steps_of(dt, bias, p.flags, ragged, ragged ? steps_left(mine, t0) : kSteps);
            total_dt = 0.0f;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                dtu[k] = dt[k] * u[k];
                y[k] = skip * u[k];
                total_dt += dt[k];
            }
            if (tile + 1 < n_tiles) fetch_rows(tile + 1);
        }
        if (ENDS) all_dt += total_dt;
        constexpr int kMarkTiles = kTile < kMark ? kMark / kTile : 1;
        if (LPC != 64 && !ENDS && marks && valid && tile % kMarkTiles == 0) {
            float* mark = marks + (row * p.marks + tile / kMarkTiles) * p.N;
            for (int n = c; n < p.N; n += LPC) mark[n] = held[n].y;
        }
        for (int chunk = 0; chunk < chunks; ++chunk, ++it) {
            if (it + 1 < total) fetch_shared(chunk + 1 < chunks ? tile : tile + 1, chunk + 1 < chunks ? chunk + 1 : 0);
            const int n0 = chunk * NC, n_end = p.N - n0 < NC ? p.N - n0 : NC;
            const float* at = tiles[it & 1].v[0][0][0][c];
            float2* state = held + n0;
            for (int n = 0; n < n_end; ++n, at += 8 * LPC, ++state) {
                float a[kSteps], v[kSteps], r[kSteps];
                const float2 e = *state;
                steps_at<LPC>(at, v);
                if (!ENDS) steps_at<LPC>(at + NC * 8 * LPC, r);
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    a[k] = exp2_fast(dt[k] * e.x);
                    v[k] *= dtu[k];
                }
                float S = v[0], P = exp2_fast(total_dt * e.x);
#pragma unroll
                for (int k = 1; k < kSteps; ++k) S = __builtin_fmaf(a[k], S, v[k]);
                S = __builtin_fmaf(P, c == 0 ? e.y : 0.0f, S);  // the first lane starts from the state that enters the tile
                scan_up<LPC>(P, S);
                if (c == LPC - 1) state->y = S;
                if (ENDS) continue;
                float h = of_lane_below<LPC>(e.y, S);
                if (LPC == 64 && marks && (c & 15) == 0) {
                    const int32_t mark = tile * (LPC / 16) + c / 16;
                    if (valid && mark < p.marks) marks[(row * p.marks + mark) * p.N + n0 + n] = h;
                }
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    h = __builtin_fmaf(a[k], h, v[k]);
                    y[k] = __builtin_fmaf(r[k], h, y[k]);
                }
            }
            if (it + 1 < total) loader.put(tiles[(it + 1) & 1]);
            __syncthreads();
        }
        if (ENDS) continue;
        if (gate_row) {
            float z[kSteps];
            widen_raw(gate_now, z);
#pragma unroll
            for (int k = 0; k < kSteps; ++k) y[k] *= z[k] * sigmoid(z[k]);
        }
        if (ragged) {
            const int left = steps_left(mine, t0);
#pragma unroll
            for (int k = 0; k < kSteps; ++k) y[k] = k < left ? y[k] : 0.0f;
        }
        if (valid) store_steps<T>(out + row * p.L, t0, p.L, !ragged, y);
    }
    if constexpr (ENDS) {
        // (the total's decay in one exponential of the summed steps, as within a tile)
        all_dt = row_sum(all_dt);
        all_dt = fmscan::lane_value(all_dt, 15) + fmscan::lane_value(all_dt, 31) + fmscan::lane_value(all_dt, 47) +
                 fmscan::lane_value(all_dt, 63);
        if (valid)
            for (int n = c; n < p.N; n += LPC)
                p.pairs[((int64_t)w.seg * p.rows + row) * p.N + n] = make_float2(exp2_fast(all_dt * held[n].x), held[n].y);
        return;
    }
#pragma unroll
    for (int k = 0; k < kSteps; ++k) y[k] = 0.0f;
    if (valid) {
        const int64_t end = (int64_t)seg_end * kTile < p.L ? (int64_t)seg_end * kTile : p.L;
        for (int64_t t0 = (int64_t)(n_tiles > first_tile ? n_tiles : first_tile) * kTile + c * kSteps; t0 < end; t0 += kTile)
            store_values<T, kSteps>(out + row * p.L, t0, p.L, y);
        if (final_state && w.seg == p.segments - 1)
            for (int n = c; n < p.N; n += LPC) final_state[row * p.N + n] = held[n].y;
    }
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

// LDS of the backward kernel: the shared tile, the waves' sums of two states (twice: one being read), and per
// channel and state A log2 e, the gradient that arrives from later steps, the sum for dA, the state before the tile
template <int WAVES>
constexpr size_t scan_sums_bytes() { return (size_t)2 * WAVES * 2 * 256 * sizeof(float); }
template <int WAVES>
size_t scan_backward_lds(int N) {
    return sizeof(SharedTile<16, 16>) + scan_sums_bytes<WAVES>() + (size_t)WAVES * 4 * state_stride(N) * sizeof(float4);
}

// Backward. The tiles are walked from the last to the first. In a tile the states are made again from the state that
// forward saved before it, the gradient of the state runs against time through the same decays, and
//   dh[t] = g[t] read[t] + a[t+1] dh[t+1]     g = out_grad * silu(gate)
//   dtokens = dt sum_n dh write + skip g      dA = sum_t dt p      p = dh a h[t-1]
//   ddt = u sum_n dh write + sum_n A p        dwrite = sum_d dh dt u      dread = sum_d g h
// The sums over n stay in registers, those over time are added up in LDS, one float a state and channel. The sums
// over the channels are made in the wave (4 channels side by side), over the block's waves in LDS and over the
// blocks by a second kernel, always in the same order.
// Rows that are too few to fill the GPU are cut into segments, as in forward: the first launch (ENDS) finds what each
// segment but the first hands on of a gradient that enters it from behind.
// Bound by vector instructions, about 28 a state and step, at two waves a SIMD (237 registers): 553 us at (8, 2048, 2048),
// N = 16 in bf16, the SIMDs busy for 85 % of it. What it leaves for the sums over the channels is 268 MB there.
template <typename T, int WAVES, bool ENDS>
__global__ __launch_bounds__(64 * WAVES) void selective_backward_kernel(Scan p, ScanGrads o) {
    constexpr int LPC = 16, NC = 16, kTile = LPC * kSteps;
    using Tile = SharedTile<LPC, NC>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    Tile& shared = *reinterpret_cast<Tile*>(lds);
    float* sums = reinterpret_cast<float*>(lds + sizeof(Tile));  // [parity][wave][state of the pair][256]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, ch = lane >> 4;

    const Place at = place_of(p);
    const uint32_t b = at.b, g = at.g;
    const int32_t local = (int32_t)(at.block * WAVES + wave) * 4 + ch;  // the lane's channel in the group
    const bool valid = local < p.per_group;
    const int32_t d = (int32_t)g * p.per_group + (valid ? local : p.per_group - 1);
    const int64_t row = (int64_t)b * p.D + d;
    const int64_t len = row_length(p.lengths, b, p.L), mine = valid ? len : 0;
    const bool all_valid = __all(valid);
    const float skip = p.skip ? param<T>(p.skip, d, p.flags & FMSELECTIVE_NARROW_SKIP) : 0.0f;
    const float bias = p.delta_bias ? param<T>(p.delta_bias, d, p.flags & FMSELECTIVE_NARROW_BIAS) : 0.0f;
    float skip_sum = 0.0f, bias_sum = 0.0f, all_dt = 0.0f;
    const T* u_row = (const T*)p.tokens + b * p.tokens_b + d * p.tokens_d;
    const T* delta_row = (const T*)p.delta + b * p.delta_b + d * p.delta_d;
    const T* gate_row = p.gate ? (const T*)p.gate + b * p.gate_b + d * p.gate_d : nullptr;
    const T* dy_row = (const T*)o.out_grad + b * o.out_b + d * o.out_d;
    const T* write_rows = (const T*)p.write + b * p.write_b + g * p.write_g;
    const T* read_rows = (const T*)p.read + b * p.read_b + g * p.read_g;

    float4* held = reinterpret_cast<float4*>(lds + sizeof(Tile) + scan_sums_bytes<WAVES>()) + (wave * 4 + ch) * state_stride(p.N);
    for (int n = c; n < p.N; n += LPC) {
        float e = 0.0f, rate = 0.0f;
        if (valid) {
            const int64_t at_n = row * p.N + n;
            rate = decay_rate(p.A[(int64_t)d * p.N + n]);
            if (!ENDS) {
                if (o.final_grad) e = o.final_grad[at_n];
#pragma unroll 4
                for (int32_t j = p.segments - 1; j > at.seg; --j) {
                    const float2 q = p.pairs[j * p.rows * p.N + at_n];
                    e = __builtin_fmaf(q.x, e, q.y);
                }
            }
        }
        held[n] = make_float4(rate, e, 0.0f, 0.0f);
    }

    const int chunks = (p.N + NC - 1) / NC;
    const int32_t row_tiles = (int32_t)((len + kTile - 1) / kTile), first_tile = at.seg * p.seg_tiles;
    const int32_t seg_end = first_tile + p.seg_tiles, n_tiles = row_tiles < seg_end ? row_tiles : seg_end;
    TileLoader<T, LPC, NC, WAVES> loader;
    auto fetch_shared = [&](int32_t tile, int chunk) {
        loader.load(write_rows, p.write_n, read_rows, p.read_n, chunk * NC, p.N, (int64_t)tile * kTile, len);
    };
    if (n_tiles > first_tile) fetch_shared(n_tiles - 1, 0);

    uint32_t parity = 0;
    float* part = ENDS ? nullptr : o.shared_part + at.line * p.N * p.marks * 256;
    for (int32_t tile = n_tiles - 1; tile >= first_tile; --tile) {
        const int64_t t0 = (int64_t)tile * kTile + c * kSteps;
        const bool ragged = (int64_t)(tile + 1) * kTile > len;
        const int left = ragged ? steps_left(mine, t0) : kSteps;
        float dt[kSteps], dtu[kSteps], gy[kSteps], sum_w[kSteps], sum_a[kSteps], y[kSteps], total_dt = 0.0f;
        const bool whole = all_valid && !ragged;
        const Raw<T> raw_d = load_raw<T>(delta_row, t0, mine, whole), raw_g = load_raw<T>(dy_row, t0, mine, whole);
        Raw<T> raw_u = {}, raw_z = {};
        {
            if (!ENDS) raw_u = load_raw<T>(u_row, t0, mine, whole);
            if (gate_row) raw_z = load_raw<T>(gate_row, t0, mine, whole);
            if (!ENDS)
                for (int n = c; n < p.N; n += LPC) held[n].w = valid ? o.marks[(row * p.marks + tile) * p.N + n] : 0.0f;
            float u[kSteps], z[kSteps];
            widen_raw(raw_d, dt);
            widen_raw(raw_g, gy);
            steps_of(dt, bias, p.flags, ragged, left);
            if (gate_row) {
                widen_raw(raw_z, z);
#pragma unroll
                for (int k = 0; k < kSteps; ++k) gy[k] *= z[k] * sigmoid(z[k]);
            }
            widen_raw(raw_u, u);
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                dtu[k] = dt[k] * u[k];
                total_dt += dt[k];
                sum_w[k] = sum_a[k] = y[k] = 0.0f;
            }
            if (ENDS) all_dt += total_dt;
        }
        for (int chunk = 0; chunk < chunks; ++chunk) {
            loader.put(shared);
            if (chunk + 1 < chunks) fetch_shared(tile, chunk + 1);
            else if (tile > first_tile) fetch_shared(tile - 1, 0);
            __syncthreads();
            const int n0 = chunk * NC, n_end = p.N - n0 < NC ? p.N - n0 : NC;
            const float* steps = shared.v[0][0][0][c];
            float4* state = held + n0;
            for (int n = 0; n < n_end; ++n, steps += 8 * LPC, ++state) {
                float w[kSteps], rd[kSteps];
                if (!ENDS) steps_at<LPC>(steps, w);
                steps_at<LPC>(steps + NC * 8 * LPC, rd);
                const float4 e = *state;
                float a[kSteps], h[kSteps], dh[kSteps];
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    a[k] = exp2_fast(dt[k] * e.x);
                    dh[k] = rd[k] * gy[k];
                    if (!ENDS) h[k] = w[k] * dtu[k];
                }
                float S = 0.0f, P = exp2_fast(total_dt * e.x), D = dh[kSteps - 1], Q = P;
#pragma unroll
                for (int k = kSteps - 1; k > 0; --k) D = __builtin_fmaf(a[k], D, dh[k - 1]);
                D = __builtin_fmaf(Q, c == LPC - 1 ? e.y : 0.0f, a[0] * D);  // the last lane starts from what arrives
                if constexpr (ENDS) {
                    scan_down(Q, D);
                    if (c == 0) state->y = D;
                    continue;
                }
                S = h[0];
#pragma unroll
                for (int k = 1; k < kSteps; ++k) S = __builtin_fmaf(a[k], S, h[k]);
                S = __builtin_fmaf(P, c == 0 ? e.w : 0.0f, S);
                scan_both(P, S, Q, D);
                const float enter = fmscan::dpp<kRowShr1>(e.w, S);
                float back = fmscan::dpp<fmscan::kRowShl1>(e.y, D);
                if (c == 0) state->y = D;
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    h[k] = __builtin_fmaf(a[k], k ? h[k - 1] : enter, h[k]);
                    y[k] = __builtin_fmaf(rd[k], h[k], y[k]);
                }
                float in_time = 0.0f, half[kSteps];
#pragma unroll
                for (int k = kSteps - 1; k >= 0; --k) {
                    dh[k] += back;
                    back = a[k] * dh[k];
                    const float pk = back * (k ? h[k - 1] : enter);
                    sum_w[k] = __builtin_fmaf(dh[k], w[k], sum_w[k]);
                    sum_a[k] = __builtin_fmaf(e.x, pk, sum_a[k]);
                    in_time = __builtin_fmaf(dt[k], pk, in_time);
                    // The 4 channels side by side: a swap exchanges halves of two registers, so that one addition
                    // settles both. First the halves of the wave: lanes below 32 keep write's sums, the others
                    // read's.
                    const auto s = __builtin_amdgcn_permlane32_swap(f2u(dh[k] * dtu[k]), f2u(gy[k] * h[k]), false, false);
                    half[k] = u2f(s[0]) + u2f(s[1]);
                }
                in_time = row_sum(in_time);
                if (c == 15) state->z = e.z + in_time;
                // then the rows of a half: the even one keeps steps 0 to 3, the odd one 4 to 7
                float4 row_sums;
                float* q = &row_sums.x;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const auto s = __builtin_amdgcn_permlane16_swap(f2u(half[k]), f2u(half[k + 4]), false, false);
                    q[k] = u2f(s[0]) + u2f(s[1]);
                }
                reinterpret_cast<float4*>(sums + ((parity * WAVES + wave) * 2 + (n & 1)) * 256)[lane] = row_sums;
                if ((n & 1) || n + 1 == n_end) {
                    // two states (or the last one): their 512 sums over the waves, dealt to all threads
                    __syncthreads();
                    constexpr int V = 512 / (64 * WAVES);
                    const int f = threadIdx.x * V, n_first = n0 + (n & ~1);
                    if (n_first + f / 256 <= n0 + n) {
                        float total[V];
                        const float* from = sums + parity * WAVES * 512 + f;
#pragma unroll
                        for (int i = 0; i < V; ++i) total[i] = from[i];
#pragma unroll
                        for (int v = 1; v < WAVES; ++v)
#pragma unroll
                            for (int i = 0; i < V; ++i) total[i] += from[v * 512 + i];
                        float* to = part + ((int64_t)(n_first + f / 256) * p.marks + tile) * 256 + f % 256;
#pragma unroll
                        for (int i = 0; i < V; ++i) to[i] = total[i];
                    }
                    parity ^= 1;
                }
            }
            __syncthreads();  // the tile may be filled again
        }
        if (ENDS) continue;
        float u[kSteps], dd[kSteps], x[kSteps], z[kSteps];
        widen_raw(raw_u, u);
        widen_raw(raw_d, x);
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            dd[k] = __builtin_fmaf(u[k], sum_w[k], kLn2 * sum_a[k]);
            if (p.flags & FMSELECTIVE_SOFTPLUS) dd[k] *= sigmoid(x[k] + bias);
            x[k] = __builtin_fmaf(dt[k], sum_w[k], skip * gy[k]);
            y[k] = __builtin_fmaf(skip, u[k], y[k]);
        }
        if (ragged) {
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                dd[k] = k < left ? dd[k] : 0.0f;
                x[k] = k < left ? x[k] : 0.0f;
            }
        }
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            bias_sum += dd[k];
            skip_sum = __builtin_fmaf(gy[k], u[k], skip_sum);
        }
        if (valid) {
            store_steps<T>((T*)o.tokens + row * p.L, t0, p.L, !ragged, x);
            store_steps<T>((T*)o.delta + row * p.L, t0, p.L, !ragged, dd);
        }
        if (gate_row) {
            widen_raw(raw_g, dd);
            widen_raw(raw_z, z);
#pragma unroll
            for (int k = 0; k < kSteps; ++k) dd[k] *= y[k] * silu_slope(z[k], sigmoid(z[k]));
            if (ragged) {
#pragma unroll
                for (int k = 0; k < kSteps; ++k) dd[k] = k < left ? dd[k] : 0.0f;
            }
            if (valid) store_steps<T>((T*)o.gate + row * p.L, t0, p.L, !ragged, dd);
        }
    }
    if constexpr (ENDS) {
        all_dt = __shfl(row_sum(all_dt), lane | 15);
        if (valid)
            for (int n = c; n < p.N; n += LPC)
                p.pairs[((int64_t)at.seg * p.rows + row) * p.N + n] = make_float2(exp2_fast(all_dt * held[n].x), held[n].y);
        return;
    }
    float zero[kSteps];
#pragma unroll
    for (int k = 0; k < kSteps; ++k) zero[k] = 0.0f;
    skip_sum = row_sum(skip_sum);
    bias_sum = row_sum(bias_sum);
    if (!valid) return;
    const int64_t end = (int64_t)seg_end * kTile < p.L ? (int64_t)seg_end * kTile : p.L;
    for (int64_t t0 = (int64_t)(n_tiles > first_tile ? n_tiles : first_tile) * kTile + c * kSteps; t0 < end; t0 += kTile) {
        store_values<T, kSteps>((T*)o.tokens + row * p.L, t0, p.L, zero);
        store_values<T, kSteps>((T*)o.delta + row * p.L, t0, p.L, zero);
        if (gate_row) store_values<T, kSteps>((T*)o.gate + row * p.L, t0, p.L, zero);
    }
    const int64_t part_row = (int64_t)at.seg * p.rows + row;
    if (c == 15) {
        if (o.skip_part) o.skip_part[part_row] = skip_sum;
        if (o.bias_part) o.bias_part[part_row] = bias_sum;
    }
    for (int n = c; n < p.N; n += LPC) {
        o.A_part[part_row * p.N + n] = held[n].z;
        if (o.initial && at.seg == 0) o.initial[row * p.N + n] = held[n].y;
    }
}

// The last sums of a backward call, in one launch. The first blocks take the parameters' gradients (column_sums); the
// others the gradients of write and read: the partial sums added up in a fixed order and rounded once, `per` waves of
// a block for one (b, g, n, mark), each every per-th partial sum, a float4 a lane, in the order that the backward
// kernel left them. Bound by memory: 62 us for 268 MB at (8, 2048, 2048), N = 16, 4.4 TB/s.
template <typename T>
__global__ __launch_bounds__(64 * kSumWaves) void selective_sums_kernel(ColumnSums columns, uint32_t column_blocks,
                                                                        const float* __restrict__ part, T* __restrict__ write_grad,
                                                                        T* __restrict__ read_grad, const int32_t* __restrict__ lengths,
                                                                        int64_t L, int64_t items, int32_t N, int32_t G,
                                                                        int32_t marks, int32_t blocks, int32_t per) {
    if (blockIdx.x < column_blocks) {
        column_sums<T>(columns, blockIdx.x);
        return;
    }
    __shared__ float4 shared[kSumWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, turn = wave & (per - 1);
    const int64_t item = ((int64_t)(blockIdx.x - column_blocks) * kSumWaves + wave) / (uint32_t)per;
    const int64_t line = item / marks;  // (b, g, n)
    const int32_t mark = (int32_t)(item - line * marks);
    const int64_t bg = line / N;
    const int32_t n = (int32_t)(line - bg * N);
    const int64_t len = item < items ? row_length(lengths, bg / G, L) : 0;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if ((int64_t)mark * kMark < len) {
        const float4* at = reinterpret_cast<const float4*>(part) + (((bg * blocks) * N + n) * marks + mark) * 64 + lane;
        const int64_t step = (int64_t)N * marks * 64;
#pragma unroll 4
        for (int32_t i = turn; i < blocks; i += per) {
            const float4 v = at[i * step];
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
    }
    shared[wave][lane] = s;
    __syncthreads();
    if (turn || item >= items) return;
    for (int w = 1; w < per; ++w) {
        const float4 v = shared[wave + w][lane];
        s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    const float sum[4] = {s.x, s.y, s.z, s.w};
    const int part_of = lane >> 4, c = lane & 15;
    T* out = (part_of < 2 ? write_grad : read_grad) + line * L;
    const int64_t t0 = (int64_t)mark * kMark + c * kSteps + (part_of & 1) * 4;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (t0 + k < L) out[t0 + k] = t0 + k < len ? (T)sum[k] : (T)0.0f;
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
// a block takes 64 channels of a row, CH times. The row's `write` and `read` serve all its channels of a group.
// Bound by the pool's traffic: what does not depend on the slot is loaded before it is known, and the new states, which
// this call does not read again, are stored past the caches (47 -> 35 us at 256 rows of 4096 channels with 16 states;
// 29 us, 4.9 TB/s, with two channels a lane). That is one pool called again and again, which the last-level cache keeps: over
// eight pools in turn, as the layers of a model have them, 41 us, 3.5 TB/s, and 44 us updating in place. 3.2 us at one row of 2048.
template <typename T, bool VEC, int CH>
__global__ __launch_bounds__(256) void selective_step_kernel(Step p, T* __restrict__ out) {
    const uint32_t b = p.tiles == 1 ? blockIdx.x : blockIdx.x / p.tiles;
    const int64_t first = (int64_t)(blockIdx.x - b * p.tiles) * (64 * CH) + threadIdx.x / 4;
    const int part = threadIdx.x & 3;
    float u[CH], dt[CH], z[CH], skip[CH], y[CH];
    int32_t g[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int64_t d = first + 64 * i < p.D ? first + 64 * i : p.D - 1;  // (a lane beyond the last channel repeats it)
        u[i] = Elem<T>::widen(((const T*)p.tokens)[b * p.tokens_b + d]);
        dt[i] = Elem<T>::widen(((const T*)p.delta)[b * p.delta_b + d]);
        z[i] = p.gate ? Elem<T>::widen(((const T*)p.gate)[b * p.gate_b + d]) : 0.0f;
        if (p.delta_bias) dt[i] += param<T>(p.delta_bias, d, p.flags & FMSELECTIVE_NARROW_BIAS);
        skip[i] = p.skip ? param<T>(p.skip, d, p.flags & FMSELECTIVE_NARROW_SKIP) : 0.0f;
        g[i] = p.per_group == p.D ? 0 : (int32_t)d / p.per_group;
        y[i] = 0.0f;
    }
    const int64_t slot = slot_of_row(p.slots, p.flags & FMSELECTIVE_SLOTS_64, (int32_t)b, p.S);
    if (slot < 0) {
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (part == 0 && first + 64 * i < p.D) out[(int64_t)b * p.D + first + 64 * i] = (T)0.0f;
        return;
    }
#pragma unroll
    for (int i = 0; i < CH; ++i)
        if (p.flags & FMSELECTIVE_SOFTPLUS) dt[i] = softplus(dt[i]);
    const T* write = (const T*)p.write + b * p.write_b;
    const T* read = (const T*)p.read + b * p.read_b;
    const float* state = p.state + slot * p.D * p.N;
    float* state_out = p.state_out + slot * p.D * p.N;
    for (int n0 = part * 4; n0 < p.N; n0 += 16) {
        float a[CH][4], h[CH][4], w[4], r[4];
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int64_t d = first + 64 * i < p.D ? first + 64 * i : p.D - 1;
            if constexpr (VEC) {  // N is a multiple of 4, the pools and A lie on 16 bytes
                *reinterpret_cast<f32x4*>(h[i]) = *reinterpret_cast<const f32x4*>(state + d * p.N + n0);
                *reinterpret_cast<f32x4*>(a[i]) = *reinterpret_cast<const f32x4*>(p.A + d * p.N + n0);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const bool in = n0 + k < p.N;
                    h[i][k] = in ? state[d * p.N + n0 + k] : 0.0f;
                    a[i][k] = in ? p.A[d * p.N + n0 + k] : 0.0f;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            if (i == 0 || g[i] != g[i ? i - 1 : 0]) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const bool in = VEC || n0 + k < p.N;
                    w[k] = in ? Elem<T>::widen(write[g[i] * p.write_g + n0 + k]) : 0.0f;
                    r[k] = in ? Elem<T>::widen(read[g[i] * p.read_g + n0 + k]) : 0.0f;
                }
            }
            const float dtu = dt[i] * u[i];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                h[i][k] = __builtin_fmaf(exp2_fast(dt[i] * decay_rate(a[i][k])), h[i][k], dtu * w[k]);
                y[i] = __builtin_fmaf(r[k], h[i][k], y[i]);
            }
            const int64_t d = first + 64 * i;
            if (d >= p.D) continue;
            if constexpr (VEC) {
                __builtin_nontemporal_store(*reinterpret_cast<f32x4*>(h[i]), reinterpret_cast<f32x4*>(state_out + d * p.N + n0));
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (n0 + k < p.N) state_out[d * p.N + n0 + k] = h[i][k];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        y[i] += fmscan::dpp<0xb1>(0.0f, y[i]);  // quad_perm 1,0,3,2
        y[i] += fmscan::dpp<0x4e>(0.0f, y[i]);  // quad_perm 2,3,0,1
        if (p.skip) y[i] = __builtin_fmaf(skip[i], u[i], y[i]);
        if (p.gate) y[i] *= z[i] * sigmoid(z[i]);
        if (part == 0 && first + 64 * i < p.D) out[(int64_t)b * p.D + first + 64 * i] = (T)y[i];
    }
}

}  // namespace fmselective
