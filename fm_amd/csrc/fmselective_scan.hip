// The selective scan's forward call and its form for one token. Contract: include/fmselective.h.
#include "fmselective_scan_host.h"

using namespace fmselective::host;
using fmselective::Scan;

namespace {

// Lanes a channel: 16, so that a wave works on 4 channels, all 64, so that four times as many waves work on tiles of
// four times the length, or 4, so that a quarter as many work on tiles of 32 steps. Measured for N = 16, bf16, on tiles of
// one wave: with up to two waves a SIMD a tile takes 5 to 7 us of 16 lanes (128 steps of four channels) or of 4 (32 of 16)
// and 7 to 8 us of 64 (512 of one), the instructions' latency; with more it is their number that counts, 3.1, 3.9 and
// 3.5 us for each of a SIMD's waves. The fastest by that is taken: (7, 1024, 515) 57 -> 40 us with 16 lanes against 64,
// (1, 4096, 16384) 680 -> 440 with 64 against 16, (1, 4096, 500) 26 -> 20; with 4 against 16 lanes (64, 4096, 8) 170 -> 51,
// (32, 2048, 64) 47 -> 28, (16, 4096, 150) 91 -> 69, but (8, 4096, 200) 47 -> 52, (16, 4096, 100) 55 both. (The rule does not
// know N or the type: it is not measured far from N = 16, nor for float32, whose kernels hold more registers.)
// Where 64 lanes leave less than two waves a SIMD the rows are cut, for four: (1, 1024, 16384) 225 -> 179 us,
// (1, 512, 16384) 112 -> 95 (against a cut for two).
constexpr int64_t kSimds = 1024;
constexpr int64_t kCutBelow = 2 * kSimds, kCutWant = 4 * kSimds;
int64_t modelled_time(int64_t tiles, int64_t waves, int64_t latency, int64_t each) {  // in units of 0.1 us / 1024
    const int64_t busy = each * waves;
    return tiles * (busy > latency * kSimds ? busy : latency * kSimds);
}

// A single token's call: blocks of 64 channels from which on a block takes 128 instead, two channels a lane. Measured with
// one, two and four (bf16, N = 16, us, four pools in turn, which no cache holds; a single one is kept by the last-level cache and
// takes 29 with two): (256, 4096) 46, 40, 45; (1024, 1024) 50, 42, 46; (64, 4096) 15 each.
constexpr int64_t kManyStepBlocks = 4096;

struct ForwardPlan {
    int lanes;
    Cut cut;
    size_t bytes;  // of the pairs between segments
};
ForwardPlan plan_forward(int64_t B, int64_t D, int64_t L, int64_t N, int64_t G) {
    ForwardPlan f;
    const int64_t waves4 = B * G * ((D / G + 15) / 16), waves16 = B * G * ((D / G + 3) / 4), waves64 = B * D;
    const int64_t tiles4 = (L + 31) / 32, tiles16 = (L + 127) / 128, tiles64 = (L + 511) / 512;
    const int64_t time4 = modelled_time(tiles4, waves4, 65, 39), time16 = modelled_time(tiles16, waves16, 65, 31);
    f.lanes = time16 <= modelled_time(tiles64, waves64, 75, 35) ? 16 : 64;
    if (f.lanes == 16 && time4 < time16) f.lanes = 4;
    // (4 or 16 lanes are only taken where the rows are short or many: not cut)
    f.cut = f.lanes == 4 ? Cut{1, (int32_t)tiles4} : f.lanes == 16 ? Cut{1, (int32_t)tiles16}
                         : cut_of(tiles64, waves64, waves64 < kCutBelow ? kCutWant : waves64);
    f.bytes = f.cut.segments > 1 ? (size_t)(f.cut.segments - 1) * B * D * N * sizeof(float2) : 0;
    return f;
}

template <typename T, int LPC, int WAVES>
int launch_forward(const char* who, const fmselective_scan_inputs& in, Cut cut, void* out, float* final_state, float* marks,
                   void* pairs, hipStream_t stream) {
    const Scan p = scan_of(in, WAVES * 64 / LPC, cut, pairs);
    const int64_t blocks = in.B * in.G * p.blocks_per_group * cut.segments;
    if (int rc = check_grid(who, blocks, 64 * WAVES)) return rc;
    static std::atomic<uint64_t> armed{0}, armed_ends{0};
    const size_t lds = fmselective::scan_forward_lds<LPC, WAVES>(p.N);
    const auto kernel = fmselective::selective_forward_kernel<T, LPC, WAVES, false>;
    if (lds > 64 * 1024)
        if (int rc = raise_lds_limit((const void*)kernel, armed, who)) return rc;
    if constexpr (LPC == 64) {
        if (cut.segments > 1) {
            const auto ends = fmselective::selective_forward_kernel<T, LPC, WAVES, true>;
            if (lds > 64 * 1024)
                if (int rc = raise_lds_limit((const void*)ends, armed_ends, who)) return rc;
            Scan q = p;  // every segment but the last
            q.segments = cut.segments - 1;
            ends<<<(unsigned)(blocks / cut.segments * q.segments), 64 * WAVES, lds, stream>>>(q, (T*)nullptr, nullptr, nullptr);
            if (int rc = launched("selective scan (ends of segments)")) return rc;
        }
    }
    kernel<<<(unsigned)blocks, 64 * WAVES, lds, stream>>>(p, (T*)out, final_state, marks);
    return launched("selective scan (forward)");
}

}  // namespace

namespace fmselective {
namespace host {
size_t forward_workspace_bytes(int64_t B, int64_t D, int64_t L, int64_t N, int64_t G) { return plan_forward(B, D, L, N, G).bytes; }
}  // namespace host
}  // namespace fmselective

extern "C" {

int fmselective_scan_forward(const fmselective_scan_inputs* in, void* out, float* final_state, float* marks, void* workspace,
                             size_t workspace_bytes, void* stream) {
    const char* who = "fmselective_scan_forward";
    if (int rc = check_scan(who, in, kScanFlags)) return rc;
    if (!out) return fail(FMSCAN_E_NULL, "%s: out must not be NULL", who);
    const int64_t states = in->B * in->D * in->N * 4, n_marks = (in->L + fmselective::kMark - 1) / fmselective::kMark;
    if (int rc = check_outputs(who, {{"out", out, in->B * in->D * in->L * esize_of(in->dtype)}, {"final_state", final_state, states},
                                     {"marks", marks, states * n_marks}}, input_ranges(*in)))
        return rc;
    ForwardPlan f = plan_forward(in->B, in->D, in->L, in->N, in->G);
    if (f.cut.segments > 1) {
        if (!workspace || workspace_bytes < f.bytes || ((uintptr_t)workspace & 7u)) {
            f.cut = {1, f.cut.segments * f.cut.seg_tiles};
        } else if (int rc = check_outputs(who, {{"workspace", workspace, (int64_t)f.bytes}}, input_ranges(*in))) {
            return rc;
        } else if (int rc = check_alias(who, {{"workspace", workspace, (int64_t)f.bytes}},
                                        {{"out", out, in->B * in->D * in->L * esize_of(in->dtype)}, {"final_state", final_state, states},
                                         {"marks", marks, states * n_marks}})) {
            return rc;
        }
    }
    int rc = 0;
    with_dtype(in->dtype, [&](auto tt) {
        using T = typename decltype(tt)::type;
        constexpr int W = fmselective::kScanWaves;
        const auto launch = f.lanes == 4 ? launch_forward<T, 4, W> : f.lanes == 16 ? launch_forward<T, 16, W> : launch_forward<T, 64, 8>;
        rc = launch(who, *in, f.cut, out, final_state, marks, workspace, (hipStream_t)stream);
    });
    return rc;
}

int fmselective_scan_step(const fmselective_scan_inputs* in, float* state_out, const void* slots, int64_t S, void* out,
                          void* stream) {
    const char* who = "fmselective_scan_step";
    if (!in) return fail(FMSCAN_E_NULL, "%s: the inputs must not be NULL", who);
    fmselective_scan_inputs one = *in;
    one.L = 1;
    if (int rc = check_scan(who, &one, kScanFlags | FMSELECTIVE_SLOTS_64)) return rc;
    if (int rc = check_pool(who, S, in->B, in->D * in->N, slots)) return rc;
    if (!in->initial_state || !state_out || !out)
        return fail(FMSCAN_E_NULL, "%s: initial_state (the pool), state_out and out must not be NULL", who);
    const int es = esize_of(in->dtype);
    const int64_t B = in->B, D = in->D, pool = S * D * in->N * 4;
    auto row = [&](const char* name, const void* p, const int64_t* s) { return Range{name, p, span({{B, s[0]}, {D, 1}}, es)}; };
    auto shared = [&](const char* name, const void* p, const int64_t* s) {
        return Range{name, p, span({{B, s[0]}, {in->G, s[1]}, {in->N, 1}}, es)};
    };
    const Range out_r = {"out", out, B * D * es}, new_r = {"state_out", state_out, pool}, old_r = {"the pool", in->initial_state, pool};
    if (int rc = check_alias(who, {out_r, new_r},
                             {row("tokens", in->tokens, in->tokens_strides), row("delta", in->delta, in->delta_strides),
                              row("gate", in->gate, in->gate_strides), shared("write", in->write, in->write_strides),
                              shared("read", in->read, in->read_strides), {"A", in->A, D * in->N * 4},
                              {"skip", in->skip, D * (in->flags & FMSELECTIVE_NARROW_SKIP ? es : 4)},
                              {"delta_bias", in->delta_bias, D * (in->flags & FMSELECTIVE_NARROW_BIAS ? es : 4)},
                              {"slots", slots, B * (in->flags & FMSELECTIVE_SLOTS_64 ? 8 : 4)}}))
        return rc;
    if (int rc = check_alias(who, {out_r}, {old_r})) return rc;
    if (state_out != in->initial_state)
        if (int rc = check_alias(who, {new_r}, {old_r})) return rc;
    fmselective::Step p = {};
    p.tokens = in->tokens; p.delta = in->delta; p.gate = in->gate; p.write = in->write; p.read = in->read;
    p.skip = in->skip; p.delta_bias = in->delta_bias; p.slots = slots; p.A = in->A; p.state = in->initial_state;
    p.state_out = state_out;
    p.tokens_b = in->tokens_strides[0]; p.delta_b = in->delta_strides[0]; p.gate_b = in->gate_strides[0];
    p.write_b = in->write_strides[0]; p.write_g = in->write_strides[1];
    p.read_b = in->read_strides[0]; p.read_g = in->read_strides[1];
    p.S = S;
    p.D = (int32_t)D; p.N = (int32_t)in->N; p.per_group = (int32_t)(D / in->G);
    const bool many = B * ((D + 63) / 64) >= kManyStepBlocks;
    p.tiles = (uint32_t)(many ? (D + 127) / 128 : (D + 63) / 64);
    p.flags = in->flags;
    if (int rc = check_grid(who, (__int128)B * p.tiles, 256)) return rc;
    const bool vec = in->N % 4 == 0 && aligned16(in->A) && aligned16(in->initial_state) && aligned16(state_out);
    with_dtype(in->dtype, [&](auto tt) {
        using T = typename decltype(tt)::type;
        with_bool(vec, [&](auto vt) {
            constexpr bool VEC = decltype(vt)::value;
            const auto kernel = many ? fmselective::selective_step_kernel<T, VEC, 2> : fmselective::selective_step_kernel<T, VEC, 1>;
            kernel<<<(unsigned)(B * p.tiles), 256, 0, (hipStream_t)stream>>>(p, (T*)out);
        });
    });
    return launched("selective scan (one token)");
}

}  // extern "C"
