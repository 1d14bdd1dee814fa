// The short convolution's entry points: forward, backward, one token. Contract: include/fmselective.h.
#include "fmselective_host.h"
#include "fmselective_conv.h"

using namespace fmselective::host;
using fmselective::ConvBack;
using fmselective::ConvRows;

namespace {

constexpr unsigned kConvFlags = FMSELECTIVE_SILU | FMSELECTIVE_NARROW_WEIGHT | FMSELECTIVE_NARROW_BIAS;

template <typename F>
void with_taps(int64_t W, F&& f) {
    if (W == 2) f(IntTag<2>{});
    else if (W == 3) f(IntTag<3>{});
    else f(IntTag<4>{});
}

int check_taps(const char* who, int64_t W) {
    return W < 2 || W > 4 ? fail(FMSCAN_E_SHAPE, "%s: W must be 2, 3 or 4 (got %lld)", who, (long long)W) : 0;
}

// How backward's rows are dealt to waves: rows of at most 64 chunks share them, long ones are cut where rows alone leave
// compute units without enough waves to hide the memory's latency, in pieces of at least two tiles. Measured (bf16, us):
// long rows for 4096, 8192, 16384 waves: (1, 4096, 2048) 14, 22, 21; (1, 4096, 4096) 24, 27, 42; (1, 4096, 16384)
// 77, 75, 83. Short ones for 4096, 8192, 16384: (256, 4096, 65) 158, 124, 128; (1024, 4096, 33) 425, 350, 322;
// (64, 4096, 256) 75, 76, 78.
constexpr int64_t kConvBackWaves = 4096, kConvShortWaves = 8192;
ConvBack plan_backward(int64_t B, int64_t D, int64_t L, int dtype) {
    ConvBack g = {};
    const int E = dtype == FMSCAN_DTYPE_F32 ? 4 : 8;
    const int64_t chunks = (L + E - 1) / E;
    g.L = L;
    g.rows = (int32_t)(B * D);
    g.B = (int32_t)B;
    g.D = (int32_t)D;
    g.chunks = (int32_t)chunks;
    if (chunks <= 64) {
        g.rows_per_wave = 64 / g.chunks;
        g.row_lanes_magic = (65536 + g.chunks - 1) / g.chunks;
        g.groups = (int32_t)((D + g.rows_per_wave - 1) / g.rows_per_wave);
        int64_t parts = (kConvShortWaves + g.groups - 1) / g.groups;
        if (parts > B) parts = B;
        g.each = (int32_t)((B + parts - 1) / parts);
        g.parts = (int32_t)((B + g.each - 1) / g.each);
        return g;
    }
    g.tiles = (int32_t)((chunks + 63) / 64);
    int64_t segments = (kConvBackWaves + g.rows - 1) / g.rows;
    if (segments > g.tiles / 2) segments = g.tiles / 2;
    if (segments < 1) segments = 1;
    g.seg_tiles = (int32_t)((g.tiles + segments - 1) / segments);
    g.segments = (g.tiles + g.seg_tiles - 1) / g.seg_tiles;
    g.parts = (int32_t)(B * g.segments);
    return g;
}

}  // namespace

extern "C" {

int fmselective_conv_forward(const void* inputs, int64_t batch_stride, int64_t channel_stride, const void* weight,
                             const void* bias, const void* initial_state, const int32_t* lengths, void* out,
                             void* final_state, int64_t B, int64_t D, int64_t L, int64_t W, int dtype,
                             unsigned flags, void* stream) {
    const char* who = "fmselective_conv_forward";
    if (int rc = check_sizes(who, B, D, L, dtype)) return rc;
    if (int rc = check_taps(who, W)) return rc;
    if (int rc = check_flags(who, flags, kConvFlags)) return rc;
    if (int rc = check_stride(who, "inputs", batch_stride)) return rc;
    if (int rc = check_stride(who, "inputs", channel_stride)) return rc;
    if (!inputs || !weight || !out) return fail(FMSCAN_E_NULL, "%s: inputs, weight and out must not be NULL", who);
    const int es = esize_of(dtype), weight_es = flags & FMSELECTIVE_NARROW_WEIGHT ? es : 4;
    const int bias_es = flags & FMSELECTIVE_NARROW_BIAS ? es : 4;
    if (int rc = check_alias(who, {{"out", out, B * D * L * es}, {"final_state", final_state, B * D * (W - 1) * es}},
                             {{"inputs", inputs, extent(B, D, L, batch_stride, channel_stride, es)},
                              {"weight", weight, D * W * weight_es}, {"bias", bias, D * bias_es},
                              {"initial_state", initial_state, B * D * (W - 1) * es}, {"lengths", lengths, B * 4}}))
        return rc;
    ConvRows g = {batch_stride, channel_stride, L, (int32_t)(B * D), (int32_t)D, 1, 1, 0, 0};
    const int E = 16 / es;
    g.chunks = (uint32_t)((L + E - 1) / E);
    // chunks a lane (1: the kernel for short rows). Measured with 1, 2, 4 (bf16, us): (32, 4096, 512) 57, 75, -;
    // (16, 4096, 1024) -, 48, 69; (8, 4096, 2048) -, 53, 44.
    const int each = g.chunks <= 64 ? 1 : g.chunks <= 128 ? 2 : 4;
    int64_t blocks;
    if (each == 1) {
        g.rows_per_block = 256 / g.chunks;
        g.magic = (65536 + g.chunks - 1) / g.chunks;
        blocks = ((int64_t)g.rows + g.rows_per_block - 1) / g.rows_per_block;
    } else {
        g.units = (g.chunks + 64 * each - 1) / (64 * each);
        blocks = ((int64_t)g.rows * g.units + 3) / 4;
    }
    if (int rc = check_grid(who, blocks, 256)) return rc;
    with_dtype(dtype, [&](auto tt) {
        using T = typename decltype(tt)::type;
        with_taps(W, [&](auto wt) {
            constexpr int TAPS = decltype(wt)::value;
            const auto kernel = each == 1 ? fmselective::conv_forward_short_kernel<T, TAPS>
                                : each == 2 ? fmselective::conv_forward_kernel<T, TAPS, 2> : fmselective::conv_forward_kernel<T, TAPS, 4>;
            kernel<<<(unsigned)blocks, 256, 0, (hipStream_t)stream>>>((const T*)inputs, weight, bias, (const T*)initial_state,
                                                                      lengths, (T*)out, (T*)final_state, g, flags);
        });
    });
    return launched("convolution (forward)");
}

size_t fmselective_conv_workspace_bytes(int64_t B, int64_t D, int64_t L, int64_t W, int dtype) {
    if (check_sizes("fmselective_conv_workspace_bytes", B, D, L, dtype) || check_taps("fmselective_conv_workspace_bytes", W))
        return 0;
    const ConvBack g = plan_backward(B, D, L, dtype);
    return (size_t)g.parts * D * (W + 1) * sizeof(float);
}

int fmselective_conv_backward(const void* inputs, int64_t batch_stride, int64_t channel_stride, const void* out_grad,
                              int64_t grad_batch_stride, int64_t grad_channel_stride, const void* weight,
                              const void* bias, const void* initial_state, const void* final_state_grad,
                              const int32_t* lengths, void* inputs_grad, void* weight_grad, void* bias_grad,
                              void* initial_state_grad, int64_t B, int64_t D, int64_t L, int64_t W, int dtype,
                              unsigned flags, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "fmselective_conv_backward";
    if (int rc = check_sizes(who, B, D, L, dtype)) return rc;
    if (int rc = check_taps(who, W)) return rc;
    if (int rc = check_flags(who, flags, kConvFlags)) return rc;
    for (int64_t s : {batch_stride, channel_stride, grad_batch_stride, grad_channel_stride})
        if (int rc = check_stride(who, "inputs and out_grad", s)) return rc;
    if (!inputs || !out_grad || !weight || !inputs_grad || !weight_grad)
        return fail(FMSCAN_E_NULL, "%s: inputs, out_grad, weight, inputs_grad and weight_grad must not be NULL", who);
    const size_t need = fmselective_conv_workspace_bytes(B, D, L, W, dtype);
    if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 3u))
        return fail(FMSCAN_E_WORKSPACE, "%s: a 4-byte aligned workspace of %zu bytes is needed (got %zu)", who, need,
                    workspace ? workspace_bytes : (size_t)0);
    const int es = esize_of(dtype), weight_es = flags & FMSELECTIVE_NARROW_WEIGHT ? es : 4;
    const int bias_es = flags & FMSELECTIVE_NARROW_BIAS ? es : 4;
    const int64_t held = B * D * (W - 1) * es;
    if (int rc = check_alias(who,
                             {{"inputs_grad", inputs_grad, B * D * L * es}, {"weight_grad", weight_grad, D * W * weight_es},
                              {"bias_grad", bias_grad, D * bias_es}, {"initial_state_grad", initial_state_grad, held},
                              {"workspace", workspace, (int64_t)need}},
                             {{"inputs", inputs, extent(B, D, L, batch_stride, channel_stride, es)},
                              {"out_grad", out_grad, extent(B, D, L, grad_batch_stride, grad_channel_stride, es)},
                              {"weight", weight, D * W * weight_es}, {"bias", bias, D * bias_es},
                              {"initial_state", initial_state, held}, {"final_state_grad", final_state_grad, held},
                              {"lengths", lengths, B * 4}}))
        return rc;
    ConvBack g = plan_backward(B, D, L, dtype);
    g.batch_stride = batch_stride;
    g.channel_stride = channel_stride;
    g.grad_batch_stride = grad_batch_stride;
    g.grad_channel_stride = grad_channel_stride;
    const bool is_short = g.chunks <= 64;
    const int64_t waves = is_short ? (int64_t)g.groups * g.parts : (int64_t)g.rows * g.segments, blocks = (waves + 3) / 4;
    if (int rc = check_grid(who, blocks, 256)) return rc;
    if (int rc = check_grid(who, (__int128)D * (W + 1) + 128, 16)) return rc;  // the sums of the parameters' gradients
    float* weight_part = (float*)workspace;
    float* bias_part = weight_part + g.parts * D * W;
    with_dtype(dtype, [&](auto tt) {
        using T = typename decltype(tt)::type;
        with_taps(W, [&](auto wt) {
            constexpr int TAPS = decltype(wt)::value;
            const auto kernel = is_short ? fmselective::conv_backward_short_kernel<T, TAPS> : fmselective::conv_backward_kernel<T, TAPS>;
            kernel<<<(unsigned)blocks, 256, 0, (hipStream_t)stream>>>(
                (const T*)inputs, (const T*)out_grad, weight, bias, (const T*)initial_state, (const T*)final_state_grad,
                lengths, (T*)inputs_grad, (T*)initial_state_grad, weight_part, bias_part, g, flags);
        });
    });
    if (int rc = launched("convolution (backward)")) return rc;
    const int64_t n = g.parts;
    launch_column_sums(dtype,
                       {{weight_part, weight_grad, n, D * W, (flags & FMSELECTIVE_NARROW_WEIGHT) != 0, 0},
                        {bias_part, bias_grad, n, D, (flags & FMSELECTIVE_NARROW_BIAS) != 0, 0}},
                       (hipStream_t)stream);
    return launched("convolution (sums of the parameters' gradients)");
}

int fmselective_conv_step(const void* inputs, int64_t batch_stride, const void* state, void* state_out,
                          const void* weight, const void* bias, const void* slots, void* out, int64_t B, int64_t D,
                          int64_t W, int64_t S, int dtype, unsigned flags, void* stream) {
    const char* who = "fmselective_conv_step";
    if (int rc = check_sizes(who, B, D, 1, dtype)) return rc;
    if (int rc = check_taps(who, W)) return rc;
    if (int rc = check_flags(who, flags, kConvFlags | FMSELECTIVE_SLOTS_64)) return rc;
    if (int rc = check_stride(who, "inputs", batch_stride)) return rc;
    if (int rc = check_pool(who, S, B, D * (W - 1), slots)) return rc;
    if (!inputs || !state || !state_out || !weight || !out)
        return fail(FMSCAN_E_NULL, "%s: inputs, state, state_out, weight and out must not be NULL", who);
    const int es = esize_of(dtype), weight_es = flags & FMSELECTIVE_NARROW_WEIGHT ? es : 4;
    const int bias_es = flags & FMSELECTIVE_NARROW_BIAS ? es : 4;
    const int64_t pool = S * D * (W - 1) * es;
    const Range out_r = {"out", out, B * D * es}, new_r = {"state_out", state_out, pool};
    const Range in_r = {"inputs", inputs, extent(B, 1, D, batch_stride, 0, es)}, w_r = {"weight", weight, D * W * weight_es},
                b_r = {"bias", bias, D * bias_es}, s_r = {"slots", slots, B * (flags & FMSELECTIVE_SLOTS_64 ? 8 : 4)},
                old_r = {"state", state, pool};
    if (int rc = check_alias(who, {out_r, new_r}, {in_r, w_r, b_r, s_r})) return rc;
    if (int rc = check_alias(who, {out_r}, {old_r})) return rc;
    if (state_out != state)
        if (int rc = check_alias(who, {new_r}, {old_r})) return rc;
    const uint32_t tiles = (uint32_t)((D + 1023) / 1024);
    if (int rc = check_grid(who, (__int128)B * tiles, 256)) return rc;
    with_dtype(dtype, [&](auto tt) {
        using T = typename decltype(tt)::type;
        with_taps(W, [&](auto wt) {
            fmselective::conv_step_kernel<T, decltype(wt)::value><<<(unsigned)(B * tiles), 256, 0, (hipStream_t)stream>>>(
                (const T*)inputs, batch_stride, (const T*)state, (T*)state_out, weight, bias, slots, (T*)out, (int32_t)D,
                tiles, S, flags);
        });
    });
    return launched("convolution (one token)");
}

}  // extern "C"
