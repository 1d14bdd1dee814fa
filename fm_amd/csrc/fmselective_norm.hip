// The norm's entry points: forward (also in 8 bits) and backward. Contract: include/fmselective.h.
#include "fmselective_host.h"
#include "fmselective_norm.h"

using namespace fmselective::host;

namespace {

constexpr unsigned kNormFlags = FMSELECTIVE_NARROW_WEIGHT;

int check_rows(const char* who, int64_t rows, int64_t D, int dtype) {
    if (rows < 1 || D < 1 || rows > INT32_MAX)
        return fail(FMSCAN_E_SHAPE, "%s: rows and D must be >= 1 and rows fit 31 bits (got %lld, %lld)", who, (long long)rows,
                    (long long)D);
    if (dtype != FMSCAN_DTYPE_F32 && dtype != FMSCAN_DTYPE_F16 && dtype != FMSCAN_DTYPE_BF16)
        return fail(FMSCAN_E_DTYPE, "%s: dtype %d is not float32 (0), float16 (1) or bfloat16 (2)", who, dtype);
    if (D > FMSELECTIVE_MAX_NORM)
        return fail(FMSCAN_E_SHAPE, "%s: D must be at most %d (got %lld)", who, FMSELECTIVE_MAX_NORM, (long long)D);
    return 0;
}

// Threads a row and chunks of 16 bytes a thread: a wave for the shortest rows, a block for the others; backward, whose
// barrier comes once a row instead of once a block, keeps to waves a little longer. Measured (bf16, us, forward / backward):
// (32768, 512) a wave 25 / 26, 256 threads 35 / 78; (32768, 1024) a wave 46 / 46, 256 threads 44 / 84; (16384, 1600) a wave
// 40 / 49, 256 threads 37 / 72; (8192, 4096) a wave 50 / 68, 256 threads 46 / 51, 1024 threads 48 / 61; (4096, 8192) 256
// threads 49 / 50, 1024 threads 46 / 55; (2048, 16384) 256 threads 50 / 76, 1024 threads 48 / 74. (Backward beyond 8192
// elements spills: 1024 threads leave a thread 128 registers, and 73 to 75 of those in 16 bits, 180 in float32, go to scratch.)
template <typename T, bool BACKWARD, typename F>
void with_row_shape(int64_t D, F&& f) {
    constexpr int E = fmselective::Elem<T>::E;
    const int64_t chunks = (D + E - 1) / E;
    if (chunks <= 64) f(IntTag<64>{}, IntTag<1>{});
    else if (chunks <= 128) f(IntTag<64>{}, IntTag<2>{});
    else if (chunks <= 256) f(IntTag<BACKWARD ? 64 : 256>{}, IntTag<BACKWARD ? 4 : 1>{});
    else if (chunks <= 512) f(IntTag<256>{}, IntTag<2>{});
    else if (chunks <= 1024) f(IntTag<BACKWARD ? 256 : 1024>{}, IntTag<BACKWARD ? 4 : 1>{});
    else if (chunks <= 2048) f(IntTag<1024>{}, IntTag<2>{});
    else if constexpr (FMSELECTIVE_MAX_NORM / E > 2048) f(IntTag<1024>{}, IntTag<4>{});  // (float32 alone)
}

// Blocks of the backward call, each with its part of the weight's gradient: all the rows' where there are few, else as
// many as keep the memory busy and leave the parts small beside the streams. Measured with 512, 768, 1024 blocks (bf16,
// us, the parts' sum included): (8192, 4096) 54, 56, 64; (16384, 1024) 30, 30, 36; (9208, 1297) 61, 51, 47.
constexpr int64_t kNormBlocks = 512;
int64_t backward_blocks(int64_t rows, int rows_per_block) {
    const int64_t n = (rows + rows_per_block - 1) / rows_per_block;
    return n > kNormBlocks ? kNormBlocks : n;
}

}  // namespace

extern "C" {

int fmselective_norm_forward(const void* inputs, const void* residual, const void* weight, void* residual_out, void* out,
                             float* scales, float* inv_rms, int64_t rows, int64_t D, int dtype, unsigned flags, float eps,
                             void* stream) {
    const char* who = "fmselective_norm_forward";
    if (int rc = check_rows(who, rows, D, dtype)) return rc;
    if (int rc = check_flags(who, flags, kNormFlags)) return rc;
    if (!(eps >= 0.0f)) return fail(FMSCAN_E_SHAPE, "%s: eps must be >= 0", who);
    if (!inputs || !weight || !out || (residual && !residual_out))
        return fail(FMSCAN_E_NULL, "%s: inputs, weight, out, and residual_out with a residual, must not be NULL", who);
    const int es = esize_of(dtype);
    if (int rc = check_alias(who,
                             {{"out", out, rows * D * (scales ? 1 : es)}, {"residual_out", residual ? residual_out : nullptr, rows * D * es},
                              {"scales", scales, rows * 4}, {"inv_rms", inv_rms, rows * 4}},
                             {{"inputs", inputs, rows * D * es}, {"residual", residual, rows * D * es},
                              {"weight", weight, D * (flags & FMSELECTIVE_NARROW_WEIGHT ? es : 4)}}))
        return rc;
    int threads = 0;  // a row
    with_dtype(dtype, [&](auto tt) {
        with_row_shape<typename decltype(tt)::type, false>(D, [&](auto pt, auto) { threads = decltype(pt)::value; });
    });
    if (int rc = check_grid(who, (__int128)rows + 3, threads)) return rc;
    with_dtype(dtype, [&](auto tt) {
        using T = typename decltype(tt)::type;
        with_row_shape<T, false>(D, [&](auto pt, auto ct) {
            constexpr int TPR = decltype(pt)::value, CH = decltype(ct)::value, RPB = TPR == 64 ? 4 : 1;
            with_bool(scales != nullptr, [&](auto qt) {
                fmselective::norm_forward_kernel<T, TPR, CH, decltype(qt)::value>
                    <<<(unsigned)((rows + RPB - 1) / RPB), TPR == 64 ? 256 : TPR, 0, (hipStream_t)stream>>>(
                        (const T*)inputs, (const T*)residual, weight, (T*)residual_out, out, scales, inv_rms, rows, (int32_t)D,
                        eps, flags);
            });
        });
    });
    return launched("norm (forward)");
}

size_t fmselective_norm_workspace_bytes(int64_t rows, int64_t D, int dtype) {
    if (check_rows("fmselective_norm_workspace_bytes", rows, D, dtype)) return 0;
    return (size_t)backward_blocks(rows, 1) * D * sizeof(float);
}

int fmselective_norm_backward(const void* out_grad, const void* residual_grad, const void* stream_in, const void* weight,
                              const float* inv_rms, void* grad, void* weight_grad, int64_t rows, int64_t D, int dtype,
                              unsigned flags, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "fmselective_norm_backward";
    if (int rc = check_rows(who, rows, D, dtype)) return rc;
    if (int rc = check_flags(who, flags, kNormFlags)) return rc;
    if (!out_grad || !stream_in || !weight || !inv_rms || !grad || !weight_grad)
        return fail(FMSCAN_E_NULL, "%s: out_grad, the stream, weight, inv_rms and the gradients must not be NULL", who);
    const size_t need = fmselective_norm_workspace_bytes(rows, D, dtype);
    if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 3u))
        return fail(FMSCAN_E_WORKSPACE, "%s: a 4-byte aligned workspace of %zu bytes is needed (got %zu)", who, need,
                    workspace ? workspace_bytes : (size_t)0);
    const int es = esize_of(dtype), ws = flags & FMSELECTIVE_NARROW_WEIGHT ? es : 4;
    if (int rc = check_alias(who,
                             {{"grad", grad, rows * D * es}, {"weight_grad", weight_grad, D * ws},
                              {"workspace", workspace, (int64_t)need}},
                             {{"out_grad", out_grad, rows * D * es}, {"residual_grad", residual_grad, rows * D * es},
                              {"the stream", stream_in, rows * D * es}, {"weight", weight, D * ws}, {"inv_rms", inv_rms, rows * 4}}))
        return rc;
    int64_t blocks = 0;
    with_dtype(dtype, [&](auto tt) {
        using T = typename decltype(tt)::type;
        with_row_shape<T, true>(D, [&](auto pt, auto ct) {
            constexpr int TPR = decltype(pt)::value, CH = decltype(ct)::value, RPB = TPR == 64 ? 4 : 1;
            blocks = backward_blocks(rows, RPB);
            fmselective::norm_backward_kernel<T, TPR, CH><<<(unsigned)blocks, TPR == 64 ? 256 : TPR, 0, (hipStream_t)stream>>>(
                (const T*)out_grad, (const T*)residual_grad, (const T*)stream_in, weight, inv_rms, (T*)grad, (float*)workspace,
                rows, (int32_t)D, flags);
        });
    });
    if (int rc = launched("norm (backward)")) return rc;
    launch_column_sums(dtype, {{(const float*)workspace, weight_grad, blocks, D, (flags & FMSELECTIVE_NARROW_WEIGHT) != 0, 0}},
                       (hipStream_t)stream);
    return launched("norm (the weight's gradient)");
}

}  // extern "C"
