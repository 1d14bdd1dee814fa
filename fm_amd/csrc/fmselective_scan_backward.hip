// The selective scan's backward call. Contract: include/fmselective.h.
#include "fmselective_scan_host.h"

using namespace fmselective::host;
using fmselective::Scan;
using fmselective::ScanGrads;

namespace {

constexpr int kBackWaves = fmselective::kScanWaves;

// The rows are cut where they leave less than a wave a SIMD, for two. Measured (bf16, N = 16, us): (1, 2048, 2048), 512
// waves, 144 with one wave a SIMD, 102 with two, 104 with four; (1, 1024, 8192) 285, 193, 194; at (1, 4096, 2048),
// 1024 waves, the cut gains nothing (203, 202).
constexpr int64_t kBackCutBelow = 1024, kBackCutWant = 2048;
struct BackPlan {
    Cut cut;
    int64_t blocks, shared, states, rows, pairs;  // blocks; floats of the partial sums and of the pairs
    size_t bytes() const { return (size_t)(shared + pairs + states + 2 * rows) * sizeof(float); }
};
BackPlan plan_backward(int64_t B, int64_t D, int64_t L, int64_t N, int64_t G) {
    const int64_t per_group = D / G, marks = (L + fmselective::kMark - 1) / fmselective::kMark;
    BackPlan b;
    b.blocks = B * G * ((per_group + 4 * kBackWaves - 1) / (4 * kBackWaves));
    const int64_t waves = b.blocks * kBackWaves;
    b.cut = cut_of(marks, waves, waves < kBackCutBelow ? kBackCutWant : waves);
    b.shared = b.blocks * N * marks * 256;
    b.pairs = b.cut.segments > 1 ? 2 * b.cut.segments * B * D * N : 0;
    b.states = b.cut.segments * B * D * N;
    b.rows = b.cut.segments * B * D;
    return b;
}

template <typename T, bool ENDS>
int launch_backward(const char* who, const Scan& p, const ScanGrads& g, int64_t blocks, hipStream_t stream) {
    static std::atomic<uint64_t> armed{0};
    const size_t lds = fmselective::scan_backward_lds<kBackWaves>(p.N);
    const auto kernel = fmselective::selective_backward_kernel<T, kBackWaves, ENDS>;
    if (lds > 64 * 1024)
        if (int rc = raise_lds_limit((const void*)kernel, armed, who)) return rc;
    kernel<<<(unsigned)blocks, 64 * kBackWaves, lds, stream>>>(p, g);
    return launched("selective scan (backward)");
}

}  // namespace

extern "C" {

size_t fmselective_scan_workspace_bytes(int64_t B, int64_t D, int64_t L, int64_t N, int64_t G, int dtype, int backward) {
    if (check_states("fmselective_scan_workspace_bytes", B, D, L, N, G, dtype)) return 0;
    return backward ? plan_backward(B, D, L, N, G).bytes() : forward_workspace_bytes(B, D, L, N, G);
}

int fmselective_scan_backward(const fmselective_scan_inputs* in, const fmselective_scan_grads* grads, void* workspace,
                              size_t workspace_bytes, void* stream) {
    const char* who = "fmselective_scan_backward";
    if (int rc = check_scan(who, in, kScanFlags)) return rc;
    if (!grads) return fail(FMSCAN_E_NULL, "%s: the gradients must not be NULL", who);
    const fmselective_scan_grads& o = *grads;
    if (!o.out_grad || !o.marks || !o.tokens || !o.delta || !o.write || !o.read || !o.A || (!o.gate != !in->gate) ||
        (!o.skip != !in->skip) || (!o.delta_bias != !in->delta_bias))
        return fail(FMSCAN_E_NULL, "%s: out_grad, marks and every input's gradient must be there, and those of gate, skip and "
                    "delta_bias where they are", who);
    for (int i = 0; i < 2; ++i)
        if (int rc = check_stride(who, "out_grad", o.out_grad_strides[i])) return rc;
    const BackPlan b = plan_backward(in->B, in->D, in->L, in->N, in->G);
    const size_t need = b.bytes();
    if (!workspace || workspace_bytes < need || !aligned16(workspace))
        return fail(FMSCAN_E_WORKSPACE, "%s: a 16-byte aligned workspace of %zu bytes is needed (got %zu)", who, need,
                    workspace ? workspace_bytes : (size_t)0);
    const int es = esize_of(in->dtype);
    const int64_t seq = in->B * in->D * in->L * es, shared = in->B * in->G * in->N * in->L * es, states = in->B * in->D * in->N * 4;
    const int64_t marks = states * ((in->L + fmselective::kMark - 1) / fmselective::kMark);
    const Range outs[] = {{"tokens' gradient", o.tokens, seq}, {"delta's gradient", o.delta, seq}, {"gate's gradient", o.gate, seq},
                          {"write's gradient", o.write, shared}, {"read's gradient", o.read, shared},
                          {"A's gradient", o.A, in->D * in->N * 4}, {"the initial state's gradient", o.initial_state, states},
                          {"skip's gradient", o.skip, in->D * (in->flags & FMSELECTIVE_NARROW_SKIP ? es : 4)},
                          {"delta_bias's gradient", o.delta_bias, in->D * (in->flags & FMSELECTIVE_NARROW_BIAS ? es : 4)},
                          {"workspace", workspace, (int64_t)need}};
    const Range more[] = {{"out_grad", o.out_grad, extent(in->B, in->D, in->L, o.out_grad_strides[0], o.out_grad_strides[1], es)},
                          {"final_state_grad", o.final_state_grad, states}, {"marks", o.marks, marks}};
    const InputRanges ins = input_ranges(*in);
    for (const Range& r : outs) {
        if (int rc = check_outputs(who, {r}, ins)) return rc;
        if (int rc = check_alias(who, {r}, {more[0], more[1], more[2]})) return rc;
        for (const Range& q : outs)
            if (&q != &r && overlap(q, r)) return fail(FMSCAN_E_ALIAS, "%s: %s overlaps %s", who, r.name, q.name);
    }
    float* const pairs = (float*)workspace + b.shared;
    const Scan p = scan_of(*in, 4 * kBackWaves, b.cut, pairs);
    const int64_t lines = in->B * in->G * in->N, items = lines * p.marks, blocks = b.blocks * b.cut.segments;
    if (int rc = check_grid(who, blocks, 64 * kBackWaves)) return rc;
    int per = 1;  // waves that share a sum of the last launch: at least four terms each
    while (per < fmselective::kSumWaves && p.blocks_per_group >= 8 * per) per *= 2;
    // (its threads: 64 a wave and a sum, and 16 a column of the parameters' gradients, three sections of whole blocks)
    if (int rc = check_grid(who, ((__int128)items * per + 64) * 64 + ((__int128)in->D * in->N + 2 * in->D + 256) * 16, 1)) return rc;
    float* part = (float*)workspace;
    ScanGrads g = {};
    g.out_grad = o.out_grad;
    g.out_b = o.out_grad_strides[0];
    g.out_d = o.out_grad_strides[1];
    g.final_grad = o.final_state_grad;
    g.marks = o.marks;
    g.tokens = o.tokens;
    g.delta = o.delta;
    g.gate = o.gate;
    g.initial = o.initial_state;
    g.shared_part = part;
    g.A_part = pairs + b.pairs;
    g.skip_part = o.skip ? g.A_part + b.states : nullptr;
    g.bias_part = o.delta_bias ? g.A_part + b.states + b.rows : nullptr;
    int rc = 0;
    with_dtype(in->dtype, [&](auto tt) {
        using T = typename decltype(tt)::type;
        const hipStream_t st = (hipStream_t)stream;
        if (b.cut.segments > 1 && (rc = launch_backward<T, true>(who, p, g, blocks, st))) return;
        if ((rc = launch_backward<T, false>(who, p, g, blocks, st))) return;
        fmselective::ColumnSums columns;
        const uint32_t column_blocks = column_sections(
            {{g.A_part, o.A, in->B * b.cut.segments, in->D * in->N, 0, 0},
             {g.skip_part, o.skip, in->B * b.cut.segments, in->D, (in->flags & FMSELECTIVE_NARROW_SKIP) != 0, 0},
             {g.bias_part, o.delta_bias, in->B * b.cut.segments, in->D, (in->flags & FMSELECTIVE_NARROW_BIAS) != 0, 0}}, &columns);
        constexpr int W = fmselective::kSumWaves;
        fmselective::selective_sums_kernel<T><<<(unsigned)(column_blocks + (items * per + W - 1) / W), 64 * W, 0, st>>>(
            columns, column_blocks, part, (T*)o.write, (T*)o.read, in->lengths, in->L, items, p.N, p.G, p.marks,
            p.blocks_per_group, per);
        rc = launched("selective scan (sums of gradients)");
    });
    return rc;
}

}  // extern "C"
