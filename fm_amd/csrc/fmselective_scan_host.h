// Host side of the selective scan, shared by its translation units. Contract: include/fmselective.h.
#pragma once

#include "fmselective_host.h"
#include "fmselective_scan.h"

namespace fmselective {
namespace host {

constexpr unsigned kScanFlags = FMSELECTIVE_SOFTPLUS | FMSELECTIVE_NARROW_BIAS | FMSELECTIVE_NARROW_SKIP;
static_assert(kMark == FMSELECTIVE_MARK, "the marks' distance is part of the interface");

// Bytes of the pairs between a forward call's segments (fmselective_scan.hip)
size_t forward_workspace_bytes(int64_t B, int64_t D, int64_t L, int64_t N, int64_t G);

inline int check_states(const char* who, int64_t B, int64_t D, int64_t L, int64_t N, int64_t G, int dtype) {
    if (int rc = check_sizes(who, B, D, L, dtype)) return rc;
    if (N < 1 || N > FMSELECTIVE_MAX_STATES)
        return fail(FMSCAN_E_SHAPE, "%s: N must be in [1, %d] (got %lld)", who, FMSELECTIVE_MAX_STATES, (long long)N);
    if (G < 1 || G > D || D % G) return fail(FMSCAN_E_SHAPE, "%s: G must divide D (got %lld, %lld)", who, (long long)G, (long long)D);
    if ((__int128)B * D * N * ((L + kMark - 1) / kMark) > ((__int128)1 << 40))
        return fail(FMSCAN_E_SHAPE, "%s: B * D * N * ceil(L / %d) must fit 40 bits", who, kMark);
    return 0;
}

inline int check_scan(const char* who, const fmselective_scan_inputs* in, unsigned known) {
    if (!in) return fail(FMSCAN_E_NULL, "%s: the inputs must not be NULL", who);
    if (int rc = check_states(who, in->B, in->D, in->L, in->N, in->G, in->dtype)) return rc;
    if (int rc = check_flags(who, in->flags, known)) return rc;
    for (const int64_t* s : {in->tokens_strides, in->delta_strides, in->gate_strides})
        for (int i = 0; i < 2; ++i)
            if (int rc = check_stride(who, "tokens, delta and gate", s[i])) return rc;
    for (const int64_t* s : {in->write_strides, in->read_strides})
        for (int i = 0; i < 3; ++i)
            if (int rc = check_stride(who, "write and read", s[i])) return rc;
    if (!in->tokens || !in->delta || !in->A || !in->write || !in->read)
        return fail(FMSCAN_E_NULL, "%s: tokens, delta, A, write and read must not be NULL", who);
    return 0;
}

// How a row is cut: `segments` of `seg_tiles` tiles
struct Cut {
    int32_t segments, seg_tiles;
};
// Enough segments for `want` waves where `waves` are there without, at least two tiles each: with one the first
// launch would be as long as the row's.
inline Cut cut_of(int64_t tiles, int64_t waves, int64_t want) {
    int64_t n = (want + waves - 1) / waves;
    if (n > tiles / 2) n = tiles / 2;
    if (n < 1) n = 1;
    Cut c;
    c.seg_tiles = (int32_t)((tiles + n - 1) / n);
    c.segments = (int32_t)((tiles + c.seg_tiles - 1) / c.seg_tiles);
    return c;
}

inline Scan scan_of(const fmselective_scan_inputs& in, int channels_per_block, Cut cut, void* pairs) {
    Scan p = {};
    p.tokens = in.tokens; p.delta = in.delta; p.gate = in.gate; p.write = in.write; p.read = in.read;
    p.skip = in.skip; p.delta_bias = in.delta_bias; p.A = in.A; p.initial = in.initial_state; p.lengths = in.lengths;
    p.tokens_b = in.tokens_strides[0]; p.tokens_d = in.tokens_strides[1];
    p.delta_b = in.delta_strides[0]; p.delta_d = in.delta_strides[1];
    p.gate_b = in.gate_strides[0]; p.gate_d = in.gate_strides[1];
    p.write_b = in.write_strides[0]; p.write_g = in.write_strides[1]; p.write_n = in.write_strides[2];
    p.read_b = in.read_strides[0]; p.read_g = in.read_strides[1]; p.read_n = in.read_strides[2];
    p.L = in.L;
    p.D = (int32_t)in.D; p.N = (int32_t)in.N; p.G = (int32_t)in.G;
    p.per_group = (int32_t)(in.D / in.G);
    p.blocks_per_group = (p.per_group + channels_per_block - 1) / channels_per_block;
    p.marks = (int32_t)((in.L + kMark - 1) / kMark);
    p.flags = in.flags;
    p.segments = cut.segments;
    p.seg_tiles = cut.seg_tiles;
    p.rows = in.B * in.D;
    p.pairs = (float2*)pairs;
    return p;
}

// the inputs of a call on sequences, as ranges of memory
struct InputRanges {
    Range r[10];
};
inline InputRanges input_ranges(const fmselective_scan_inputs& in) {
    const int es = esize_of(in.dtype);
    auto seq = [&](const char* name, const void* p, const int64_t* s) { return Range{name, p, extent(in.B, in.D, in.L, s[0], s[1], es)}; };
    auto shared = [&](const char* name, const void* p, const int64_t* s) {
        return Range{name, p, span({{in.B, s[0]}, {in.G, s[1]}, {in.N, s[2]}, {in.L, 1}}, es)};
    };
    return {{seq("tokens", in.tokens, in.tokens_strides), seq("delta", in.delta, in.delta_strides),
             seq("gate", in.gate, in.gate_strides), shared("write", in.write, in.write_strides),
             shared("read", in.read, in.read_strides), {"A", in.A, in.D * in.N * 4},
             {"skip", in.skip, in.D * (in.flags & FMSELECTIVE_NARROW_SKIP ? es : 4)},
             {"delta_bias", in.delta_bias, in.D * (in.flags & FMSELECTIVE_NARROW_BIAS ? es : 4)},
             {"initial_state", in.initial_state, in.B * in.D * in.N * 4}, {"lengths", in.lengths, in.B * 4}}};
}
inline int check_outputs(const char* who, std::initializer_list<Range> outs, const InputRanges& ins) {
    if (int rc = check_alias(who, outs, {})) return rc;
    for (const Range& o : outs)
        for (const Range& i : ins.r)
            if (overlap(o, i)) return fail(FMSCAN_E_ALIAS, "%s: %s overlaps %s", who, o.name, i.name);
    return 0;
}

}  // namespace host
}  // namespace fmselective
