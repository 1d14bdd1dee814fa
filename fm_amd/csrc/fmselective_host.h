// Host-side pieces shared by the selective layer's translation units: checks of arguments and the launch of the
// column sums. Contract of the calls: include/fmselective.h.
#pragma once

#include "../../include/fmselective.h"
#include "fmscan_host.h"
#include "fmselective_device.h"

#include <utility>

namespace fmselective {
namespace host {

using namespace fmscan::host;

inline int esize_of(int dtype) { return dtype == FMSCAN_DTYPE_F32 ? 4 : 2; }

// B, D, L of a call on sequences: a row index fits 31 bits, so does the number of blocks
inline int check_sizes(const char* who, int64_t B, int64_t D, int64_t L, int dtype) {
    if (B < 1 || D < 1 || L < 1)
        return fail(FMSCAN_E_SHAPE, "%s: B, D and L must be >= 1 (got %lld, %lld, %lld)", who, (long long)B,
                    (long long)D, (long long)L);
    if (dtype != FMSCAN_DTYPE_F32 && dtype != FMSCAN_DTYPE_F16 && dtype != FMSCAN_DTYPE_BF16)
        return fail(FMSCAN_E_DTYPE, "%s: dtype %d is not float32 (0), float16 (1) or bfloat16 (2)", who, dtype);
    // (a kernel's last block may reach beyond D and L: their 32-bit indexes have room for that)
    if (D > (1 << 30) || (__int128)B * D > (__int128)INT32_MAX || L > (1 << 30) || (__int128)B * D * L > ((__int128)1 << 40))
        return fail(FMSCAN_E_SHAPE, "%s: D and L must be at most 2^30, B * D below 2^31 and B * D * L at most 2^40", who);
    return 0;
}
inline int check_flags(const char* who, unsigned flags, unsigned known) {
    return flags & ~known ? fail(FMSCAN_E_FLAGS, "%s: unknown flag bits 0x%x", who, flags & ~known) : 0;
}
inline int check_stride(const char* who, const char* name, int64_t s) {
    return s < 0 || s > ((int64_t)1 << 44) ? fail(FMSCAN_E_SHAPE, "%s: the strides of %s must be in [0, 2^44]", who, name) : 0;
}

// S states of `each` elements: a pool whose size in bytes fits 63 bits with room, and one state a row without slots
inline int check_pool(const char* who, int64_t S, int64_t B, int64_t each, const void* slots) {
    if (S < 1 || S > INT32_MAX || (__int128)S * each > ((__int128)1 << 44))
        return fail(FMSCAN_E_SHAPE, "%s: the pool must hold 1 to 2^31 - 1 states and at most 2^44 elements (got %lld)", who,
                    (long long)S);
    if (!slots && S != B)
        return fail(FMSCAN_E_SHAPE, "%s: without slots the pool holds a state a row: %lld, got %lld", who, (long long)B,
                    (long long)S);
    return 0;
}

// the bytes between the first and the last element of a strided tensor (at most 2^62: a range, not a size to allocate)
inline int64_t span(std::initializer_list<std::pair<int64_t, int64_t>> axes, int esize) {
    __int128 n = 1;
    for (const auto& a : axes) n += (__int128)(a.first - 1) * a.second;
    n *= esize;
    return n > ((__int128)1 << 62) ? (int64_t)1 << 62 : (int64_t)n;
}
inline int64_t extent(int64_t B, int64_t D, int64_t L, int64_t sb, int64_t sd, int esize) {
    return span({{B, sb}, {D, sd}, {L, 1}}, esize);
}

// A launch's threads are counted in 32 bits
inline int check_grid(const char* who, __int128 blocks, int threads) {
    return blocks * threads >= ((__int128)1 << 32) ? fail(FMSCAN_E_SHAPE, "%s: these sizes are too large for one launch", who) : 0;
}

inline int check_alias(const char* who, std::initializer_list<Range> outs, std::initializer_list<Range> ins) {
    for (const Range* o = outs.begin(); o != outs.end(); ++o) {
        for (const Range& i : ins)
            if (overlap(*o, i)) return fail(FMSCAN_E_ALIAS, "%s: %s overlaps %s", who, o->name, i.name);
        for (const Range* q = outs.begin(); q != o; ++q)
            if (overlap(*o, *q)) return fail(FMSCAN_E_ALIAS, "%s: %s overlaps %s", who, o->name, q->name);
    }
    return 0;
}

// The sections of one launch, and its blocks
inline uint32_t column_sections(std::initializer_list<ColumnSum> parts, ColumnSums* s) {
    uint32_t blocks = 0;
    int k = 0;
    *s = {};
    for (const ColumnSum& p : parts) {
        if (!p.out) continue;
        s->part[k] = p;
        s->part[k].first_block = blocks;
        blocks += (uint32_t)((p.cols + 63) / 64);
        ++k;
    }
    return blocks;
}
inline void launch_column_sums(int dtype, std::initializer_list<ColumnSum> parts, hipStream_t stream) {
    ColumnSums s;
    const uint32_t blocks = column_sections(parts, &s);
    with_dtype(dtype, [&](auto tt) {
        using T = typename decltype(tt)::type;
        column_sums_kernel<T><<<blocks, 64 * kSumWaves, 0, stream>>>(s);
    });
}

}  // namespace host
}  // namespace fmselective
