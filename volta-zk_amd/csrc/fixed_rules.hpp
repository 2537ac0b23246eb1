// fixed_rules.hpp -- which kernels take attention behind a prefix, from sizes alone: host
// code that the CPU tests call too (host_check.cpp), so that the GPU tests of a kernel
// know that their cases reach it.
#pragma once

#include <algorithm>

#include "fixed.hpp"

namespace vmx {
namespace fx {

constexpr int FEW = 16;  // rows of a workgroup where rows are few (fixed_attention.hip)

// Microseconds that sequences behind a prefix take with those of up to `limit` rows together
// (fixed_prefix.hip) and each other by itself.  Measured, one token a sequence behind `tiles`,
// with units of 16 rows, together and by itself:
//   heads of 64 (12 key heads)       of 128 (8 key heads)
//   24 x 250     31.6 and 42.2       16 x 250     47.6 and 46.8
//   48 x 63      21.9 and 20.7       32 x 63      30.8 and 26.3
//   96 x 63      23.8 and 35.0       64 x 63      34.1 and 35.0
//   768 x 4      25.5 and 17.8       512 x 4      33.7 and 22.4
//   768 x 16     26.6 and 29.4       512 x 16     35.1 and 37.5
//   768 x 250    49.1 and 266        512 x 250    82.7 and 372
// and prompts by themselves: 96 workgroups of 128 rows x 39 tiles 70, 480 x 37 132; heads of 96, 40 x
// 175 290.
inline double prefix_us(const FxCache& cache, const FxAttention& t, const FxSeq* first, const FxSeq* end, size_t limit) {
    const bool wide = cache.dim > 64;
    const size_t group = t.heads / cache.kv_heads, kv = cache.kv_heads, shared = (t.prefix + FX_TILE - 1) / FX_TILE;
    size_t sequences = 0, rows32 = 0, own = 0;                // together: sequences, rows, own tiles of 32 rows
    size_t units = 0, reads = 0, longest_few = 0, cols = 0;  // by itself, few rows: units of 16, tiles they read
    size_t blocks_tiles = 0, longest_many = 0;               // many rows: tiles that blocks of 128 read
    for (const FxSeq* s = first; s != end; ++s) {
        const size_t rows = size_t{s->count} * group, tiles = (s->length + FX_TILE - 1) / FX_TILE, all = shared + tiles;
        if (rows <= limit) {
            ++sequences;
            rows32 += rows;
            own += tiles * ((rows + 31) / 32);
        } else if (rows <= FEW) {
            units += kv;
            reads += kv * all;
            longest_few = std::max(longest_few, all);
            cols = std::max(cols, rows);
        } else {
            blocks_tiles += (rows + 127) / 128 * kv * all;
            longest_many = std::max(longest_many, all);
        }
    }
    double us = 0;
    if (sequences) {
        const double work = static_cast<double>(kv * ((rows32 + 31) / 32 * shared + own));
        us += (sequences + FX_SEQS - 1) / FX_SEQS * (wide ? 30.0 : 20.0) + work * (wide ? 0.0034 : 0.0048);
    }
    if (units) {
        const double tiles = static_cast<double>(longest_few), all = static_cast<double>(reads);
        const bool kept = tiles * ((wide ? 750 : 550) - (wide ? 9.0 : 5.0) * static_cast<double>(units)) <= 10000 &&
                          longest_few * cols * 256 <= 65536;
        us += kept ? (wide ? 10 : 9) + std::max(tiles * (wide ? 0.45 : 0.4), all * (wide ? 0.0029 : 0.0014))
                   : (wide ? 10 + 0.14 * tiles + 0.0027 * all : 9 + 0.11 * tiles + 0.0011 * all);
    }
    if (blocks_tiles)
        us += 8 + std::max(static_cast<double>(longest_many) * (wide ? 1.66 : 1.75),
                           static_cast<double>(blocks_tiles) * (wide ? 0.012 : 0.0077));
    return us;
}

// Sequences of up to so many rows read the prefix together: none (0), those of few rows, or all
// (SIZE_MAX), whichever the estimates have done first.
inline size_t prefix_limit(const FxCache& cache, const FxAttention& t, const FxSeq* first, const FxSeq* end) {
    const size_t limits[] = {0, cache.dim <= 64 ? size_t{47} : size_t{98}, SIZE_MAX};
    size_t limit = 0;
    double best = 0;
    for (const size_t here : limits) {
        const double us = prefix_us(cache, t, first, end, here);
        if (here == 0 || us < best) best = us, limit = here;
    }
    return limit;
}

}  // namespace fx
}  // namespace vmx
