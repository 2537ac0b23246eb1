// fixed_prefix.hip -- attention behind a prefix that all sequences share, for all of
// their rows together (the mathematics is at the head of fixed_attention.hip, and there
// the choice between this and each sequence by itself, which many rows or short
// prefixes prefer).
//
// The rows of all sequences are one long list for the prefix: 32 of them at a
// time meet each of its tiles on the matrix cores, so that its keys and values are
// read once for 32 rows, not once a sequence.  A row's maximum runs over the
// prefix and its own sequence, and an exponential is a table's entry, so there are
// two passes: the maxima of every part of the tokens (TOPS), then the parts' sums
// with scores computed again (SUMS); a third launch adds the parts' sums (whole
// numbers: any order gives the same) and divides.  Scores computed twice cost
// 128 multiply-adds each, on matrix cores that wait for memory; kept, they would take
// 4 bytes a row and token, written and read.
//
// 64 sequences of one token, 32 heads of 128 on 8 key heads, own tokens up to 255 behind
// 8,192: 20 + 38 + 5 us, where each by itself takes 226.  The sums are bound by their chain:
// with 192 registers of sums a SIMD has one wave, whose products, exponentials and loads of
// values follow each other (matrix cores busy 0.19, vector issue 0.23; reads of the table,
// at 64 places, conflict).
//
// A workgroup takes 32 rows of a key head and a part of what they read: the prefix's
// tiles, then the own tiles of the sequences that the rows are of, each of which only
// its sequence's rows see.  (As parts of their own, of few rows, those cost another
// beginning and end each.)  Its waves take the tiles in turn, straight from memory ahead
// of their use, and add their sums in LDS.
#include <algorithm>
#include <climits>

#include "fixed_attention.hpp"

namespace vmx {
namespace {

using namespace fx;

constexpr int ROWS = 32;

// The sequence of item `at` of an ascending list of firsts.
__device__ inline uint32_t search(const uint32_t* first, uint32_t count, uint32_t at) {
    uint32_t lo = 0, hi = count;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (first[mid] <= at)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// Sequences of a launch.  Their tokens, in turn, are numbered from 0.
struct Batch {
    FxSeq s[FX_SEQS];
    uint32_t before[FX_SEQS + 1];  // tokens before each sequence's
    uint32_t tiles[FX_SEQS + 1];   // own tiles before each sequence's
    uint32_t count;
    uint32_t each;                 // tokens of every sequence, 0 if they differ
    bool joined;                   // the sequences' rows follow each other
    __device__ uint32_t sequence_of(uint32_t token) const { return each ? token / each : search(before, count, token); }
};

struct PartArgs {
    uint32_t blocks;     // of 32 rows of all sequences
    uint32_t splits;     // parts of what a block reads, of this launch
    uint32_t top_parts;  // of the maxima
    int* tops;           // parts x tokens x heads
    int64_t* sums;       // parts x tokens x heads x places (64 or 128): sum e (v - 128)
    int* totals;         // parts x tokens x heads: sum e
};

// Keys of 32 tokens, and the extra of token lane & 31.
template <int DC>
struct Keys {
    v4i h[2 * DC], l[2 * DC];
    int extra;
};

template <int DC>
__device__ inline void load_keys(const unsigned char* rec, int block, int lane, Keys<DC>* k) {
    const v4i* p = reinterpret_cast<const v4i*>(rec) + block * 2 * DC * 128 + lane;
#pragma unroll
    for (int u = 0; u < 2 * DC; ++u) k->h[u] = p[u * 128], k->l[u] = p[u * 128 + 64];
    k->extra = reinterpret_cast<const int*>(rec + Record<DC>::EXTRA)[block * 32 + (lane & 31)];
}

template <int DC>
__device__ inline Raw products(const Keys<DC>& k, const Query<DC>& q) {
    Raw s;
#pragma unroll
    for (int u = 0; u < 2 * DC; ++u) {
        s.hh = mfma32(k.h[u], q.h[u], s.hh);
        s.mid = mfma32(k.h[u], q.l[u], s.mid);
        s.ll = mfma32(k.l[u], q.l[u], s.ll);
        s.mid = mfma32(k.l[u], q.h[u], s.mid);
    }
    return s;
}

// Waves of a workgroup.  The sums of 32 rows and 128 places take 192 registers a lane:
// with heads over 64 a wave has a SIMD for itself.
template <int DC, bool SUMS>
constexpr int WAVES = SUMS && DC == 2 ? 4 : 8;

template <int DC, bool SUMS>
__global__ __launch_bounds__((64 * WAVES<DC, SUMS>)) void fx_prefix_kernel(AttentionArgs a, PartArgs f, Batch q) {
    constexpr int W = WAVES<DC, SUMS>, THREADS = 64 * W, PLACES = 64 * DC;
    constexpr int PITCH = ROWS + 1;  // a place's rows follow each other: neither writes nor reads conflict
    __shared__ __attribute__((aligned(16))) uint16_t table[SUMS ? FX_TABLE_MAX : 8];
    __shared__ int64_t sums[SUMS ? W : 1][SUMS ? PLACES * PITCH : 1];
    __shared__ int tops[W][ROWS];  // and totals
    // Heads vary fastest, then the blocks of rows: an XCD gets few heads, and the blocks that
    // read the same tiles of the prefix run together.
    const uint32_t item = blockIdx.x / static_cast<uint32_t>(a.kv_heads), part = item / f.blocks;
    const int head = static_cast<int>(blockIdx.x - item * static_cast<uint32_t>(a.kv_heads));
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t tokens = q.before[q.count], heads = static_cast<uint32_t>(a.kv_heads) * a.group;
    const int row0 = static_cast<int>(item - part * f.blocks) * ROWS;
    const int cols = min(static_cast<int>(tokens) * a.group - row0, ROWS);
    // this lane's row, its token, that token's sequence and place in the packed rows
    const int row = row0 + min(lane & 31, cols - 1);
    const bool live = (lane & 31) < cols;
    const uint32_t token = static_cast<uint32_t>(row) / a.group, member = row % a.group;
    // the sequences of the first row and of the last, and this part's tiles
    const uint32_t seq0 = q.sequence_of(static_cast<uint32_t>(row0) / a.group);
    const uint32_t seq1 = q.sequence_of(static_cast<uint32_t>(row0 + cols - 1) / a.group);
    const int shared = (static_cast<int>(a.prefix) + FX_TILE - 1) / FX_TILE;
    const int tiles = shared + static_cast<int>(q.tiles[seq1 + 1] - q.tiles[seq0]);
    const int each = (tiles + static_cast<int>(f.splits) - 1) / static_cast<int>(f.splits);
    const int from = static_cast<int>(part) * each, to = min(from + each, tiles);
    const uint32_t seq = q.sequence_of(token);
    const int limit = limit_of(a, q.s[seq], static_cast<int>(token - q.before[seq]) * a.group);
    const size_t packed = q.s[seq].row + (token - q.before[seq]);
    const size_t slot_bytes = a.kv_heads * a.tiles * static_cast<size_t>(Record<DC>::BYTES);
    const unsigned char* base = a.data + static_cast<size_t>(head) * a.tiles * static_cast<size_t>(Record<DC>::BYTES);
    // The i-th tile, asked for in ascending order: its record, its first token, the sequence that alone sees it (-1: all do) and its
    // slot's tokens.
    struct Tile {
        const unsigned char* rec;
        int first, seq, written;
    };
    uint32_t own = seq0;
    auto tile = [&](int i) {
        if (i < shared)
            return Tile{base + a.prefix_slot * slot_bytes + static_cast<size_t>(i) * Record<DC>::BYTES, i * FX_TILE, -1,
                        static_cast<int>(a.prefix)};
        const uint32_t at = static_cast<uint32_t>(i - shared) + q.tiles[seq0];
        while (q.tiles[own + 1] <= at) ++own;
        const uint32_t j = at - q.tiles[own];
        return Tile{base + q.s[own].slot * slot_bytes + j * static_cast<size_t>(Record<DC>::BYTES),
                    static_cast<int>(j) * FX_TILE, static_cast<int>(own), static_cast<int>(q.s[own].length)};
    };
    const int begin = from + wave;
    // Keys that are on their way: of this tile and, for the maxima, of the next.
    constexpr int AHEAD = SUMS ? 1 : 2;
    Keys<DC> keys[AHEAD][2];
    Tile now[AHEAD] = {};
    if (begin < to) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            now[k] = tile(min(begin + k * W, to - 1));
#pragma unroll
            for (int b = 0; b < 2; ++b) load_keys<DC>(now[k].rec, b, lane, &keys[k][b]);
        }
    }
    Table<THREADS> to_table;
    if constexpr (SUMS) to_table.load(a.table, static_cast<int>(a.entries));
    Query<DC> mine;
    load_query<DC>(a.q + packed * a.q_stride + (static_cast<size_t>(head) * a.group + member) * a.dim, live, a.dim, lane, &mine);
    const bool no_offset = !__any(mine.o);
    // index of this lane's row in a part's tops
    const size_t mine_at = static_cast<size_t>(token) * heads + static_cast<size_t>(head) * a.group + member;
    // Whether block b of tile t needs no offsets.
    auto is_plain = [&](const Tile& t, int b, const Keys<DC>& k) {
        return no_offset && !__any(t.first + b * 32 + (lane & 31) < t.written && (k.extra & 128));
    };
    // Whether all rows see tile t whole, without offsets: most tiles, and the first ones.
    auto is_whole = [&](const Tile& t, const Keys<DC>* k) {
        return a.s2 == 0 && t.seq < 0 && t.first + FX_TILE <= t.written && is_plain(t, 0, k[0]) && is_plain(t, 1, k[1]);
    };
    // Scores of block b of tile t from keys k, which then are on their way for tile `next`.
    auto scores_of = [&](const Tile& t, int b, Keys<DC>* k, const Tile& next) {
        const Raw raw = products<DC>(*k, mine);
        const bool plain = is_plain(t, b, *k);
        load_keys<DC>(next.rec, b, lane, k);
        return scores<DC>(raw, reinterpret_cast<const int*>(t.rec + Record<DC>::EXTRA), mine, b, lane, a.s1, a.s2, plain);
    };
    // Keys of a tile that this lane's row sees.
    auto limit_in = [&](const Tile& t) { return t.seq < 0 ? t.written : t.seq == static_cast<int>(seq) ? limit : 0; };

    if constexpr (!SUMS) {
        int top = INT_MIN;
        // past the last, keys that are not used
        auto use = [&](int i, Tile* t, Keys<DC>* k) {
            const Tile next = tile(min(i + AHEAD * W, to - 1));
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int first = t->first + b * 32;
                const v16i z = scores_of(*t, b, &k[b], next);
                if (t->seq < 0 && first + 32 <= t->written) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) top = max(top, z[r]);
                } else {
                    const int here = limit_in(*t);
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (first + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3) < here) top = max(top, z[r]);
                }
            }
            *t = next;
        };
        for (int i = begin; i < to; i += 2 * W) {
            use(i, &now[0], keys[0]);
            if (i + W < to) use(i + W, &now[AHEAD - 1], keys[AHEAD - 1]);
        }
        top = max(top, __shfl_xor(top, 32));
        if (lane < ROWS) tops[wave][lane] = top;
        __syncthreads();
        if (wave == 0 && lane < cols) {
            for (int w = 1; w < W; ++w) top = max(top, tops[w][lane]);
            f.tops[static_cast<size_t>(part) * tokens * heads + mine_at] = top;
        }
    } else {
        int top = INT_MIN;
        for (uint32_t i = 0; i < f.top_parts; ++i)
            top = max(top, f.tops[static_cast<size_t>(i) * tokens * heads + mine_at]);
        to_table.store(a.table, static_cast<int>(a.entries), table);
        __syncthreads();
        const uint32_t last = a.entries - 1;
        v16i hh[2 * DC] = {}, mid[2 * DC] = {}, ll[2 * DC] = {};
        int sum_h = 0, sum_l = 0;
        // of 32 tokens with scores z(r), from `first` on, of which the lane's row sees those below `here`
        auto exponentials = [&](auto&& z, bool whole, int first, int here, v4i* eh, v4i* el) {
            uint32_t e[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) e[r] = table[min(static_cast<uint32_t>(top) - static_cast<uint32_t>(z(r)), last)];
            if (!whole) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (first + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3) >= here) e[r] = 0;
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const uint32_t a01 = e[4 * g] | e[4 * g + 1] << 16, a23 = e[4 * g + 2] | e[4 * g + 3] << 16;
                (*eh)[g] = __builtin_amdgcn_perm(a23, a01, 0x07050301u);
                (*el)[g] = __builtin_amdgcn_perm(a23, a01, 0x06040200u);
                sum_h = __builtin_amdgcn_sdot4((*eh)[g], 0x01010101, sum_h, false);
                sum_l = __builtin_amdgcn_sdot4((*el)[g], 0x01010101, sum_l, false);
            }
        };
        struct Values {
            v4i h[2 * DC], l[2 * DC];
        };
        auto load_values = [&](const Tile& t, int b, Values* v) {
            const v4i* p = reinterpret_cast<const v4i*>(t.rec + Record<DC>::VALUES) + b * 2 * DC * 128 + lane;
#pragma unroll
            for (int d = 0; d < 2 * DC; ++d) v->h[d] = p[d * 128], v->l[d] = p[d * 128 + 64];
        };
        auto add = [&](const Values& v, v4i eh, v4i el) {
#pragma unroll
            for (int d = 0; d < 2 * DC; ++d) {
                hh[d] = mfma32(v.h[d], eh, hh[d]);
                mid[d] = mfma32(v.h[d], el, mid[d]);
                ll[d] = mfma32(v.l[d], el, ll[d]);
                mid[d] = mfma32(v.l[d], eh, mid[d]);
            }
        };
        // (Sums added beside the next block's exponentials, in an order set for it, would overlap the matrix
        // cores and the vector units; the registers that takes spilled: 105 us for 40.)
        Values values;
        int i = begin;
        for (; i < to; i += W) {
            const Tile t = now[0];
            if (!is_whole(t, keys[0])) break;
            const Tile next = tile(min(i + W, to - 1));
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                load_values(t, b, &values);
                const Raw s = products<DC>(keys[0][b], mine);
                load_keys<DC>(next.rec, b, lane, &keys[0][b]);
                v4i eh, el;
                exponentials([&](int r) { return score(s, r, a.s1); }, true, 0, 0, &eh, &el);
                add(values, eh, el);
            }
            now[0] = next;
        }
        for (; i < to; i += W) {
            const Tile t = now[0], next = tile(min(i + W, to - 1));
            const int here = limit_in(t);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                load_values(t, b, &values);
                const v16i z = scores_of(t, b, &keys[0][b], next);
                v4i eh, el;
                exponentials([&](int r) { return z[r]; }, false, t.first + b * 32, here, &eh, &el);
                add(values, eh, el);
            }
            now[0] = next;
        }
        // Each wave's sums to LDS, then their sums to memory.  (Additions by LDS atomics took 5 us more.)
        int total = 256 * sum_h + sum_l;
        total += __shfl_xor(total, 32);
        if (lane < ROWS) tops[wave][lane] = total;
#pragma unroll
        for (int d = 0; d < 2 * DC; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                sums[wave][(d * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)) * PITCH + (lane & 31)] =
                    join(hh[d][r], mid[d][r], ll[d][r]);
        __syncthreads();
        for (int i = threadIdx.x; i < cols * PLACES; i += THREADS) {
            const int col = i / PLACES, place = i % PLACES;
            const uint32_t at = static_cast<uint32_t>(row0 + col) / a.group, m = (row0 + col) % a.group;
            const size_t to_row = (static_cast<size_t>(part) * tokens + at) * heads + static_cast<size_t>(head) * a.group + m;
            int64_t sum = 0;
            int all = 0;
#pragma unroll
            for (int w = 0; w < W; ++w) sum += sums[w][place * PITCH + col], all += tops[w][col];
            f.sums[to_row * PLACES + place] = sum;
            if (place == 0) f.totals[to_row] = all;
        }
    }
}

// The parts' sums of a row, added and divided: four places a thread.
template <int DC>
__global__ __launch_bounds__(256) void fx_prefix_join_kernel(AttentionArgs a, PartArgs f, Batch q) {
    constexpr int PLACES = 64 * DC, PIECES = PLACES / 4;
    const uint32_t tokens = q.before[q.count], heads = static_cast<uint32_t>(a.kv_heads) * a.group;
    const uint32_t id = blockIdx.x * 256 + threadIdx.x, row = id / PIECES;
    const int place = static_cast<int>(id % PIECES) * 4;
    if (row >= tokens * heads || place >= a.dim) return;
    const size_t rows = static_cast<size_t>(tokens) * heads;
    int64_t total = 0, sums[4] = {};
#pragma unroll 4  // so many loads under way
    for (uint32_t i = 0; i < f.splits; ++i) {
        typedef long v2l __attribute__((ext_vector_type(2)));
        const v2l* p = reinterpret_cast<const v2l*>(f.sums + (i * rows + row) * PLACES + place);
        const v2l lo = p[0], hi = p[1];
        total += f.totals[i * rows + row];
        sums[0] += lo[0], sums[1] += lo[1], sums[2] += hi[0], sums[3] += hi[1];
    }
    const Divide divide(total);
    int v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = divide(2.0 * static_cast<double>(sums[r]));
    const uint32_t token = row / heads, at = q.joined ? 0 : q.sequence_of(token);
    store4(a.out + (static_cast<size_t>(q.s[at].row) + (token - q.before[at])) * a.out_stride +
               static_cast<size_t>(row - token * heads) * a.dim + place,
           a.dim - place, v);
}

// What a launch group needs: its sequences, and the parts of both passes.
struct Launch {
    Batch q{};
    PartArgs tops{}, sums{};
    size_t rows() const { return q.before[q.count]; }  // of all heads
};

template <int DC>
Launch plan(Context* c, const AttentionArgs& a, const FxSeq* seqs, size_t count) {
    Launch l;
    l.q.joined = true;
    l.q.each = seqs[0].count;
    for (size_t i = 0; i < count; ++i) {
        l.q.s[i] = seqs[i];
        l.q.before[i + 1] = l.q.before[i] + seqs[i].count;
        l.q.tiles[i + 1] = l.q.tiles[i] + (seqs[i].length + FX_TILE - 1) / FX_TILE;
        if (i && seqs[i].row != seqs[i - 1].row + seqs[i - 1].count) l.q.joined = false;
        if (seqs[i].count != l.q.each) l.q.each = 0;
    }
    l.q.count = static_cast<uint32_t>(count);
    const size_t cus = static_cast<size_t>(c->cu_count);
    PartArgs f{};
    f.blocks = static_cast<uint32_t>((l.rows() * a.group + ROWS - 1) / ROWS);
    // As many workgroups as CUs, as each has one for itself, and a tile a wave at least.
    const size_t units = f.blocks * a.kv_heads;
    const size_t tiles = (a.prefix + FX_TILE - 1) / FX_TILE + l.q.tiles[count] / f.blocks;
    auto splits = [&](size_t waves) {
        return static_cast<uint32_t>(std::max<size_t>(1, std::min(cus / units, (tiles + waves - 1) / waves)));
    };
    l.tops = l.sums = f;
    l.tops.splits = splits(WAVES<DC, false>);
    l.sums.splits = splits(WAVES<DC, true>);
    l.tops.top_parts = l.sums.top_parts = l.tops.splits;
    return l;
}

template <int DC>
int launch(Context* c, const AttentionArgs& a, const Launch& l) {
    auto grid = [&](const PartArgs& f) {
        return dim3(static_cast<unsigned>(f.blocks * f.splits * a.kv_heads));
    };
    hipLaunchKernelGGL((fx_prefix_kernel<DC, false>), grid(l.tops), dim3(64 * WAVES<DC, false>), 0, c->stream, a, l.tops,
                       l.q);
    VMX_HIP(c, hipGetLastError());
    hipLaunchKernelGGL((fx_prefix_kernel<DC, true>), grid(l.sums), dim3(64 * WAVES<DC, true>), 0, c->stream, a, l.sums,
                       l.q);
    VMX_HIP(c, hipGetLastError());
    const size_t threads = l.rows() * a.kv_heads * a.group * (16 * DC);
    hipLaunchKernelGGL(fx_prefix_join_kernel<DC>, dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), 0, c->stream,
                       a, l.sums, l.q);
    VMX_HIP(c, hipGetLastError());
    return 0;
}

}  // namespace

int fx_prefix_attention(Context* c, const FxCache& cache, const FxAttention& t, const FxSeq* seqs, size_t count,
                        bool* no_space) {
    const AttentionArgs a = attention_args(cache, t);
    const bool wide = cache.dim > 64;
    // Sequences in launches of FX_SEQS; a launch reuses the space of the one before, as they run in order.
    auto make = [&](size_t at) {
        const size_t here = std::min<size_t>(count - at, FX_SEQS);
        return wide ? plan<2>(c, a, seqs + at, here) : plan<1>(c, a, seqs + at, here);
    };
    const size_t places = fx_head_pad(cache.dim);
    auto rows_of = [&](const Launch& l) { return l.sums.splits * l.rows() * t.heads; };
    size_t most = 0;
    for (size_t at = 0; at < count; at += FX_SEQS) {
        const Launch l = make(at);
        most = std::max(most, rows_of(l) * (8 * places + 4) + 4 * l.tops.top_parts * l.rows() * t.heads);
    }
    *no_space = most > FX_SPACE_MAX || !try_ws(c, WS_FIXED, workspace_step(most, FX_SPACE_MAX));
    if (*no_space) return 0;
    for (size_t at = 0; at < count; at += FX_SEQS) {
        Launch l = make(at);
        l.sums.sums = ws<int64_t>(c, WS_FIXED);
        l.sums.totals = reinterpret_cast<int*>(l.sums.sums + rows_of(l) * places);
        l.tops.tops = l.sums.tops = l.sums.totals + rows_of(l);
        if (wide ? launch<2>(c, a, l) : launch<1>(c, a, l)) return -1;
    }
    return 0;
}

}  // namespace vmx
