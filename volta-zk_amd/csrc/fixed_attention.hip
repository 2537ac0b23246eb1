// fixed_attention.hip -- attention over a cache of keys and values in 16-bit
// integers, and the cache's append (layout in fixed.hpp).
//
// z = (q . k) >> shift, d = max_j z - z, e = table[min(d, entries - 1)],
// out = sum e v / sum e rounded to the nearest integer, halves up.  The maximum
// runs over the keys a query may see, and a query without any gives zeros.
//
// Rows of a launch are the pairs (token, query head) of one key head's group,
// so grouped heads share the keys and values that a workgroup reads.  Scores are
// computed transposed, S^T = K Q^T: a lane then holds scores of one query only,
// its statistics are one register, and the exponentials are already in the
// layout in which O^T = V^T E^T reads them.
//
// 16-bit scores from four i8 products, as in fixed.hpp, with offsets only for
// keys and queries that hold a value over 32,639; s - 2^16 sum qh kh fits 32 bits
// for heads of up to 128, so z = ((hh << 16 - s1) + (c >> s1)) >> s2 with
// s1 = min(shift, 16) never needs 64-bit arithmetic.  e (at most 2^14) is
// 256 h + l with signed bytes; values keep the constant offset of 128, whose
// correction is 128 sum e.
#include <algorithm>
#include <climits>
#include <vector>

#include "fixed.hpp"

namespace vmx {
namespace {

using namespace fx;

struct Seqs {
    FxSeq s[FX_SEQS];
    uint32_t first[FX_SEQS + 1];  // work items before each sequence (of each, for many rows)
    uint32_t count;
};

// The sequence of work item `at` (first[] ascends; a scalar search).
__device__ inline uint32_t sequence_of(const Seqs& q, uint32_t at) {
    uint32_t lo = 0, hi = q.count;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (q.first[mid] <= at)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// Parts of a record (fixed.hpp), in bytes.
template <int DC>
struct Record {
    static constexpr int VALUES = DC * 8192, EXTRA = DC * 16384, BYTES = DC * 16384 + 256;
};

// Sixteen i16 less o (0 or 128) as their signed high and low bytes.
__device__ inline void split16(v4i lo, v4i hi, int o, v4i* h, v4i* l) {
    const int up = o ? 0 : 0x00800080, flip = o ? 0x80808080 : 0;
    v4i a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int x = lo[i], y = hi[i];
        a[i] = __builtin_bit_cast(int, __builtin_bit_cast(v2s, x) + __builtin_bit_cast(v2s, up));
        b[i] = __builtin_bit_cast(int, __builtin_bit_cast(v2s, y) + __builtin_bit_cast(v2s, up));
    }
    const uint32_t top = 0x07050301u, bottom = 0x06040200u;
    *h = v4i{static_cast<int>(__builtin_amdgcn_perm(a[1], a[0], top)),
             static_cast<int>(__builtin_amdgcn_perm(a[3], a[2], top)),
             static_cast<int>(__builtin_amdgcn_perm(b[1], b[0], top)),
             static_cast<int>(__builtin_amdgcn_perm(b[3], b[2], top))};
    *l = v4i{static_cast<int>(__builtin_amdgcn_perm(lo[1], lo[0], bottom)) ^ flip,
             static_cast<int>(__builtin_amdgcn_perm(lo[3], lo[2], bottom)) ^ flip,
             static_cast<int>(__builtin_amdgcn_perm(hi[1], hi[0], bottom)) ^ flip,
             static_cast<int>(__builtin_amdgcn_perm(hi[3], hi[2], bottom)) ^ flip};
}

// Whether one of eight i16 is over HALVES_MAX.
__device__ inline bool large8(v4i v) {
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) any |= static_cast<int16_t>(v[i]) > HALVES_MAX || (v[i] >> 16) > HALVES_MAX;
    return any;
}

// ---- append ---------------------------------------------------------------------------
// One workgroup per (key head, 64-token tile that new tokens touch).  A token
// after others of its tile is written byte by byte, as its tile's pieces hold other
// tokens' bytes; a tile from its first token on in pieces of 16, where no token past the
// last shares them: what the cache holds of those stays.  Bound by memory,
// one token by its latency: 16 prompts of 10,575 tokens, 12 heads of 64 (67 MB)
// 13.7 us, 4.9 TB/s, what a copy reaches; one token of 12 heads 2.2 us.
struct AppendArgs {
    unsigned char* data;
    size_t kv_heads, tiles;
    int dim;
    const int16_t *k, *v;
    size_t k_stride, v_stride;
};

template <int DC>
__global__ __launch_bounds__(256) void fx_append_kernel(AppendArgs a, Seqs q) {
    __shared__ int sums[64], large[64];
    const uint32_t at = sequence_of(q, blockIdx.x);
    const FxSeq s = q.s[at];
    const int past = static_cast<int>(s.length - s.count);
    const int tile = past / FX_TILE + static_cast<int>(blockIdx.x - q.first[at]);
    const int head = blockIdx.y;
    unsigned char* rec =
        a.data + ((static_cast<size_t>(s.slot) * a.kv_heads + head) * a.tiles + tile) * Record<DC>::BYTES;
    unsigned char* values = rec + Record<DC>::VALUES;
    int* extra = reinterpret_cast<int*>(rec + Record<DC>::EXTRA);
    const int from = max(past - tile * FX_TILE, 0), to = min(static_cast<int>(s.length) - tile * FX_TILE, FX_TILE);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // row of token j of this tile
    const size_t row0 = static_cast<size_t>(s.row) + tile * FX_TILE - past;
    const int16_t* k0 = a.k + static_cast<size_t>(head) * a.dim;
    const int16_t* v0 = a.v + static_cast<size_t>(head) * a.dim;
    if (from == 0) {
        // A tile from its first token on.
        if (threadIdx.x < 64) sums[threadIdx.x] = large[threadIdx.x] = 0;
        __syncthreads();
        const int j = threadIdx.x & 63;
        v4i lo[DC], hi[DC];
#pragma unroll
        for (int c = 0; c < DC; ++c) {
            lo[c] = hi[c] = v4i{0, 0, 0, 0};
            if (j < to) {
                load16(k0 + (row0 + j) * a.k_stride, (c * 4 + wave) * 16, a.dim, &lo[c], &hi[c]);
                atomicAdd(&sums[j], sum8(hi[c], sum8(lo[c], 0)));
                if (large8(lo[c]) || large8(hi[c])) large[j] = 128;
            }
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < DC; ++c) {
            const int piece = c * 4 + wave;  // places 16 piece ..
            if (j >= to) continue;
            v4i h, l;
            split16(lo[c], hi[c], large[j], &h, &l);
            v4i* p = reinterpret_cast<v4i*>(rec) + ((j >> 5) * 2 * DC + (piece >> 1)) * 128 + (j & 31) + 32 * (piece & 1);
            p[0] = h;
            p[64] = l;
        }
        if (threadIdx.x < 64 && j < to) extra[j] = sums[j] * 256 + large[j];
#pragma unroll
        for (int c = 0; c < DC; ++c) {
            // piece (32-token block, half of it, place)
            const int i = c * 256 + threadIdx.x, d = i % (64 * DC), part = i / (64 * DC), block = part >> 1, half = part & 1;
            union {
                v4i v;
                uint8_t b[16];
            } h, l;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int t = block * 32 + 8 * (e >> 2) + 4 * half + (e & 3);
                const int x = t < to && d < a.dim ? v0[(row0 + t) * a.v_stride + d] : 0;
                h.b[e] = static_cast<uint8_t>(x >> 8);
                l.b[e] = static_cast<uint8_t>(x ^ 0x80);
            }
            v4i* p = reinterpret_cast<v4i*>(values) + (block * 2 * DC + (d >> 5)) * 128 + (d & 31) + 32 * half;
            if (block * 32 + 4 * half + 27 < to) {
                p[0] = h.v;
                p[64] = l.v;
            } else {
                uint8_t* bytes = reinterpret_cast<uint8_t*>(p);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    if (block * 32 + 8 * (e >> 2) + 4 * half + (e & 3) >= to) continue;
                    bytes[e] = h.b[e];
                    bytes[1024 + e] = l.b[e];
                }
            }
        }
        return;
    }
    // Tokens after others of their tile: their own bytes, a token a wave.
    for (int j = from + wave; j < to; j += 4) {
        int sum = 0;
        bool over = false;
        int kd[DC], vd[DC];
#pragma unroll
        for (int c = 0; c < DC; ++c) {
            const int d = c * 64 + lane;
            kd[c] = d < a.dim ? k0[(row0 + j) * a.k_stride + d] : 0;
            vd[c] = d < a.dim ? v0[(row0 + j) * a.v_stride + d] : 0;
            sum += kd[c];
            over |= kd[c] > HALVES_MAX;
        }
        const int o = __any(over) ? 128 : 0;
        for (int m = 32; m; m >>= 1) sum += __shfl_xor(sum, m);
#pragma unroll
        for (int c = 0; c < DC; ++c) {
            const int d = c * 64 + lane, kk = halves(kd[c] - o);
            unsigned char* pk = rec + (((j >> 5) * 2 * DC + (d >> 5)) * 128 + (j & 31) + 32 * ((d >> 4) & 1)) * 16 + (d & 15);
            pk[0] = static_cast<unsigned char>(kk >> 8);
            pk[1024] = static_cast<unsigned char>(kk);
            unsigned char* pv = values + (((j >> 5) * 2 * DC + (d >> 5)) * 128 + (d & 31) + 32 * ((j >> 2) & 1)) * 16 +
                                ((j >> 3) & 3) * 4 + (j & 3);
            pv[0] = static_cast<unsigned char>(vd[c] >> 8);
            pv[1024] = static_cast<unsigned char>(vd[c] ^ 0x80);
        }
        if (lane == 0) extra[j] = sum * 256 + o;
    }
}

// ---- attention --------------------------------------------------------------------------
struct AttentionArgs {
    const unsigned char* data;
    size_t kv_heads, tiles;
    const int16_t* q;
    size_t q_stride;
    int16_t* out;
    size_t out_stride;
    const uint16_t* table;
    int dim, group;
    uint32_t entries;
    uint32_t s1, s2;  // shift = s1 + s2, s1 = min(shift, 16)
    bool causal;
};

// Keys that row `row` of a sequence may see.
__device__ inline int limit_of(const AttentionArgs& a, const FxSeq& s, int row) {
    return static_cast<int>(s.length) - (a.causal ? static_cast<int>(s.count) - row / a.group - 1 : 0);
}

// A lane's query: its planes (32 places a step) and sum_d (q - o) and o.
template <int DC>
struct Query {
    v4i h[2 * DC], l[2 * DC];
    int sum, o;
};

// The 16 places of a step that lane holds start at 16 (lane >> 5).
template <int DC>
__device__ inline void load_query(const AttentionArgs& a, const FxSeq& s, int head, int row, int lane, Query<DC>* q) {
    const bool live = row < static_cast<int>(s.count) * a.group;
    const int token = live ? row / a.group : 0, member = live ? row - token * a.group : 0;
    const int16_t* p = a.q + (static_cast<size_t>(s.row) + token) * a.q_stride +
                       (static_cast<size_t>(head) * a.group + member) * a.dim;
    v4i lo[2 * DC], hi[2 * DC];
    int sum = 0, large = 0;
#pragma unroll
    for (int u = 0; u < 2 * DC; ++u) {
        lo[u] = hi[u] = v4i{0, 0, 0, 0};
        if (live) load16(p, u * 32 + 16 * (lane >> 5), a.dim, &lo[u], &hi[u]);
        sum = sum8(hi[u], sum8(lo[u], sum));
        large |= large8(lo[u]) || large8(hi[u]);
    }
    sum += __shfl_xor(sum, 32);
    large |= __shfl_xor(large, 32);
    q->o = large ? 128 : 0;
    q->sum = sum - q->o * 64 * DC;
#pragma unroll
    for (int u = 0; u < 2 * DC; ++u) split16(lo[u], hi[u], q->o, &q->h[u], &q->l[u]);
}

// The three sums of 32 tokens' scores (block `block` of a record's keys) with this
// lane's query: token 8 (r >> 2) + 4 (lane >> 5) + (r & 3) in place r.
struct Raw {
    v16i hh = {}, mid = {}, ll = {};
};

template <int DC>
__device__ inline Raw products(const unsigned char* keys, const Query<DC>& q, int block, int lane) {
    Raw s;
    const v4i* p = reinterpret_cast<const v4i*>(keys) + block * 2 * DC * 128 + lane;
    v4i kh[2 * DC], kl[2 * DC];
#pragma unroll
    for (int u = 0; u < 2 * DC; ++u) kh[u] = p[u * 128], kl[u] = p[u * 128 + 64];
    __builtin_amdgcn_sched_barrier(0);  // all reads first: one wait for LDS, not one a step
#pragma unroll
    for (int u = 0; u < 2 * DC; ++u) {
        s.hh = mfma32(kh[u], q.h[u], s.hh);
        s.mid = mfma32(kh[u], q.l[u], s.mid);
        s.ll = mfma32(kl[u], q.l[u], s.ll);
        s.mid = mfma32(kl[u], q.h[u], s.mid);
    }
    return s;
}

// Scores z, up to a shift of 16.
__device__ inline int score(const Raw& s, int r, uint32_t s1) {
    return (s.hh[r] << (16 - s1)) + (static_cast<int>((static_cast<uint32_t>(s.mid[r]) << 8) + s.ll[r]) >> s1);
}

// Scores z.  `plain`: neither a key of the tile nor a query of the wave has an offset.
template <int DC>
__device__ inline v16i scores(const unsigned char* keys, const int* extra, const Query<DC>& q, int block, int lane,
                              uint32_t s1, uint32_t s2, bool plain) {
    Raw s = products<DC>(keys, q, block, lane);
    if (!plain) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int x = extra[block * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)];
            s.ll[r] = static_cast<int>(static_cast<uint32_t>(s.ll[r]) + static_cast<uint32_t>((x & 128) * q.sum) +
                                       static_cast<uint32_t>((x >> 8) * q.o));
        }
    }
    v16i z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = score(s, r, s1);
    if (s2) {
#pragma unroll
        for (int r = 0; r < 16; ++r) z[r] >>= s2;
    }
    return z;
}

// e (at most 2^14) as its two signed bytes: high in bits 15..8, low in bits 7..0.
__device__ inline uint32_t encoded(uint32_t e) { return halves(static_cast<int>(min(e, 16384u))); }

// Results of a row from its sums, 0 where sum e is 0: a = 2 sum e (v - 128), less
// than 2^50 and so exact in a double.
struct Divide {
    double below, inv, add;
    __device__ explicit Divide(int64_t total)
        : below(2.0 * static_cast<double>(total)), inv(total ? 1.0 / below : 0.0), add(257.0 * static_cast<double>(total)) {}
    __device__ int operator()(double a) const {
        return inv == 0.0 ? 0 : static_cast<int>(floor_div(a + add, below, inv));
    }
};

__device__ inline double twice(int hh, int mid, int ll) {
    return __builtin_fma(hh, 131072.0, __builtin_fma(mid, 512.0, 2.0 * ll));
}

__device__ inline void store4(int16_t* p, int live, const int* v) {
    if (live >= 4) {
        reinterpret_cast<Row8*>(p)->v =
            make_uint2((v[0] & 0xffff) | v[1] << 16, (v[2] & 0xffff) | v[3] << 16);
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (r < live) p[r] = static_cast<int16_t>(v[r]);
    }
}

// Eight entries of the exponential table, encoded.
__device__ inline v4i encoded8(v4i v) {
    typedef unsigned short v2u __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int pair = v[k];
        const v2u e = __builtin_elementwise_min(__builtin_bit_cast(v2u, pair), v2u{16384, 16384});
        const v2u up = e + v2u{128, 128};
        v[k] = (__builtin_bit_cast(int, up) & 0xff00ff00) | (__builtin_bit_cast(int, e) & 0x00ff00ff);
    }
    return v;
}

// The exponential table on its way to LDS, encoded there: loads are under way
// from load() on, so that they cost no wait of their own.
template <int THREADS>
struct Table {
    static constexpr int PIECES = FX_TABLE_MAX / 8 / THREADS;
    v4i piece[PIECES];
    __device__ void load(const uint16_t* from, int entries) {
#pragma unroll
        for (int k = 0; k < PIECES; ++k) {
            const int i = (k * THREADS + static_cast<int>(threadIdx.x)) * 8;
            if (i + 8 <= entries) piece[k] = load8(reinterpret_cast<const int16_t*>(from) + i);
        }
    }
    __device__ void store(const uint16_t* from, int entries, uint16_t* to) {
#pragma unroll
        for (int k = 0; k < PIECES; ++k) {
            const int i = (k * THREADS + static_cast<int>(threadIdx.x)) * 8;
            if (i + 8 <= entries)
                *reinterpret_cast<v4i*>(to + i) = encoded8(piece[k]);
            else
                for (int e = i; e < entries; ++e) to[e] = static_cast<uint16_t>(encoded(from[e]));
        }
    }
};

// Many rows: a workgroup takes 128 rows of a sequence and key head and goes over
// the tiles of 64 tokens twice: for the maximum, then for the sums.  Keys and
// values come to LDS by direct copies, three tiles ahead in the first pass, two
// tiles (DC = 1) or two phases (DC = 2) in the second.
//
// With heads up to 64 (DC = 1) a workgroup is one or two teams of four waves, 32
// rows a wave.  Two teams take the tiles in turn, each with buffers of its own,
// and join their maxima and sums through LDS: where workgroups are few the
// longest one decides, and it is done sooner; elsewhere two workgroups a CU hide
// each other's waits better.  Prompts of 1,024 tokens, 12 heads, us with one team
// and with two: one 42.7 and 32.9, four (384 workgroups) 48.1 and 40.1, six (576)
// 52.9 and 61.3, sixteen 118 and 134.
//
// With heads over 64 (DC = 2) the two waves of a group take 32 tokens of a tile
// each, exchange the exponentials through LDS, and keep half of the result's
// places each: 96 accumulators a lane either way.  The second pass then has two
// phases a tile, scores with exponentials and the sums; the two halves of the
// workgroup run one phase apart, so that a SIMD's two waves are never both at
// the vector work.
//
// Bound by issue and waits together: a score takes about 20 vector instructions, of
// both passes (0.34 of the issue), which overlap with matrix instructions (0.22) only
// in part (a loop of 1,086 cycles of matrix work and one of 1,821 of vector work, on a
// SIMD's two waves, ran 2,330), and waves wait 0.35 of their time, at a barrier for
// each tile and for LDS.  Keys or queries over 32,639 in every tile, whose scores take
// the extras: 16 prompts of 9,450 tokens 69 us where 59 without, 8,192 tokens of 16
// heads of 128 926 and 786.  16 prompts of 10,575 tokens, 12 heads of 64: 74 us, 0.97 POP/s with
// scores counted twice, as they are computed; 8,192 tokens, 16 heads of 128 on 4:
// 800 us, 2.1 POP/s.
template <int DC, int TEAMS>
__global__ __launch_bounds__((256 * DC * TEAMS), 2) void fx_attention_kernel(AttentionArgs a, Seqs q) {
    constexpr int WAVES = 4 * DC;             // of a team
    constexpr bool SHARED = DC * TEAMS == 2;  // two waves have the same rows
    constexpr int PART = Record<DC>::VALUES;       // bytes of a tile's keys, and of its values
    constexpr int PARTS = DC == 1 ? 6 : 4, RING = 4;
    __shared__ __attribute__((aligned(1024))) unsigned char all_parts[TEAMS][PARTS][PART];
    __shared__ __attribute__((aligned(16))) int all_extras[TEAMS][RING][64];
    __shared__ __attribute__((aligned(16))) uint16_t table[FX_TABLE_MAX];
    __shared__ __attribute__((aligned(16))) v4i swap[DC == 2 ? WAVES * 128 : 1];
    __shared__ int share[WAVES * TEAMS][32];
    // heads vary fastest: an XCD gets few of them, and their keys stay in its L2
    uint32_t item = blockIdx.x / static_cast<uint32_t>(a.kv_heads);
    const int lane = threadIdx.x & 63, head = static_cast<int>(blockIdx.x - item * static_cast<uint32_t>(a.kv_heads));
    // The longest work first: first[] holds the sequences' counts of 128 rows,
    // falling; the last such place of all sequences comes first, then the one
    // before it, each with the sequences that reach it.
    uint32_t reach = 0, place = 0;
    for (;; ++reach) {
        const uint32_t here = (q.first[reach] - q.first[reach + 1]) * (reach + 1);
        if (item < here) break;
        item -= here;
    }
    place = q.first[reach] - 1 - item / (reach + 1);
    const FxSeq s = q.s[item % (reach + 1)];
    const int id = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int team = id / WAVES, wave = id % WAVES, group = wave / DC, part = wave % DC;
    auto& parts = all_parts[team];
    auto& extras = all_extras[team];
    const int rows = static_cast<int>(s.count) * a.group;
    const int row0 = static_cast<int>(place) * 128;
    const int row = row0 + group * 32 + (lane & 31);
    const unsigned char* base = a.data + (static_cast<size_t>(s.slot) * a.kv_heads + head) * a.tiles *
                                             static_cast<size_t>(Record<DC>::BYTES);
    const int limit = limit_of(a, s, min(row, rows - 1));
    // what all rows of the wave see, what any of them does, and any of the workgroup's
    const int all = limit_of(a, s, min(row0 + group * 32, rows - 1));
    const int some = row0 + group * 32 < rows ? limit_of(a, s, min(row0 + group * 32 + 31, rows - 1)) : 0;
    const int tiles = (limit_of(a, s, min(row0 + 127, rows - 1)) + FX_TILE - 1) / FX_TILE;

    // A wave's share of a tile's keys with its extras (KEYS instructions), or of its values (VALUES).
    constexpr int VALUES_COPIES = 2, KEYS_COPIES = 3;
    auto stage_keys = [&](int t, unsigned char* to, int* extra) {
        const unsigned char* rec = base + static_cast<size_t>(t) * Record<DC>::BYTES;
        copy_to_lds(rec + wave * 1024, lane * 16, to + wave * 1024);
        copy_to_lds(rec + (WAVES + wave) * 1024, lane * 16, to + (WAVES + wave) * 1024);
        if (lane < 16) copy_to_lds(rec + Record<DC>::EXTRA, lane * 16, extra);  // every wave the same
    };
    auto stage_values = [&](int t, unsigned char* to) {
        const unsigned char* rec = base + static_cast<size_t>(t) * Record<DC>::BYTES + Record<DC>::VALUES;
        copy_to_lds(rec + wave * 1024, lane * 16, to + wave * 1024);
        copy_to_lds(rec + (WAVES + wave) * 1024, lane * 16, to + (WAVES + wave) * 1024);
    };
    // a team's tiles: mine_of(0), mine_of(1), ...; `turns` of them and of the longer team's
    auto mine_of = [&](int i) { return i * TEAMS + team; };
    const int turns = (tiles + TEAMS - 1) / TEAMS;
    Table<64 * WAVES * TEAMS> to_table;
    to_table.load(a.table, static_cast<int>(a.entries));
#pragma unroll
    for (int i = 0; i < RING - 1; ++i)
        if (mine_of(i) < tiles) stage_keys(mine_of(i), parts[i], extras[i]);
    Query<DC> mine;
    load_query<DC>(a, s, head, row, lane, &mine);
    const bool no_offset = !__any(mine.o);
    to_table.store(a.table, static_cast<int>(a.entries), table);
    const uint32_t last = a.entries - 1;
    auto is_plain = [&](int t, const int* extra) {
        return no_offset && !__any(lane + t * FX_TILE < static_cast<int>(s.length) && (extra[lane] & 128));
    };

    int top = INT_MIN;
    for (int i = 0; i < turns; ++i) {
        const int t = mine_of(i);
        if (mine_of(i + RING - 2) < tiles)
            lds_copies_done<(RING - 2) * KEYS_COPIES>();
        else
            lds_copies_done<0>();
        __syncthreads();  // this tile has landed for all waves, and all have left the one before
        if (mine_of(i + RING - 1) < tiles)
            stage_keys(mine_of(i + RING - 1), parts[(i + RING - 1) % RING], extras[(i + RING - 1) % RING]);
        if (TEAMS == 2 && t >= tiles) break;  // the other team's last turn
        const unsigned char* keys = parts[i % RING];
        const int* extra = extras[i % RING];
        const bool plain = is_plain(t, extra);
        if (DC == 1 && plain && a.s2 == 0 && (t + 1) * FX_TILE <= all) {
            // Most tiles, without a branch: one block's vector work beside the other's products.
            const Raw s0 = products<DC>(keys, mine, 0, lane), s1 = products<DC>(keys, mine, 1, lane);
#pragma unroll
            for (int r = 0; r < 16; ++r) top = max(top, score(s0, r, a.s1));
#pragma unroll
            for (int r = 0; r < 16; ++r) top = max(top, score(s1, r, a.s1));
            continue;
        }
#pragma unroll
        for (int b = 0; b < 2 / DC; ++b) {
            const int block = DC == 2 ? part : b, token = t * FX_TILE + block * 32;
            if (token >= some) continue;
            const v16i z = scores<DC>(keys, extra, mine, block, lane, a.s1, a.s2, plain);
            if (token + 32 <= all) {
#pragma unroll
                for (int r = 0; r < 16; ++r) top = max(top, z[r]);
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (token + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3) < limit) top = max(top, z[r]);
            }
        }
    }
    top = max(top, __shfl_xor(top, 32));
    // the other half of the tokens: the other team, or the other wave of the group
    const int other = DC == 1 ? id ^ 4 : id ^ 1;
    if (SHARED && lane < 32) share[id][lane] = top;
    __syncthreads();  // and the first pass's buffers are free
    if (SHARED) top = max(top, share[other][lane & 31]);

    v16i hh[2] = {}, mid[2] = {}, ll[2] = {};  // 32 places each, of this wave's 64
    int sum_h = 0, sum_l = 0;
    // exponentials of 32 tokens with scores z(r), all of which are seen or those below the lane's limit
    auto exponentials = [&](auto&& z, int token, bool whole, v4i* eh, v4i* el) {
        uint32_t e[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) e[r] = table[min(static_cast<uint32_t>(top) - static_cast<uint32_t>(z(r)), last)];
        if (!whole) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (token + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3) >= limit) e[r] = 0;
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
    auto block_exponentials = [&](const unsigned char* keys, const int* extra, int block, int token, bool plain, v4i* eh,
                                  v4i* el) {
        const v16i z = scores<DC>(keys, extra, mine, block, lane, a.s1, a.s2, plain);
        exponentials([&](int r) { return z[r]; }, token, token + 32 <= all, eh, el);
    };
    // the 64 places' values of a block of 32 tokens
    struct Values {
        v4i h[2], l[2];
    };
    auto read = [&](const unsigned char* values, int block) {
        Values v;
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            const v4i* p = reinterpret_cast<const v4i*>(values) + (block * 2 * DC + part * 2 + d) * 128 + lane;
            v.h[d] = p[0];
            v.l[d] = p[64];
        }
        return v;
    };
    auto add = [&](const Values& v, v4i eh, v4i el) {
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            hh[d] = mfma32(v.h[d], eh, hh[d]);
            mid[d] = mfma32(v.h[d], el, mid[d]);
            ll[d] = mfma32(v.l[d], el, ll[d]);
            mid[d] = mfma32(v.l[d], eh, mid[d]);
        }
    };
    if constexpr (DC == 1) {
        constexpr int AHEAD = 2;  // tiles, of three in LDS
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (mine_of(i) < tiles) stage_keys(mine_of(i), parts[2 * i], extras[i]), stage_values(mine_of(i), parts[2 * i + 1]);
        int now = 0;
        auto begin = [&](int i) {
            if (mine_of(i + 1) < tiles)
                lds_copies_done<KEYS_COPIES + VALUES_COPIES>();
            else
                lds_copies_done<0>();
            __syncthreads();
            if (mine_of(i + AHEAD) < tiles) {
                const int next = now == 0 ? 2 : now - 1;
                stage_keys(mine_of(i + AHEAD), parts[2 * next], extras[next]);
                stage_values(mine_of(i + AHEAD), parts[2 * next + 1]);
            }
        };
        // Tiles that all rows see, as long as they need no offset: without branches,
        // the second block's products under way before the first's sums, and its
        // vector work beside them.
        bool begun = false;
        int i = 0;
        for (; i < turns; ++i) {
            begin(i);
            const int t = mine_of(i);
            begun = true;
            if (a.s2 || (t + 1) * FX_TILE > all || !is_plain(t, extras[now])) break;
            v4i eh, el;
            const Raw s0 = products<DC>(parts[2 * now], mine, 0, lane);
            const Values v0 = read(parts[2 * now + 1], 0);
            exponentials([&](int r) { return score(s0, r, a.s1); }, 0, true, &eh, &el);
            const Raw s1 = products<DC>(parts[2 * now], mine, 1, lane);
            add(v0, eh, el);
            const Values v1 = read(parts[2 * now + 1], 1);
            exponentials([&](int r) { return score(s1, r, a.s1); }, 0, true, &eh, &el);
            add(v1, eh, el);
            now = now == 2 ? 0 : now + 1;
            begun = false;
        }
        for (; i < turns; ++i) {
            if (!begun) begin(i);
            begun = false;
            const int t = mine_of(i);
            if (TEAMS == 2 && t >= tiles) break;
            const bool plain = is_plain(t, extras[now]);
#pragma unroll
            for (int block = 0; block < 2; ++block) {
                const int token = t * FX_TILE + block * 32;
                if (token >= some) continue;
                v4i eh, el;
                block_exponentials(parts[2 * now], extras[now], block, token, plain, &eh, &el);
                add(read(parts[2 * now + 1], block), eh, el);
            }
            now = now == 2 ? 0 : now + 1;
        }
    } else {
        // Keys in parts 0 and 1, values in parts 2 and 3.  Phase 2 t has the first
        // half's scores of tile t and the second half's sums of tile t - 1, phase
        // 2 t + 1 the other way round.  At its start keys (even) or values (odd) of
        // tile t + 1 go where those of t - 1 were, which all have left by then;
        // they are waited for two phases later.
        constexpr int COPIES = 3;
        auto stage = [&](int t, int odd) {
            const unsigned char* rec = base + static_cast<size_t>(t) * Record<DC>::BYTES;
            const unsigned char* from = rec + (odd ? Record<DC>::VALUES : 0) + wave * 1024;
            unsigned char* to = parts[2 * odd + (t & 1)] + wave * 1024;
            copy_to_lds(from, lane * 16, to);
            copy_to_lds(from + WAVES * 1024, lane * 16, to + WAVES * 1024);
            if (lane < 16) copy_to_lds(rec + Record<DC>::EXTRA, lane * 16, extras[t & 1]);
        };
        auto begin = [&](int phase) {
            const int t = phase >> 1, odd = phase & 1;
            if (t + odd < tiles)
                lds_copies_done<COPIES>();
            else
                lds_copies_done<0>();
            __syncthreads();
            if (t + 1 < tiles) stage(t + 1, odd);
        };
        if (tiles > 0) stage(0, 0), stage(0, 1);
        const int behind = group >> 1;
        int phase = 0;
        if (behind) begin(phase++);
        for (int t = 0; t < tiles; ++t) {
            begin(phase++);
            const int token = t * FX_TILE + part * 32;
            v4i eh = {}, el = {};
            if (token < some)
                block_exponentials(parts[t & 1], extras[t & 1], part, token, is_plain(t, extras[t & 1]), &eh, &el);
            swap[wave * 128 + lane] = eh;
            swap[wave * 128 + 64 + lane] = el;
            begin(phase++);
            const v4i* p = swap + group * 256 + lane;
            const v4i e0h = p[0], e0l = p[64], e1h = p[128], e1l = p[192];
            const Values v0 = read(parts[2 + (t & 1)], 0), v1 = read(parts[2 + (t & 1)], 1);
            __builtin_amdgcn_sched_barrier(0);
            add(v0, e0h, e0l);
            add(v1, e1h, e1l);
        }
        if (!behind) begin(phase++);
    }
    int total = 256 * sum_h + sum_l;
    total += __shfl_xor(total, 32);
    __syncthreads();
    if (SHARED && lane < 32) share[id][lane] = total;
    if constexpr (TEAMS == 2) {
        // The teams' sums: each gives the other those of 32 places and finishes the rest.
        static_assert(sizeof(all_parts) >= 8 * 48 * 64 * sizeof(int), "room for the exchange");
        int* mail = reinterpret_cast<int*>(all_parts) + lane;
        auto send = [&](const v16i& x, const v16i& y, const v16i& z) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                mail[(id * 48 + r) * 64] = x[r];
                mail[(id * 48 + 16 + r) * 64] = y[r];
                mail[(id * 48 + 32 + r) * 64] = z[r];
            }
        };
        if (team == 0) {
            send(hh[1], mid[1], ll[1]);
        } else {
            send(hh[0], mid[0], ll[0]);
            hh[0] = hh[1], mid[0] = mid[1], ll[0] = ll[1];
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            hh[0][r] += mail[(other * 48 + r) * 64];
            mid[0][r] += mail[(other * 48 + 16 + r) * 64];
            ll[0][r] += mail[(other * 48 + 32 + r) * 64];
        }
    } else {
        __syncthreads();
    }
    if (SHARED) total += share[other][lane & 31];
    if (row >= rows) return;
    const int token = row / a.group, member = row - token * a.group;
    int16_t* out = a.out + (static_cast<size_t>(s.row) + token) * a.out_stride +
                   (static_cast<size_t>(head) * a.group + member) * a.dim;
    const Divide divide(total);
#pragma unroll
    for (int d = 0; d < 2 / TEAMS; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int place = team * 32 + part * 64 + d * 32 + 8 * g + 4 * (lane >> 5);
            if (place >= a.dim) continue;
            int v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = divide(twice(hh[d][4 * g + r], mid[d][4 * g + r], ll[d][4 * g + r]));
            store4(out + place, a.dim - place, v);
        }
}

// ---- few rows ----------------------------------------------------------------------------
// A workgroup takes 16 rows of a sequence and key head and a run of its tiles;
// its waves take the tiles in turn, straight from memory, and add their sums in
// LDS.  Scores are computed once and kept for the second pass, which needs the
// maximum over the whole run:
//   ONE     a tile a wave at most: kept in registers, with the wave's values
//           and the table under way while the scores are computed;
//   FUSED   one workgroup has all tiles: kept in LDS, one launch;
//   SCORES, VALUES   the tiles are split over `splits` workgroups: kept in memory,
//           with a maximum per split, between two launches; a third adds the
//           splits' sums (integers: any order gives the same) and divides.
// Bound by memory, or by the chain of a call where it is short: 64 sequences of up to
// 4,095 tokens, 8 key heads of 128 (639 MB) 135 us, 4.7 TB/s; one of 1,024 tokens, 12
// heads of 64, 10 us, of which a launch and an empty kernel are about 3.
enum Pass { ONE, FUSED, SCORES, VALUES };
constexpr int FEW = 16;

// Waves of a workgroup: ONE has room for 16 with heads up to 64 (128 registers a lane).
template <int DC, Pass PASS>
constexpr int FEW_WAVES = PASS == ONE && DC == 1 ? 16 : 8;

struct FewArgs {
    int cols;       // rows of a unit that scores are kept for, at most FEW
    int max_tiles;  // of a sequence
    int splits;
    int* z;        // units x max_tiles x cols x 64
    int* tops;     // units x splits x FEW
    int64_t* sums;  // units x splits x cols x (head + 1): sum e (v - 128), sum e
};

// A lane's query for 16 x 16 products: row lane & 15, 16 of 64 places from 16 (lane >> 4).
template <int DC>
struct FewQuery {
    v4i h[DC], l[DC];
    int sum, o;
};

template <int DC, Pass PASS>
__global__ __launch_bounds__((64 * FEW_WAVES<DC, PASS>)) void fx_attention_few_kernel(AttentionArgs a, FewArgs f, Seqs q) {
    constexpr int WAVES = FEW_WAVES<DC, PASS>, THREADS = 64 * WAVES;
    extern __shared__ __attribute__((aligned(16))) int kept[];  // FUSED: scores
    __shared__ __attribute__((aligned(16))) uint16_t table[PASS == ONE ? FX_TABLE_MAX : 8];
    __shared__ unsigned long long sums[PASS == SCORES ? 1 : FEW * 64 * DC];
    __shared__ unsigned long long totals[FEW];
    __shared__ int tops[WAVES][FEW];
    const uint32_t item = blockIdx.x / static_cast<uint32_t>(a.kv_heads);
    const uint32_t at = sequence_of(q, item);
    const FxSeq s = q.s[at];
    const int lane = threadIdx.x & 63, head = static_cast<int>(blockIdx.x - item * static_cast<uint32_t>(a.kv_heads));
    const int split = blockIdx.y;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rows = static_cast<int>(s.count) * a.group;
    const int row0 = static_cast<int>(item - q.first[at]) * FEW, row = row0 + (lane & 15);
    const int cols = min(rows - row0, FEW);  // at most f.cols
    const bool mine = (lane & 15) < cols;
    const size_t unit = blockIdx.x;
    const unsigned char* base =
        a.data + (static_cast<size_t>(s.slot) * a.kv_heads + head) * a.tiles * static_cast<size_t>(Record<DC>::BYTES);
    const int limit = limit_of(a, s, min(row, rows - 1));
    const int tiles = (limit_of(a, s, min(row0 + FEW, rows) - 1) + FX_TILE - 1) / FX_TILE;
    const int each = (f.max_tiles + f.splits - 1) / f.splits;
    const int from = split * each, to = min(from + each, tiles);
    const uint32_t last = a.entries - 1;
    int* z_of = PASS == FUSED ? kept : f.z + unit * f.max_tiles * f.cols * 64;
    // this lane's token in place r of its quarter t of a tile: first + 8 t + r
    const int first = 32 * (lane >> 5) + 4 * ((lane >> 4) & 1);
    // where its scores of tile t are kept
    auto z_at = [&](int t) {
        return z_of + ((PASS == FUSED ? t - from : t) * f.cols + (lane & 15)) * 64 + 4 * (lane >> 4);
    };

    // values of a tile: places 16 b + (lane & 15), half (lane >> 4) & 1 of 32-token block lane >> 5
    const int in_values = ((lane >> 5) * 2 * DC) * 128 + (lane & 15) + 32 * ((lane >> 4) & 1);
    struct Values {
        v4i h[4 * DC], l[4 * DC];
    };
    auto read_values = [&](int t, Values* v) {
        const v4i* p = reinterpret_cast<const v4i*>(base + static_cast<size_t>(t) * Record<DC>::BYTES + Record<DC>::VALUES) +
                       in_values;
#pragma unroll
        for (int b = 0; b < 4 * DC; ++b) {
            v->h[b] = p[(b >> 1) * 128 + (b & 1) * 16];
            v->l[b] = p[(b >> 1) * 128 + (b & 1) * 16 + 64];
        }
    };

    int top = INT_MIN;
    v4i z[4] = {};
    Values ahead;
    Table<THREADS> to_table;
    if constexpr (PASS == ONE) {
        if (wave < to) read_values(wave, &ahead);
        to_table.load(a.table, static_cast<int>(a.entries));
    }
    if constexpr (PASS != VALUES) {
        FewQuery<DC> mq;
        {
            const int token = mine ? row / a.group : 0, member = mine ? row - token * a.group : 0;
            const int16_t* p = a.q + (static_cast<size_t>(s.row) + token) * a.q_stride +
                               (static_cast<size_t>(head) * a.group + member) * a.dim;
            v4i lo[DC], hi[DC];
            int sum = 0, large = 0;
#pragma unroll
            for (int c = 0; c < DC; ++c) {
                lo[c] = hi[c] = v4i{0, 0, 0, 0};
                if (mine) load16(p, c * 64 + 16 * (lane >> 4), a.dim, &lo[c], &hi[c]);
                sum = sum8(hi[c], sum8(lo[c], sum));
                large |= large8(lo[c]) || large8(hi[c]);
            }
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            large |= __shfl_xor(large, 16);
            large |= __shfl_xor(large, 32);
            mq.o = large ? 128 : 0;
            mq.sum = sum - mq.o * 64 * DC;
#pragma unroll
            for (int c = 0; c < DC; ++c) split16(lo[c], hi[c], mq.o, &mq.h[c], &mq.l[c]);
        }
        const bool no_offset = !__any(mq.o);
        // the key that this lane reads for row i = lane & 15 of quarter t: 8 t past
        // token 32 (i >> 3) + 4 ((i >> 2) & 1) + (i & 3)
        const int in_tile = (((lane >> 3) & 1) * 2 * DC + (lane >> 5)) * 128 + (lane & 7) + 32 * ((lane >> 4) & 1);
        for (int t = from + wave; t < to; t += WAVES) {
            const unsigned char* rec = base + static_cast<size_t>(t) * Record<DC>::BYTES;
            const v4i* keys = reinterpret_cast<const v4i*>(rec) + in_tile;
            const int* extra = reinterpret_cast<const int*>(rec + Record<DC>::EXTRA);
            const bool offset = lane + t * FX_TILE < static_cast<int>(s.length) && (extra[lane] & 128);
            v4i hh[4] = {}, mid[4] = {}, ll[4] = {};
#pragma unroll
            for (int c = 0; c < DC; ++c)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const v4i kh = keys[c * 256 + k * 8], kl = keys[c * 256 + 64 + k * 8];
                    hh[k] = mfma(kh, mq.h[c], hh[k]);
                    mid[k] = mfma(kh, mq.l[c], mid[k]);
                    ll[k] = mfma(kl, mq.l[c], ll[k]);
                    mid[k] = mfma(kl, mq.h[c], mid[k]);
                }
            if (!no_offset || __any(offset)) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int x = extra[first + 8 * k + r];
                        ll[k][r] = static_cast<int>(static_cast<uint32_t>(ll[k][r]) +
                                                    static_cast<uint32_t>((x & 128) * mq.sum) +
                                                    static_cast<uint32_t>((x >> 8) * mq.o));
                    }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int low = static_cast<int>((static_cast<uint32_t>(mid[k][r]) << 8) + ll[k][r]);
                    z[k][r] = ((hh[k][r] << (16 - a.s1)) + (low >> a.s1)) >> a.s2;
                    if (t * FX_TILE + first + 8 * k + r < limit) top = max(top, z[k][r]);
                }
                if (PASS != ONE && mine) *reinterpret_cast<v4i*>(z_at(t) + 16 * k) = z[k];
            }
        }
        top = max(top, __shfl_xor(top, 16));
        top = max(top, __shfl_xor(top, 32));
        if (lane < FEW) tops[wave][lane] = top;
        if constexpr (PASS == ONE) to_table.store(a.table, static_cast<int>(a.entries), table);
        if constexpr (PASS == SCORES) {
            __syncthreads();
            if (threadIdx.x < FEW) {
                for (int w = 0; w < WAVES; ++w) top = max(top, tops[w][threadIdx.x]);
                f.tops[(unit * f.splits + split) * FEW + threadIdx.x] = top;
            }
            return;
        }
    } else {
        for (int i = 0; i < f.splits; ++i) top = max(top, f.tops[(unit * f.splits + i) * FEW + (lane & 15)]);
    }

    if constexpr (PASS != SCORES) {
        for (int i = threadIdx.x; i < FEW * 64 * DC; i += THREADS) sums[i] = 0;
        if (threadIdx.x < FEW) totals[threadIdx.x] = 0;
        __syncthreads();
        if constexpr (PASS != VALUES)
            for (int w = 0; w < WAVES; ++w) top = max(top, tops[w][lane & 15]);
        v4i hh[4 * DC] = {}, mid[4 * DC] = {}, ll[4 * DC] = {};
        int sum_h = 0, sum_l = 0;
        auto use = [&](int t, const Values& v) {
            v4i eh, el;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t e[4] = {};
                if (mine) {
                    const v4i zk = PASS == ONE ? z[k] : *reinterpret_cast<const v4i*>(z_at(t) + 16 * k);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const uint32_t d = min(static_cast<uint32_t>(top) - static_cast<uint32_t>(zk[r]), last);
                        if (t * FX_TILE + first + 8 * k + r < limit) e[r] = PASS == ONE ? table[d] : encoded(a.table[d]);
                    }
                }
                const uint32_t a01 = e[0] | e[1] << 16, a23 = e[2] | e[3] << 16;
                eh[k] = __builtin_amdgcn_perm(a23, a01, 0x07050301u);
                el[k] = __builtin_amdgcn_perm(a23, a01, 0x06040200u);
                sum_h = __builtin_amdgcn_sdot4(eh[k], 0x01010101, sum_h, false);
                sum_l = __builtin_amdgcn_sdot4(el[k], 0x01010101, sum_l, false);
            }
#pragma unroll
            for (int b = 0; b < 4 * DC; ++b) {
                hh[b] = mfma(v.h[b], eh, hh[b]);
                mid[b] = mfma(v.h[b], el, mid[b]);
                ll[b] = mfma(v.l[b], el, ll[b]);
                mid[b] = mfma(v.l[b], eh, mid[b]);
            }
        };
        if constexpr (PASS == ONE) {
            if (wave < to) use(wave, ahead);
        } else {
            for (int t = from + wave; t < to; t += WAVES) {
                Values v;
                read_values(t, &v);
                use(t, v);
            }
        }
        if (mine) {
            atomicAdd(&totals[lane & 15], static_cast<unsigned long long>(static_cast<int64_t>(256 * sum_h + sum_l)));
#pragma unroll
            for (int b = 0; b < 4 * DC; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    atomicAdd(&sums[(lane & 15) * 64 * DC + 16 * b + 4 * (lane >> 4) + r],
                              static_cast<unsigned long long>(join(hh[b][r], mid[b][r], ll[b][r])));
        }
        __syncthreads();
        if constexpr (PASS == VALUES) {
            constexpr int WIDTH = 64 * DC + 1;
            int64_t* kept_sums = f.sums + (unit * f.splits + split) * f.cols * WIDTH;
            for (int i = threadIdx.x; i < cols * 64 * DC; i += THREADS)
                kept_sums[i / (64 * DC) * WIDTH + i % (64 * DC)] = static_cast<int64_t>(sums[i]);
            if (threadIdx.x < cols)
                kept_sums[threadIdx.x * WIDTH + 64 * DC] = static_cast<int64_t>(totals[threadIdx.x]);
            return;
        }
        // four places a thread
        for (int i = threadIdx.x; i < cols * 16 * DC; i += THREADS) {
            const int col = i / (16 * DC), place = i % (16 * DC) * 4;
            if (place >= a.dim) continue;
            const int token = (row0 + col) / a.group, member = row0 + col - token * a.group;
            int v[4];
            const Divide divide(static_cast<int64_t>(totals[col]));
#pragma unroll
            for (int r = 0; r < 4; ++r)
                v[r] = divide(2.0 * static_cast<double>(static_cast<int64_t>(sums[col * 64 * DC + place + r])));
            store4(a.out + (static_cast<size_t>(s.row) + token) * a.out_stride +
                       (static_cast<size_t>(head) * a.group + member) * a.dim + place,
                   a.dim - place, v);
        }
    }
}

// The splits' sums of a unit, added and divided: a workgroup a unit, four places a thread.
// A launch of its own: the last split to arrive doing it, after a fence and an atomic
// count, cost more than the 4 us that this launch does.
template <int DC>
__global__ __launch_bounds__(256) void fx_attention_join_kernel(AttentionArgs a, FewArgs f, Seqs q) {
    constexpr int WIDTH = 64 * DC + 1;
    const uint32_t item = blockIdx.x / static_cast<uint32_t>(a.kv_heads);
    const uint32_t at = sequence_of(q, item);
    const FxSeq s = q.s[at];
    const int head = static_cast<int>(blockIdx.x - item * static_cast<uint32_t>(a.kv_heads));
    const int row0 = static_cast<int>(item - q.first[at]) * FEW;
    const int cols = min(static_cast<int>(s.count) * a.group - row0, FEW);
    for (int i = threadIdx.x; i < cols * 16 * DC; i += 256) {
        const int col = i / (16 * DC), place = i % (16 * DC) * 4;
        if (place >= a.dim) continue;
        const int64_t* p = f.sums + (static_cast<size_t>(blockIdx.x) * f.splits * f.cols + col) * WIDTH;
        int64_t total = 0, sums[4] = {};
        for (int k = 0; k < f.splits; ++k, p += f.cols * WIDTH) {
            total += p[64 * DC];
#pragma unroll
            for (int r = 0; r < 4; ++r) sums[r] += p[place + r];
        }
        const Divide divide(total);
        int v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = divide(2.0 * static_cast<double>(sums[r]));
        const int token = (row0 + col) / a.group, member = row0 + col - token * a.group;
        store4(a.out + (static_cast<size_t>(s.row) + token) * a.out_stride +
                   (static_cast<size_t>(head) * a.group + member) * a.dim + place,
               a.dim - place, v);
    }
}

// Sequences in groups of FX_SEQS with work items counted by `items`; one launch each.
template <class Items, class Launch>
int each_group(Context* c, const FxSeq* seqs, size_t count, Items&& items, Launch&& launch) {
    for (size_t at = 0; at < count; at += FX_SEQS) {
        Seqs q{};
        uint32_t total = 0;
        for (size_t i = at; i < count && i < at + FX_SEQS; ++i) {
            q.first[q.count] = total;
            q.s[q.count++] = seqs[i];
            total += items(seqs[i]);
        }
        q.first[q.count] = total;
        if (!total) continue;
        launch(q, total);
        VMX_HIP(c, hipGetLastError());
    }
    return 0;
}

template <int DC>
int launch_few(Context* c, const AttentionArgs& a, const FewArgs& f, const FxSeq* seqs, size_t count, Pass pass) {
    return each_group(
        c, seqs, count, [&](const FxSeq& s) { return (s.count * a.group + FEW - 1) / FEW; },
        [&](const Seqs& q, uint32_t total) {
            const dim3 grid(total * static_cast<unsigned>(a.kv_heads), static_cast<unsigned>(f.splits));
            if (pass == ONE) {
                hipLaunchKernelGGL((fx_attention_few_kernel<DC, ONE>), grid, dim3(64 * FEW_WAVES<DC, ONE>), 0, c->stream,
                                   a, f, q);
            } else if (pass == FUSED) {
                hipLaunchKernelGGL((fx_attention_few_kernel<DC, FUSED>), grid, dim3(64 * FEW_WAVES<DC, FUSED>),
                                   static_cast<unsigned>(f.max_tiles * f.cols * 256), c->stream, a, f, q);
            } else {
                hipLaunchKernelGGL((fx_attention_few_kernel<DC, SCORES>), grid, dim3(64 * FEW_WAVES<DC, SCORES>), 0,
                                   c->stream, a, f, q);
                hipLaunchKernelGGL((fx_attention_few_kernel<DC, VALUES>), grid, dim3(64 * FEW_WAVES<DC, VALUES>), 0,
                                   c->stream, a, f, q);
                hipLaunchKernelGGL(fx_attention_join_kernel<DC>, dim3(grid.x), dim3(256), 0, c->stream, a, f, q);
            }
        });
}

// Space for the scores and sums of the sequences of a launch.  One sequence of up to 16
// rows may take more, but no more than a quarter of its cache: 4 bytes a row and token,
// of 260 that a token takes there.
constexpr size_t SPLIT_MAX = size_t{512} << 20;

// *no_space, with nothing launched, where its space may not grow: the other kernel
// needs none.  What is returned is an error, of whatever sign, or 0.
int few_rows(Context* c, const AttentionArgs& a, std::vector<FxSeq>& seqs, size_t tiles, size_t cols, bool* no_space) {
    std::sort(seqs.begin(), seqs.end(), [](const FxSeq& x, const FxSeq& y) { return x.length > y.length; });
    auto units_of = [&](const FxSeq& s) { return (size_t{s.count} * a.group + FEW - 1) / FEW * a.kv_heads; };
    // Ends of the launches, in order of at most `most` units each, or of one sequence:
    // a launch reuses the space of the one before, as they run in order.
    std::vector<size_t> ends;
    size_t units = 0;  // of the largest launch
    auto divide = [&](size_t most) {
        ends.clear();
        units = 0;
        for (size_t at = 0, end = 0; at < seqs.size(); at = end) {
            size_t here = 0;
            do here += units_of(seqs[end++]);
            while (end < seqs.size() && end - at < FX_SEQS && here + units_of(seqs[end]) <= most);
            ends.push_back(end);
            units = std::max(units, here);
        }
    };
    divide(SIZE_MAX);
    FewArgs f{};
    f.cols = static_cast<int>(cols);
    f.max_tiles = static_cast<int>(std::max<size_t>(tiles, 1));
    f.splits = 1;
    const size_t score_bytes = f.max_tiles * cols * 256;
    // us, one token a sequence, for units x tiles with heads of 64 (of 128):
    //   units x tiles       ONE        FUSED        split
    //   12 x 4              8.8        8.4 (10.9)   15.1
    //   12 x 16             9.9        12.5         15.7
    //   192 x 16            13.9       17.8         23.9
    //   512 x 16            30.7       27.4         39.1
    //   12 x 32                        19.9 (25.0)  16.8 (18.3)
    //   192 x 32                       28.1 (40.2)  43.1 (66.0)
    //   12 x 128                       73.0 (96.7)  21.8 (26.5)
    //   192 x 128                      112 (184)    133 (246)
    // ONE, with heads over 64, is 0.3 to 2 us ahead of FUSED up to its 8 tiles.
    // Two launches more cost 10 us; what they save is a tile's time alone on a CU,
    // 0.55 us (0.75), less its share of the whole card's, 5 ns (9) a unit.  Scores of
    // up to 64 KiB are kept.  That limit is low for many units of heads over 64: one
    // token each of 64 sequences of 4,097, 32 heads of 128 on 8, takes 278 us split and
    // 218 kept in 65 KiB (4,096 tokens: 143), of 8,192 563 and 458; of 16 sequences of
    // 8,192, 163 and 162; with heads of 64, 406 both.
    const bool wide = a.dim > 64;
    const int64_t alone = wide ? 750 : 550, shared = wide ? 9 : 5;
    Pass pass = SCORES;
    if (wide ? tiles <= FEW_WAVES<2, ONE> : tiles > 4 && tiles <= FEW_WAVES<1, ONE> && units <= static_cast<size_t>(c->cu_count))
        pass = ONE;
    else if (score_bytes <= 65536 &&
             static_cast<int64_t>(tiles) * (alone - shared * static_cast<int64_t>(units)) <= 10000)
        pass = FUSED;
    if (pass == SCORES) {
        // splits of all units: 2 x CUs and one a unit at most
        const size_t split_bytes = cols * (a.dim <= 64 ? 65 : 129) * 8 + FEW * 4;
        divide((SPLIT_MAX - 2 * c->cu_count * split_bytes) / (score_bytes + split_bytes));
        const size_t want = (2 * c->cu_count + units - 1) / units, most = (tiles + 7) / 8;
        f.splits = static_cast<int>(std::max<size_t>(1, std::min(want, most)));
        const size_t z = units * score_bytes, sums = units * f.splits * (split_bytes - FEW * 4);
        *no_space = !try_ws(c, WS_FIXED, workspace_step(z + units * f.splits * split_bytes, SPLIT_MAX));
        if (*no_space) return 0;
        f.z = ws<int>(c, WS_FIXED);
        f.sums = reinterpret_cast<int64_t*>(ws<unsigned char>(c, WS_FIXED) + z);
        f.tops = reinterpret_cast<int*>(ws<unsigned char>(c, WS_FIXED) + z + sums);
    }
    for (size_t at = 0, i = 0; i < ends.size(); at = ends[i++]) {
        const FxSeq* first = seqs.data() + at;
        if (a.dim <= 64 ? launch_few<1>(c, a, f, first, ends[i] - at, pass) : launch_few<2>(c, a, f, first, ends[i] - at, pass))
            return -1;
    }
    return 0;
}

}  // namespace

int fx_kv_append(Context* c, const FxCache& cache, const int16_t* k, size_t k_stride, const int16_t* v, size_t v_stride,
                 const FxSeq* seqs, size_t count) {
    const AppendArgs a{cache.data, cache.kv_heads, fx_tiles(cache.capacity), static_cast<int>(cache.dim),
                       k,          v,              k_stride,                 v_stride};
    return each_group(
        c, seqs, count,
        [](const FxSeq& s) { return s.count ? (s.length - 1) / FX_TILE - (s.length - s.count) / FX_TILE + 1 : 0; },
        [&](const Seqs& q, uint32_t total) {
            const dim3 grid(total, static_cast<unsigned>(cache.kv_heads));
            if (cache.dim <= 64)
                hipLaunchKernelGGL(fx_append_kernel<1>, grid, dim3(256), 0, c->stream, a, q);
            else
                hipLaunchKernelGGL(fx_append_kernel<2>, grid, dim3(256), 0, c->stream, a, q);
        });
}

int fx_attention(Context* c, const FxCache& cache, const FxAttention& t, const FxSeq* seqs, size_t count) {
    const uint32_t group = t.heads / static_cast<uint32_t>(cache.kv_heads);
    const uint32_t s1 = t.shift < 16 ? t.shift : 16;
    const AttentionArgs a{cache.data,
                          cache.kv_heads,
                          fx_tiles(cache.capacity),
                          t.q,
                          t.q_stride,
                          t.out,
                          t.out_stride,
                          t.table,
                          static_cast<int>(cache.dim),
                          static_cast<int>(group),
                          t.entries,
                          s1,
                          t.shift - s1,
                          t.causal};
    // Where many rows leave CUs idle, the kernel for few rows, which splits the
    // tiles, is faster.  Estimates in ns from measurements (rows x tokens, heads
    // of 128 on 4 key heads): 32 x 8,192 268 us by rows and 40 by tiles, 512 x
    // 8,192 368 and 92, eight of 128 x 4,096 191 and 96, 16 of 64 x 2,048 on 8
    // key heads 78 and 96, one prompt of 4,096 190 and more than that.
    auto rows_of = [&](const FxSeq& s) { return size_t{s.count} * group; };
    auto tiles_of = [&](const FxSeq& s) {  // of a middle row
        return static_cast<double>(s.length - (t.causal ? s.count / 2 : 0)) / FX_TILE + 1;
    };
    double by_rows = 0, by_tiles = 0, longest = 0;
    size_t tiles = 0, units = 0, workgroups = 0;
    for (size_t i = 0; i < count; ++i) {
        const FxSeq& s = seqs[i];
        tiles = std::max<size_t>(tiles, (s.length + FX_TILE - 1) / FX_TILE);
        units += (rows_of(s) + FEW - 1) / FEW * cache.kv_heads;
        if (rows_of(s) <= FEW) continue;
        by_rows += static_cast<double>((rows_of(s) + 127) / 128 * cache.kv_heads) * tiles_of(s) * 11;
        by_tiles += static_cast<double>((rows_of(s) + FEW - 1) / FEW * cache.kv_heads) * tiles_of(s) * 5;
        longest = std::max(longest, (s.length + FX_TILE - 1) / FX_TILE * (cache.dim <= 64 ? 1500.0 : 2200.0));
    }
    const bool split = by_tiles + 5000 < std::max(by_rows, longest) && units * tiles * FEW * 256 <= size_t{1} << 29;
    std::vector<FxSeq> many, few;
    size_t cols = 0;
    tiles = 0;
    for (size_t i = 0; i < count; ++i) {
        const FxSeq& s = seqs[i];
        if (rows_of(s) > FEW && !split) {
            many.push_back(s);
            workgroups += (rows_of(s) + 127) / 128 * cache.kv_heads;
            continue;
        }
        few.push_back(s);
        tiles = std::max<size_t>(tiles, (s.length + FX_TILE - 1) / FX_TILE);
        cols = std::max<size_t>(cols, std::min<size_t>(rows_of(s), FEW));
    }
    if (!few.empty()) {
        bool no_space = false;
        if (few_rows(c, a, few, tiles, cols, &no_space)) return -1;
        if (no_space) {
            many.assign(seqs, seqs + count);
            workgroups = SIZE_MAX;
        }
    }
    auto items = [&](const FxSeq& s) { return (s.count * group + 127) / 128; };
    std::sort(many.begin(), many.end(), [&](const FxSeq& x, const FxSeq& y) { return items(x) > items(y); });
    return each_group(
        c, many.data(), many.size(), items, [&](Seqs& q, uint32_t total) {
            for (uint32_t i = 0; i < q.count; ++i) q.first[i] = items(q.s[i]);
            q.first[q.count] = 0;
            const dim3 grid(total * static_cast<unsigned>(cache.kv_heads));
            if (cache.dim > 64)
                hipLaunchKernelGGL((fx_attention_kernel<2, 1>), grid, dim3(512), 0, c->stream, a, q);
            else if (workgroups <= 2 * static_cast<size_t>(c->cu_count))
                hipLaunchKernelGGL((fx_attention_kernel<1, 2>), grid, dim3(512), 0, c->stream, a, q);
            else
                hipLaunchKernelGGL((fx_attention_kernel<1, 1>), grid, dim3(256), 0, c->stream, a, q);
        });
}

}  // namespace vmx
