// fixed_attention.hpp -- what the attention kernels share: sequences as kernel
// arguments, records of the cache, queries, scores, exponentials and quotients
// (the mathematics is at the head of fixed_attention.hip).
#pragma once

#include "fixed.hpp"

namespace vmx {
namespace fx {

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
    int window, sinks;             // WINDOW
    uint32_t prefix_slot, prefix;  // PREFIX: its tokens
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

// The query at p (nothing if not `live`).  The 16 places of a step that lane holds start
// at 16 (lane >> 5).
template <int DC>
__device__ inline void load_query(const int16_t* p, bool live, int dim, int lane, Query<DC>* q) {
    v4i lo[2 * DC], hi[2 * DC];
    int sum = 0, large = 0;
#pragma unroll
    for (int u = 0; u < 2 * DC; ++u) {
        lo[u] = hi[u] = v4i{0, 0, 0, 0};
        if (live) load16(p, u * 32 + 16 * (lane >> 5), dim, &lo[u], &hi[u]);
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

// That of row `row` of a sequence.
template <int DC>
__device__ inline void load_query(const AttentionArgs& a, const FxSeq& s, int head, int row, int lane, Query<DC>* q) {
    const bool live = row < static_cast<int>(s.count) * a.group;
    const int token = live ? row / a.group : 0, member = live ? row - token * a.group : 0;
    load_query<DC>(a.q + (static_cast<size_t>(s.row) + token) * a.q_stride +
                       (static_cast<size_t>(head) * a.group + member) * a.dim,
                   live, a.dim, lane, q);
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

// Scores z of block `block` from its sums.  `plain`: neither a key of the tile nor a query of
// the wave has an offset.
template <int DC>
__device__ inline v16i scores(Raw s, const int* extra, const Query<DC>& q, int block, int lane, uint32_t s1, uint32_t s2,
                              bool plain) {
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

template <int DC>
__device__ inline v16i scores(const unsigned char* keys, const int* extra, const Query<DC>& q, int block, int lane,
                              uint32_t s1, uint32_t s2, bool plain) {
    return scores<DC>(products<DC>(keys, q, block, lane), extra, q, block, lane, s1, s2, plain);
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

inline AttentionArgs attention_args(const FxCache& cache, const FxAttention& t) {
    const uint32_t s1 = t.shift < 16 ? t.shift : 16;
    return AttentionArgs{cache.data,
                         cache.kv_heads,
                         fx_tiles(cache.capacity),
                         t.q,
                         t.q_stride,
                         t.out,
                         t.out_stride,
                         t.table,
                         static_cast<int>(cache.dim),
                         static_cast<int>(t.heads / cache.kv_heads),
                         t.entries,
                         s1,
                         t.shift - s1,
                         t.causal,
                         static_cast<int>(t.window < FX_CACHE_MAX ? t.window : FX_CACHE_MAX),
                         static_cast<int>(t.sinks < FX_CACHE_MAX ? t.sinks : FX_CACHE_MAX),
                         t.prefix_slot,
                         t.prefix};
}

}  // namespace fx
}  // namespace vmx
