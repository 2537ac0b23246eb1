// fixed_attention.hip -- attention over a cache of keys and values in 16-bit
// integers, and the cache's append (layout in fixed.hpp).
//
// z = (q . k) >> shift, d = max_j z - z, e = table[min(d, entries - 1)],
// out = sum e v / sum e rounded to the nearest integer, halves up.  The maximum
// runs over the keys a query may see, and a query without any gives zeros.
//
// Rows of a launch are the pairs (token, query head) of one key head's group,
// so grouped heads share the keys and values that a wave reads.  Scores are
// computed transposed, S^T = K Q^T: a lane then holds scores of one query only,
// its statistics are one register, and the exponentials are already in the
// layout in which O^T = V^T E^T reads them.
//
// 16-bit scores from four i8 products, as in fixed.hpp; s - 2^16 sum qh kh fits
// 32 bits for heads of up to 128, so z = (hh << 16 - s1) + (c >> s1) >> s2 with
// s1 = min(shift, 16) never needs 64-bit arithmetic.  e (at most 2^14) is
// 256 h + l with signed bytes, so sum e v needs no correction but
// 128 sum e for the values' low bytes.
#include "fixed.hpp"

#include <climits>

namespace vmx {
namespace {

using namespace fx;

struct Seqs {
    FxSeq s[FX_SEQS];
    uint32_t first[FX_SEQS + 1];  // work items before each sequence
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

template <int DC>
constexpr size_t RECORD = DC * 16384 + 256;

// ---- append ---------------------------------------------------------------------------
// One workgroup per (key head, 64-token tile that new tokens touch).
struct AppendArgs {
    unsigned char* data;
    size_t kv_heads, tiles;
    int dim;
    const int16_t *k, *v;
    size_t k_stride, v_stride;
};

template <int DC>
__global__ __launch_bounds__(256) void fx_append_kernel(AppendArgs a, Seqs q) {
    constexpr int DP = DC * 64;
    const uint32_t at = sequence_of(q, blockIdx.x);
    const FxSeq s = q.s[at];
    const int past = static_cast<int>(s.length - s.count);
    const int tile = past / FX_TILE + static_cast<int>(blockIdx.x - q.first[at]);
    const int head = blockIdx.y;
    unsigned char* rec = a.data + ((static_cast<size_t>(s.slot) * a.kv_heads + head) * a.tiles + tile) * RECORD<DC>;
    unsigned char* keys = rec;
    unsigned char* values = rec + DP * 128;
    int* offs = reinterpret_cast<int*>(rec + DP * 256);
    const int from = max(past - tile * FX_TILE, 0), to = min(static_cast<int>(s.length) - tile * FX_TILE, FX_TILE);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int j = from + wave; j < to; j += 4) {
        const size_t row = s.row + (tile * FX_TILE + j - past);
        const int16_t* k = a.k + row * a.k_stride + static_cast<size_t>(head) * a.dim;
        const int16_t* v = a.v + row * a.v_stride + static_cast<size_t>(head) * a.dim;
        int sum = 0;
#pragma unroll
        for (int c = 0; c < DC; ++c) {
            const int d = c * 64 + lane;
            const int kd = d < a.dim ? k[d] : 0, vd = d < a.dim ? v[d] : 0;
            sum += kd;
            unsigned char* pk = keys + (((j >> 4) * DC + c) * 2) * 1024 + ((j & 15) + 16 * (lane >> 4)) * 16 + (lane & 15);
            pk[0] = static_cast<unsigned char>(kd >> 8);
            pk[1024] = static_cast<unsigned char>(kd ^ 0x80);
            unsigned char* pv = values + (d >> 4) * 2048 + ((d & 15) + 16 * ((j & 15) >> 2)) * 16 + (j >> 4) * 4 + (j & 3);
            pv[0] = static_cast<unsigned char>(vd >> 8);
            pv[1024] = static_cast<unsigned char>(vd ^ 0x80);
        }
        for (int m = 32; m; m >>= 1) sum += __shfl_xor(sum, m);
        if (lane == 0) offs[j] = 128 * sum;
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

// A lane's query: its planes along d and 128 sum_d (q - 128).
template <int DC>
struct Query {
    v4i h[DC], l[DC];
    int offset;
    int limit;  // keys it may see
};

template <int DC>
__device__ inline void load_query(const AttentionArgs& a, const FxSeq& s, int head, int row, int lane, Query<DC>* q) {
    const int rows = static_cast<int>(s.count) * a.group;
    const bool live = row < rows;
    const int token = live ? row / a.group : 0, member = live ? row - token * a.group : 0;
    const int16_t* p = a.q + (static_cast<size_t>(s.row) + token) * a.q_stride +
                       (static_cast<size_t>(head) * a.group + member) * a.dim;
    int sum = 0;
#pragma unroll
    for (int c = 0; c < DC; ++c) {
        v4i x0 = {}, x1 = {};
        if (live) load16(p, c * 64 + 16 * (lane >> 4), a.dim, &x0, &x1);
        sum = sum8(x1, sum8(x0, sum));
        split16(x0, x1, &q->h[c], &q->l[c]);
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    q->offset = 128 * sum - 16384 * 64 * DC;
    const int length = static_cast<int>(s.length);
    q->limit = !live ? 0 : a.causal ? length - static_cast<int>(s.count) + token + 1 : length;
}

// Scores z of the 16 tokens of a subtile (this lane: tokens 4 (lane >> 4) .. + 3).
template <int DC>
__device__ inline v4i scores(const v4i* keys, const int* offs, const Query<DC>& q, int sub, int lane, uint32_t s1,
                             uint32_t s2) {
    v4i hh = {}, mid = {}, ll = *reinterpret_cast<const v4i*>(offs + sub * 16 + 4 * (lane >> 4));
#pragma unroll
    for (int c = 0; c < DC; ++c) {
        const v4i kh = keys[(sub * DC + c) * 128 + lane], kl = keys[(sub * DC + c) * 128 + 64 + lane];
        hh = mfma(kh, q.h[c], hh);
        mid = mfma(kh, q.l[c], mid);
        ll = mfma(kl, q.l[c], ll);
        mid = mfma(kl, q.h[c], mid);
    }
    v4i z;
#pragma unroll
    for (int r = 0; r < 4; ++r)
        z[r] = ((hh[r] << (16 - s1)) + ((static_cast<int>((static_cast<uint32_t>(mid[r]) << 8) + ll[r] + q.offset)) >> s1)) >> s2;
    return z;
}

// e (at most 2^14) as its two signed bytes: high in bits 15..8, low in bits 7..0.
__device__ inline uint32_t encoded(uint32_t e) { return (min(e, 16384u) + 128) ^ 128; }

template <int DC>
__device__ inline void store_out(const AttentionArgs& a, const FxSeq& s, int head, int row, int d, const int64_t* sums,
                                 int64_t total) {
    if (row >= static_cast<int>(s.count) * a.group) return;
    const int token = row / a.group, member = row - token * a.group;
    int16_t* p = a.out + (static_cast<size_t>(s.row) + token) * a.out_stride +
                 (static_cast<size_t>(head) * a.group + member) * a.dim + d;
    const double below = 2.0 * static_cast<double>(total), inv = total ? 1.0 / below : 0.0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (d + r >= a.dim) break;
        const double num = static_cast<double>(2 * (sums[r] + 128 * total) + total);
        p[r] = total ? static_cast<int16_t>(floor_div(num, below, inv)) : 0;
    }
}

// One wave per 16 rows, one pass for the maximum and one for the sums.
template <int DC>
__global__ __launch_bounds__(256) void fx_attention_kernel(AttentionArgs a, Seqs q) {
    const uint32_t at = sequence_of(q, blockIdx.x);
    const FxSeq s = q.s[at];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, head = blockIdx.y;
    const int row = static_cast<int>(blockIdx.x - q.first[at]) * 64 + wave * 16 + (lane & 15);
    const unsigned char* base = a.data + (static_cast<size_t>(s.slot) * a.kv_heads + head) * a.tiles * RECORD<DC>;
    Query<DC> mine;
    load_query<DC>(a, s, head, row, lane, &mine);
    int last = mine.limit;
    for (int m = 32; m; m >>= 1) last = max(last, __shfl_xor(last, m));
    const int tiles = (last + FX_TILE - 1) / FX_TILE;

    int top = INT_MIN;
    for (int t = 0; t < tiles; ++t) {
        const unsigned char* rec = base + static_cast<size_t>(t) * RECORD<DC>;
#pragma unroll
        for (int sub = 0; sub < 4; ++sub) {
            const v4i z = scores<DC>(reinterpret_cast<const v4i*>(rec), reinterpret_cast<const int*>(rec + DC * 16384),
                                     mine, sub, lane, a.s1, a.s2);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (t * FX_TILE + sub * 16 + 4 * (lane >> 4) + r < mine.limit) top = max(top, z[r]);
        }
    }
    top = max(top, __shfl_xor(top, 16));
    top = max(top, __shfl_xor(top, 32));

    v4i hh[DC * 4] = {}, mid[DC * 4] = {}, ll[DC * 4] = {};
    int sum_h = 0, sum_l = 0;
    for (int t = 0; t < tiles; ++t) {
        const unsigned char* rec = base + static_cast<size_t>(t) * RECORD<DC>;
        v4i eh, el;
#pragma unroll
        for (int sub = 0; sub < 4; ++sub) {
            const v4i z = scores<DC>(reinterpret_cast<const v4i*>(rec), reinterpret_cast<const int*>(rec + DC * 16384),
                                     mine, sub, lane, a.s1, a.s2);
            uint32_t e[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const bool seen = t * FX_TILE + sub * 16 + 4 * (lane >> 4) + r < mine.limit;
                const uint32_t d = min(static_cast<uint32_t>(top) - static_cast<uint32_t>(z[r]), a.entries - 1);
                e[r] = seen ? encoded(a.table[d]) : 0;
            }
            const uint32_t a01 = e[0] | e[1] << 16, a23 = e[2] | e[3] << 16;
            eh[sub] = __builtin_amdgcn_perm(a23, a01, 0x07050301u);
            el[sub] = __builtin_amdgcn_perm(a23, a01, 0x06040200u);
            sum_h = __builtin_amdgcn_sdot4(eh[sub], 0x01010101, sum_h, false);
            sum_l = __builtin_amdgcn_sdot4(el[sub], 0x01010101, sum_l, false);
        }
        const v4i* values = reinterpret_cast<const v4i*>(rec + DC * 8192) + lane;
#pragma unroll
        for (int b = 0; b < DC * 4; ++b) {
            const v4i vh = values[b * 128], vl = values[b * 128 + 64];
            hh[b] = mfma(vh, eh, hh[b]);
            mid[b] = mfma(vh, el, mid[b]);
            ll[b] = mfma(vl, el, ll[b]);
            mid[b] = mfma(vl, eh, mid[b]);
        }
    }
    int total = 256 * sum_h + sum_l;
    total += __shfl_xor(total, 16);
    total += __shfl_xor(total, 32);
#pragma unroll
    for (int b = 0; b < DC * 4; ++b) {
        int64_t sums[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) sums[r] = join(hh[b][r], mid[b][r], ll[b][r]);
        store_out<DC>(a, s, head, row, b * 16 + 4 * (lane >> 4), sums, total);
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
    return each_group(
        c, seqs, count, [&](const FxSeq& s) { return (s.count * group + 63) / 64; },
        [&](const Seqs& q, uint32_t total) {
            const dim3 grid(total, static_cast<unsigned>(cache.kv_heads));
            if (cache.dim <= 64)
                hipLaunchKernelGGL(fx_attention_kernel<1>, grid, dim3(256), 0, c->stream, a, q);
            else
                hipLaunchKernelGGL(fx_attention_kernel<2>, grid, dim3(256), 0, c->stream, a, q);
        });
}

}  // namespace vmx
