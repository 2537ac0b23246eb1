// fixed_choose.hip -- the next token of each row of i64 logits: penalties for the
// tokens of its history, biases, a mask of what is allowed, and the largest.
//
// For a token that occurs n > 0 times in the row's history, with r = repetition
// at 2^-16: l = l r / 2^16 (l < 0) or l 2^16 / r (l >= 0), to the nearest integer,
// halves up, less frequency n + presence.  Then l += (sum of the token's biases)
// << bias_shift, all exact, clamped to [-2^63 + 1, 2^63 - 1] once; a token that is
// not allowed gets -2^63.  The choice is the lowest index of the largest allowed
// l, -1 where nothing is allowed.  Sums of integers and a maximum with the index as
// its tie-break: no order of threads or workgroups changes a result.
//
// A workgroup takes a chunk of a row's vocabulary.  It counts the history's entries that
// fall into it in LDS, 15 bits a token (31 behind histories that need them), and goes over
// its logits once.  Few tokens are in a list, but nearly every 64 hold one: a wave queues
// those with their logits and changes 64 at a time, all lanes at work.  (In place, all waves
// went through the arithmetic; in a second pass over the lists their logits came from memory
// again.  256 rows of 50,257, 6,100 tokens of history each, the same in each launch: 50 and 48
// us, 35 by the queue, 110 MB at 3.1 TB/s.  The call takes 42 to 43 us on the same logits, which
// the last-level cache holds, and 48 to 49 on others.)  The sum of a token's biases is in a hash
// table in LDS, which a bit beside the count says to look into.  A second launch joins the
// chunks' best.  Where no workspace may grow, a workgroup takes a row, with a count and a sum for
// each token of a small chunk at a time.
#include <algorithm>
#include <climits>

#include "fixed.hpp"

namespace vmx {
namespace {

using namespace fx;

constexpr int DENSE = 2048;            // tokens of a chunk with wide counts and sums
// A chunk's lists in LDS: occurrences of its tokens, each with a bit that says that it has
// biases, and a table of the biases' sums.  Short lists have two tokens a word and a small table.
template <bool WIDE>
struct Lists {
    static constexpr uint32_t BIASED = WIDE ? 1u << 31 : 0x8000, MOST = BIASED - 1;
    static constexpr uint32_t CHUNK = (WIDE ? 20 : 56) * 1024;  // tokens of a chunk, at most
    // Half of the slots hold all biases of a row, or, where those are more, those of a chunk
    // of FEW tokens.
    static constexpr uint32_t BITS = WIDE ? 12 : 10, SLOTS = 1u << BITS, BIASES = SLOTS / 2, FEW = SLOTS / 16 * 11;
    __device__ static uint32_t slot_of(uint32_t token) { return (token * 0x9e3779b1u) >> (32 - BITS); }
    __device__ static uint32_t word(uint32_t t) { return WIDE ? t : t >> 1; }
    __device__ static uint32_t shift(uint32_t t) { return WIDE ? 0 : 16 * (t & 1); }
    __device__ static uint32_t of(const uint32_t* counts, uint32_t t) {
        return WIDE ? counts[t] : counts[t >> 1] >> (16 * (t & 1)) & 0xffff;
    }
    // of t and t + 1, t even
    __device__ static uint2 two(const uint32_t* counts, uint32_t t) {
        if constexpr (WIDE) return *reinterpret_cast<const uint2*>(counts + t);
        return make_uint2(counts[t >> 1] & 0xffff, counts[t >> 1] >> 16);
    }
};
constexpr int THREADS = 1024, PAIRS = 4;           // pairs of logits of a thread on their way

struct Settings {
    FxChoice row[FX_CHOICES];
};

// A candidate: INT64_MIN and -1 where there is none.
struct Best {
    int64_t value;
    int32_t token;
    int32_t reserved;
};

struct __attribute__((packed, aligned(8))) Pair {
    int64_t v[2];
};
struct __attribute__((packed, aligned(4))) Four {
    v4i v;
};

__device__ inline void take(Best* b, int64_t value, int token) {
    if (value > b->value || (value == b->value && token < b->token)) b->value = value, b->token = token;
}

// The best of a wave's candidates, in all lanes.  A lane without one has INT64_MIN,
// below every candidate.
__device__ inline Best wave_best(Best b) {
#pragma unroll
    for (int m = 32; m; m >>= 1) {
        const int64_t value = __shfl_xor(static_cast<long long>(b.value), m);
        const int token = __shfl_xor(b.token, m);
        take(&b, value, token);
    }
    return b;
}

__device__ inline int64_t clamped(__int128 x) {
    const __int128 most = INT64_MAX;
    return static_cast<int64_t>(x < -most ? -most : x > most ? most : x);
}

// l of a token that occurs n times in the history (n > 0).
__device__ inline __int128 penalized(int64_t l, uint32_t n, const FxChoice& r) {
    __int128 x;
    if (l < 0) {
        x = (static_cast<__int128>(l) * r.repetition + 32768) >> 16;
    } else {
        // l = q r + m: l 2^16 / r = q 2^16 + m 2^16 / r, and m 2^17 stays below 2^49
        const uint64_t q = static_cast<uint64_t>(l) / r.repetition, m = static_cast<uint64_t>(l) % r.repetition;
        x = (static_cast<__int128>(q) << 16) + ((m << 17) + r.repetition) / (2 * static_cast<uint64_t>(r.repetition));
    }
    return x - static_cast<__int128>(r.frequency) * n - r.presence;
}

// What a row does to the logits of its lists' tokens.
//
// Most logits are below 2^35 and most penalties ordinary (r from 1/2 to 2, frequencies below
// 2^31): then l r + 2^15 and l 2^17 + r are whole numbers below 2^53, which doubles hold,
// and the quotient is below 2^37.  Its estimate is off by less than 2^-14, so that its floor
// with that much added is right or one too high, which the exact remainder's sign shows.
struct Rule {
    FxChoice r;
    uint32_t bias_shift;
    double rep, below, inv;  // r, 2 r, and 1 over it
    int64_t bias_max;        // sums of biases below this stay below 2^60
    bool narrow;
    __device__ Rule(const FxChoice& choice, uint32_t shift) : r(choice), bias_shift(shift) {
        rep = r.repetition;
        below = 2.0 * rep;
        inv = 1.0 / below;
        bias_max = int64_t{1} << (60 - shift);
        auto small = [](int64_t x, int bits) { return x < int64_t{1} << bits && x > -(int64_t{1} << bits); };
        narrow = r.repetition >= 1u << 15 && r.repetition <= 1u << 17 && small(r.frequency, 31) && small(r.presence, 55);
    }
    // l with n > 0 occurrences, where it fits.
    __device__ int64_t narrow_penalty(int64_t l, uint32_t n) const {
        const int high = static_cast<int>(l >> 32);
        const uint32_t low = static_cast<uint32_t>(l);
        const double x = __builtin_fma(static_cast<double>(high), 4294967296.0, static_cast<double>(low));
        const double top = __builtin_fma(x, 131072.0, rep);
        const double est = __builtin_floor(__builtin_fma(top, inv, 0x1p-14));
        const double up = __builtin_fma(-est, below, top) < 0 ? est - 1 : est;
        const double down = __builtin_floor(__builtin_fma(x, rep, 32768.0) * 0x1p-16);
        const double q = high < 0 ? down : up;
        const double q_high = __builtin_floor(q * 0x1p-32);
        const uint32_t q_low = static_cast<uint32_t>(__builtin_fma(q_high, -4294967296.0, q));
        const int64_t turned = static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(static_cast<int>(q_high))) << 32 | q_low);
        return turned - (static_cast<int64_t>(static_cast<int>(r.frequency)) * static_cast<int>(n) + r.presence);
    }
    // l with n occurrences and a sum of biases below 2^55 in size (before the shift, which
    // is at most 46).
    __device__ int64_t operator()(int64_t l, uint32_t n, int64_t bias) const {
        if (__all(narrow && bias < bias_max && bias > -bias_max && static_cast<uint32_t>(l >> 32) + 8 < 16))
            return (n ? narrow_penalty(l, n) : l) + static_cast<int64_t>(static_cast<uint64_t>(bias) << bias_shift);
        const __int128 x = n ? penalized(l, n, r) : static_cast<__int128>(l);
        return clamped(x + (static_cast<__int128>(bias) << bias_shift));
    }
};

// A logit, masked, and the best so far.
__device__ inline int64_t masked(int64_t l, bool allowed, uint32_t token, Best* best) {
    l = l == INT64_MIN ? -INT64_MAX : l;
    if (!allowed) return INT64_MIN;
    take(best, l, static_cast<int32_t>(token));
    return l;
}

// The best of a workgroup's candidates, in its first thread.
template <int WAVES>
__device__ inline Best group_best(Best best, Best* bests) {
    best = wave_best(best);
    if ((threadIdx.x & 63) == 0) bests[threadIdx.x >> 6] = best;
    __syncthreads();
    if (threadIdx.x < WAVES) best = bests[threadIdx.x];
    return threadIdx.x < 64 ? wave_best(best) : best;
}

// Entries i .. i + 3 of a list, -1 (a token outside the vocabulary) from `count` on.
__device__ inline v4i entries(const int32_t* list, uint32_t i, uint32_t count) {
    if (i + 4 <= count) return reinterpret_cast<const Four*>(list + i)->v;
    v4i four;
#pragma unroll
    for (int k = 0; k < 4; ++k) four[k] = i + k < count ? list[i + k] : -1;
    return four;
}

struct Row {
    const int64_t* logits;
    int64_t* adjusted;  // null: not kept
    const uint32_t* mask;
    const int32_t *history, *bias_tokens, *bias_values;
    __device__ Row(const FxChoose& a, const FxChoice& r, size_t row)
        : logits(a.logits + row * a.logits_stride),
          adjusted(a.adjusted ? a.adjusted + row * a.adjusted_stride : nullptr),
          mask(r.mask < 0 ? nullptr : a.allowed + r.mask),
          history(a.history + r.history),
          bias_tokens(a.bias_tokens + r.bias),
          bias_values(a.bias_values + r.bias) {}
};

// Bound by memory where rows are many, by the chain of a call where they are few.
template <bool WIDE>
__global__ __launch_bounds__(THREADS) void fx_choose_kernel(FxChoose a, Settings settings, const FxChoice* rows,
                                                            uint32_t chunk, Best* bests_of) {
    using L = Lists<WIDE>;
    extern __shared__ __attribute__((aligned(16))) uint32_t counts[];
    const uint32_t chunks = (a.vocab + chunk - 1) / chunk;
    __shared__ uint32_t keys[L::SLOTS];
    __shared__ unsigned long long biases[L::SLOTS];
    __shared__ Best bests[THREADS / 64];
    __shared__ int64_t queued[THREADS / 64][128];     // logits
    __shared__ uint32_t queued_at[THREADS / 64][128];  // tokens of the chunk, and bit 31: allowed
    const uint32_t row_at = blockIdx.x / chunks, part = blockIdx.x - row_at * chunks;
    const FxChoice r = row_at < FX_CHOICES ? settings.row[row_at] : rows[row_at - FX_CHOICES];
    const Row row(a, r, row_at);
    const uint32_t base = part * chunk, here = min(a.vocab - base, chunk);
    const bool listed = r.history_count | r.bias_count;
    const Rule rule(r, a.bias_shift);
    Pair pairs[PAIRS];
    uint32_t bits[PAIRS];
    auto load = [&](uint32_t from) {
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            const uint32_t t = from + (i * THREADS + threadIdx.x) * 2;
            if (t + 2 <= here)
                pairs[i] = *reinterpret_cast<const Pair*>(row.logits + base + t);
            else if (t < here)
                pairs[i].v[0] = row.logits[base + t];
            bits[i] = row.mask && t < here ? row.mask[(base + t) >> 5] >> (t & 31) : ~0u;
        }
    };
    load(0);  // on their way while the lists are counted
    if (listed) {
        for (uint32_t i = threadIdx.x; i < (WIDE ? (here + 3) / 4 : (here + 7) / 8); i += THREADS)
            reinterpret_cast<uint4*>(counts)[i] = make_uint4(0, 0, 0, 0);
        if (r.bias_count)
            for (uint32_t i = threadIdx.x; i < L::SLOTS; i += THREADS) keys[i] = ~0u, biases[i] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x * 4; i < r.history_count; i += THREADS * 4) {
            const v4i four = entries(row.history, i, r.history_count);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t t = static_cast<uint32_t>(four[k]) - base;
                if (t < here) atomicAdd(&counts[L::word(t)], 1u << L::shift(t));
            }
        }
        for (uint32_t i = threadIdx.x; i < r.bias_count; i += THREADS) {
            const uint32_t t = static_cast<uint32_t>(row.bias_tokens[i]) - base;
            if (t >= here) continue;
            atomicOr(&counts[L::word(t)], L::BIASED << L::shift(t));
            // at most FEW of the slots are taken: there is a free one, or the token's own
            uint32_t slot = L::slot_of(t);
            for (uint32_t old = atomicCAS(&keys[slot], ~0u, t); old != ~0u && old != t; old = atomicCAS(&keys[slot], ~0u, t))
                slot = (slot + 1) % L::SLOTS;
            atomicAdd(&biases[slot], static_cast<unsigned long long>(static_cast<int64_t>(row.bias_values[i])));
        }
        __syncthreads();
    }
    Best best{INT64_MIN, -1, 0};
    const int lane = threadIdx.x & 63;
    int64_t* queue = queued[threadIdx.x >> 6];
    uint32_t* queue_at = queued_at[threadIdx.x >> 6];
    int waiting = 0;  // of the wave's queue: below 64 between calls
    // Changes the queue's first 64 logits (or all that are there).
    auto change = [&] {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (lane < waiting) {
            const int64_t l = queue[lane];
            const uint32_t at = queue_at[lane], t = at & 0x7fffffff;
            const uint32_t count = L::of(counts, t);
            int64_t bias = 0;
            if (count & L::BIASED) {
                uint32_t slot = L::slot_of(t);
                while (keys[slot] != t) slot = (slot + 1) % L::SLOTS;
                bias = static_cast<int64_t>(biases[slot]);
            }
            const bool allowed = at >> 31;
            const int64_t changed = allowed ? rule(l, count & L::MOST, bias) : INT64_MIN;
            if (allowed) take(&best, changed, static_cast<int>(base + t));
            if (row.adjusted) row.adjusted[base + t] = changed;
        }
        // the others to the front
        const bool more = lane + 64 < waiting;
        const int64_t l = more ? queue[64 + lane] : 0;
        const uint32_t at = more ? queue_at[64 + lane] : 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (more) queue[lane] = l, queue_at[lane] = at;
        waiting = max(waiting - 64, 0);
    };
    // All lanes of the wave together.
    auto push = [&](bool listed_token, uint32_t t, int64_t l, bool allowed) {
        const uint64_t which = __ballot(listed_token);
        if (!which) return;
        if (listed_token) {
            const int at = waiting + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(which >> 32),
                                                               __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(which), 0));
            queue[at] = l;
            queue_at[at] = t | (allowed ? 1u << 31 : 0);
        }
        waiting += __popcll(which);
        if (waiting >= 64) change();
    };
    for (uint32_t from = 0; from < here; from += PAIRS * THREADS * 2) {
        if (from) load(from);
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            const uint32_t t = from + (i * THREADS + threadIdx.x) * 2;
            const bool one = t < here, two = t + 2 <= here;
            const uint2 count = listed && one ? L::two(counts, t) : make_uint2(0, 0);
            Pair p = pairs[i];
            if (listed) {
                push(one && count.x, t, p.v[0], bits[i] & 1);
                push(two && count.y, t + 1, p.v[1], bits[i] & 2);
            }
            const bool first = one && !count.x, second = two && !count.y;
            if (first) p.v[0] = masked(p.v[0], bits[i] & 1, base + t, &best);
            if (second) p.v[1] = masked(p.v[1], bits[i] & 2, base + t + 1, &best);
            if (!row.adjusted) continue;
            if (first && second) {
                *reinterpret_cast<Pair*>(row.adjusted + base + t) = p;
            } else {
                if (first) row.adjusted[base + t] = p.v[0];
                if (second) row.adjusted[base + t + 1] = p.v[1];
            }
        }
    }
    if (listed) change();
    best = group_best<THREADS / 64>(best, bests);
    if (threadIdx.x == 0) {
        if (chunks == 1)
            a.tokens[row_at] = best.token;
        else
            bests_of[blockIdx.x] = best;
    }
}

// Settings of more rows than a launch's arguments hold, to memory.
__global__ __launch_bounds__(FX_CHOICES) void fx_choose_settings_kernel(Settings settings, FxChoice* rows, uint32_t count) {
    if (threadIdx.x < count) rows[threadIdx.x] = settings.row[threadIdx.x];
}

// A wave a row: the best of its chunks' candidates.
__global__ __launch_bounds__(64) void fx_choose_join_kernel(const Best* bests, uint32_t groups, int32_t* tokens) {
    Best b{INT64_MIN, -1, 0};
    for (uint32_t i = threadIdx.x; i < groups; i += 64) {
        const Best x = bests[static_cast<size_t>(blockIdx.x) * groups + i];
        take(&b, x.value, x.token);
    }
    b = wave_best(b);
    if (threadIdx.x == 0) tokens[blockIdx.x] = b.token;
}

// Lists of any length, a chunk of DENSE tokens at a time.
__global__ __launch_bounds__(256) void fx_choose_dense_kernel(FxChoose a, Settings settings, uint32_t first_row) {
    __shared__ uint32_t counts[DENSE];
    __shared__ unsigned long long biases[DENSE];
    __shared__ Best bests[4];
    const FxChoice& r = settings.row[blockIdx.x];
    const Row row(a, r, static_cast<size_t>(first_row) + blockIdx.x);
    const Rule rule(r, a.bias_shift);
    Best best{INT64_MIN, -1, 0};
    for (uint32_t base = 0; base < a.vocab; base += DENSE) {
        const uint32_t here = min(a.vocab - base, static_cast<uint32_t>(DENSE));
        __syncthreads();  // the chunk before is done
        for (int i = threadIdx.x; i < DENSE; i += 256) counts[i] = 0, biases[i] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < r.history_count; i += 256) {
            const uint32_t t = static_cast<uint32_t>(row.history[i]) - base;
            if (t < here) atomicAdd(&counts[t], 1u);
        }
        for (uint32_t i = threadIdx.x; i < r.bias_count; i += 256) {
            const uint32_t t = static_cast<uint32_t>(row.bias_tokens[i]) - base;
            if (t < here) atomicAdd(&biases[t], static_cast<unsigned long long>(static_cast<int64_t>(row.bias_values[i])));
        }
        __syncthreads();
        for (uint32_t t = threadIdx.x; t < here; t += 256) {
            const uint32_t token = base + t, n = counts[t];
            const int64_t bias = static_cast<int64_t>(biases[t]);
            int64_t l = row.logits[token];
            if (n || bias) l = rule(l, n, bias);
            l = masked(l, !row.mask || (row.mask[token >> 5] >> (token & 31) & 1), token, &best);
            if (row.adjusted) row.adjusted[token] = l;
        }
    }
    best = group_best<4>(best, bests);
    if (threadIdx.x == 0) a.tokens[first_row + blockIdx.x] = best.token;
}

// Rows of one launch, at most; a grid holds less than 2^32 threads.
constexpr size_t CALL_ROWS = 4096, CALL_GROUPS = size_t{1} << 21;

int choose_rows(Context* c, const FxChoose& a, const FxChoice* rows, size_t count) {
    uint32_t history = 0, biases = 0;
    for (size_t i = 0; i < count; ++i) {
        history = std::max(history, rows[i].history_count);
        biases = std::max(biases, rows[i].bias_count);
    }
    // Long lists, us by the wide lists and by a count and a sum a token (fx_choose_dense_kernel): one,
    // 64 and 256 rows of 50,257, 40,000 tokens of history 12, 25, 76 and 633, 713, 2,873; 600 biases
    // 11, 20, 51 and 84, 178, 505; 64 rows, 5,000 biases 46 and 268.  Counts of 31 bits need three
    // chunks a row, and each reads the row's lists: without them the 256 rows take 31.
    const bool wide = history > Lists<false>::MOST || biases > Lists<false>::BIASES;
    const uint32_t longest =
        !wide ? Lists<false>::CHUNK : biases <= Lists<true>::BIASES ? Lists<true>::CHUNK : Lists<true>::FEW;
    // Chunks of at least 1,024 tokens (many rows: a pass of all threads), for a workgroup a CU:
    // each counts all of its row's lists.  us with one, two (of half the threads), four and
    // eight a CU: 256 rows of 50,257 43.7, 49.0, 55.8, 68.7; 64 rows 20.9, 20.9, 25.0, 36.9.
    const size_t want = (c->cu_count + count - 1) / count;
    const uint32_t least = (a.vocab + longest - 1) / longest, short_chunk = count < 32 ? 1024 : PAIRS * THREADS * 2,
                   most = (a.vocab + short_chunk - 1) / short_chunk;
    uint32_t groups = std::max(least, static_cast<uint32_t>(std::min<size_t>(want, most)));
    // whole words of a mask (of which CHUNK and FEW are multiples)
    const uint32_t chunk = ((a.vocab + groups - 1) / groups + 63) / 64 * 64;
    groups = (a.vocab + chunk - 1) / chunk;
    // Candidates, and settings that are no arguments; where no space is to be had, a workgroup a row.
    Best* bests = nullptr;
    FxChoice* in_memory = nullptr;
    bool dense = false;
    if (groups > 1 || count > FX_CHOICES) {
        const size_t best_bytes = count * groups * sizeof(Best);
        dense = count * groups > CALL_GROUPS ||
                !try_ws(c, WS_FIXED, workspace_step(best_bytes + count * sizeof(FxChoice), FX_SPACE_MAX));
        bests = ws<Best>(c, WS_FIXED);
        if (count > FX_CHOICES) in_memory = reinterpret_cast<FxChoice*>(ws<unsigned char>(c, WS_FIXED) + best_bytes);
    }
    Settings s;
    for (size_t at = dense || !in_memory ? 0 : FX_CHOICES; at < count; at += FX_CHOICES) {
        const size_t here = std::min<size_t>(count - at, FX_CHOICES);
        std::copy(rows + at, rows + at + here, s.row);
        if (dense)
            hipLaunchKernelGGL(fx_choose_dense_kernel, dim3(static_cast<unsigned>(here)), dim3(256), 0, c->stream, a, s,
                               static_cast<uint32_t>(at));
        else if (in_memory)
            hipLaunchKernelGGL(fx_choose_settings_kernel, dim3(1), dim3(FX_CHOICES), 0, c->stream, s,
                               in_memory + at - FX_CHOICES, static_cast<uint32_t>(here));
        VMX_HIP(c, hipGetLastError());
    }
    if (dense) return 0;
    std::copy(rows, rows + std::min<size_t>(count, FX_CHOICES), s.row);
    const auto kernel = wide ? fx_choose_kernel<true> : fx_choose_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(count * groups)), dim3(THREADS),
                       history || biases ? chunk * (wide ? 4 : 2) : 0, c->stream, a, s, in_memory, chunk, bests);
    VMX_HIP(c, hipGetLastError());
    if (groups > 1) {
        hipLaunchKernelGGL(fx_choose_join_kernel, dim3(static_cast<unsigned>(count)), dim3(64), 0, c->stream, bests, groups,
                           a.tokens);
        VMX_HIP(c, hipGetLastError());
    }
    return 0;
}

}  // namespace

int fx_choose(Context* c, const FxChoose& a, const FxChoice* rows, size_t count) {
    FxChoose part = a;
    for (size_t row = 0; row < count; row += CALL_ROWS) {
        part.logits = a.logits + row * a.logits_stride;
        part.adjusted = a.adjusted ? a.adjusted + row * a.adjusted_stride : nullptr;
        part.tokens = a.tokens + row;
        if (choose_rows(c, part, rows + row, std::min(count - row, CALL_ROWS))) return -1;
    }
    return 0;
}

}  // namespace vmx
