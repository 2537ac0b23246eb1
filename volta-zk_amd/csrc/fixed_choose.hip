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
// A workgroup takes a chunk of a row's vocabulary: it counts the history's and sums
// the biases' entries that fall into the chunk in LDS, then goes over the logits
// once.  The chunks' best are joined by a second launch.
#include <algorithm>
#include <climits>

#include "fixed.hpp"

namespace vmx {
namespace {

using namespace fx;

constexpr int CHUNK = 2048;

struct Settings {
    FxChoice row[FX_CHOICES];
};

// A candidate: INT64_MIN and -1 where there is none.
struct Best {
    int64_t value;
    int32_t token;
    int32_t reserved;
};

struct ChooseArgs {
    FxChoose a;
    uint32_t chunks;  // of a row
    Best* best;
};

struct __attribute__((packed, aligned(8))) Pair {
    int64_t v[2];
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

__global__ __launch_bounds__(256) void fx_choose_kernel(ChooseArgs c, Settings settings, uint32_t first_row) {
    __shared__ uint32_t counts[CHUNK];
    __shared__ unsigned long long biases[CHUNK];
    __shared__ Best bests[4];
    const FxChoose& a = c.a;
    const FxChoice& r = settings.row[blockIdx.y];
    const size_t row = static_cast<size_t>(first_row) + blockIdx.y;
    const int64_t* logits = a.logits + row * a.logits_stride;
    int64_t* adjusted = a.adjusted ? a.adjusted + row * a.adjusted_stride : nullptr;
    const uint32_t* mask = r.mask < 0 ? nullptr : a.allowed + r.mask;
    const int32_t* history = a.history + r.history;
    const int32_t *bias_tokens = a.bias_tokens + r.bias, *bias_values = a.bias_values + r.bias;
    Best best{INT64_MIN, -1, 0};
    for (uint32_t chunk = blockIdx.x; chunk < c.chunks; chunk += gridDim.x) {
        const uint32_t base = chunk * CHUNK, here = min(a.vocab - base, static_cast<uint32_t>(CHUNK));
        if (r.history_count | r.bias_count) {
            __syncthreads();  // the chunk before is done
            for (int i = threadIdx.x; i < CHUNK; i += 256) counts[i] = 0, biases[i] = 0;
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < r.history_count; i += 256) {
                const uint32_t t = static_cast<uint32_t>(history[i]) - base;
                if (t < here) atomicAdd(&counts[t], 1u);
            }
            for (uint32_t i = threadIdx.x; i < r.bias_count; i += 256) {
                const uint32_t t = static_cast<uint32_t>(bias_tokens[i]) - base;
                if (t < here) atomicAdd(&biases[t], static_cast<unsigned long long>(static_cast<int64_t>(bias_values[i])));
            }
            __syncthreads();
        }
        auto one = [&](uint32_t t, int64_t l, uint32_t bits) {
            if (r.history_count | r.bias_count) {
                const uint32_t n = counts[t];
                const int64_t bias = static_cast<int64_t>(biases[t]);
                if (n || bias) {
                    __int128 x = n ? penalized(l, n, r) : static_cast<__int128>(l);
                    // below 2^55 in size before the shift, which is at most 46
                    x += static_cast<__int128>(bias) << a.bias_shift;
                    l = clamped(x);
                }
            }
            l = l == INT64_MIN ? -INT64_MAX : l;
            if (!(bits & 1))
                l = INT64_MIN;
            else if (l > best.value)  // a thread's tokens ascend
                best.value = l, best.token = static_cast<int32_t>(base + t);
            return l;
        };
        for (uint32_t t = threadIdx.x * 2; t < here; t += 512) {
            const uint32_t bits = mask ? mask[(base + t) >> 5] >> (t & 31) : ~0u;
            if (t + 2 <= here) {
                Pair p = *reinterpret_cast<const Pair*>(logits + base + t);
                p.v[0] = one(t, p.v[0], bits);
                p.v[1] = one(t + 1, p.v[1], bits >> 1);
                if (adjusted) *reinterpret_cast<Pair*>(adjusted + base + t) = p;
            } else {
                const int64_t l = one(t, logits[base + t], bits);
                if (adjusted) adjusted[base + t] = l;
            }
        }
    }
    best = wave_best(best);
    if ((threadIdx.x & 63) == 0) bests[threadIdx.x >> 6] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 4; ++w) take(&best, bests[w].value, bests[w].token);
        if (gridDim.x == 1)
            a.tokens[row] = best.token;
        else
            c.best[row * gridDim.x + blockIdx.x] = best;
    }
}

// A wave a row: the best of its workgroups' candidates.
__global__ __launch_bounds__(64) void fx_choose_join_kernel(const Best* best, uint32_t groups, int32_t* tokens) {
    Best b{INT64_MIN, -1, 0};
    for (uint32_t i = threadIdx.x; i < groups; i += 64) {
        const Best x = best[static_cast<size_t>(blockIdx.x) * groups + i];
        take(&b, x.value, x.token);
    }
    b = wave_best(b);
    if (threadIdx.x == 0) tokens[blockIdx.x] = b.token;
}

}  // namespace

int fx_choose(Context* c, const FxChoose& a, const FxChoice* rows, size_t count) {
    ChooseArgs args{a, (a.vocab + CHUNK - 1) / CHUNK, nullptr};
    uint32_t groups = std::min(args.chunks, 65535u);
    if (groups > 1) {
        // where no space is to be had, a row's chunks are one workgroup's
        if (try_ws(c, WS_FIXED, workspace_step(count * groups * sizeof(Best), FX_SPACE_MAX)))
            args.best = ws<Best>(c, WS_FIXED);
        else
            groups = 1;
    }
    for (size_t at = 0; at < count; at += FX_CHOICES) {
        Settings s;
        const size_t here = std::min<size_t>(count - at, FX_CHOICES);
        std::copy(rows + at, rows + at + here, s.row);
        hipLaunchKernelGGL(fx_choose_kernel, dim3(groups, static_cast<unsigned>(here)), dim3(256), 0, c->stream, args, s,
                           static_cast<uint32_t>(at));
        VMX_HIP(c, hipGetLastError());
    }
    if (groups > 1) {
        hipLaunchKernelGGL(fx_choose_join_kernel, dim3(static_cast<unsigned>(count)), dim3(64), 0, c->stream, args.best,
                           groups, a.tokens);
        VMX_HIP(c, hipGetLastError());
    }
    return 0;
}

}  // namespace vmx
