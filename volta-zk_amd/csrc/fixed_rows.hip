// fixed_rows.hip -- row operators of the fixed-point model: the norm with its
// residual addition, the embedding of tokens and positions, and heads normed and
// rotated.  All are bound by memory: eight elements a thread at a time, whatever
// the rows' alignment.
#include <algorithm>

#include "fixed.hpp"

namespace vmx {
namespace {

using namespace fx;

union Eight {
    v4i v;
    int16_t e[8];
};

// Elements at .. at + 7 of a row of `len`, zero from len on.
__device__ inline v4i load8(const int16_t* p, int at, int len) {
    Eight u;
    if (at + 8 <= len) {
        u.v = fx::load8(p + at);
    } else {
        u.v = v4i{0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (at + e < len) u.e[e] = p[at + e];
    }
    return u.v;
}

__device__ inline void store8(int16_t* p, int at, int len, v4i v) {
    if (at + 8 <= len) {
        reinterpret_cast<Row16*>(p + at)->v = v;
    } else {
        Eight u;
        u.v = v;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (at + e < len) p[at + e] = u.e[e];
    }
}

__device__ inline v4i add_sat(v4i a, v4i b) {
    v4i c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int x = a[i], y = b[i];
        c[i] = __builtin_bit_cast(int, __builtin_elementwise_add_sat(__builtin_bit_cast(v2s, x), __builtin_bit_cast(v2s, y)));
    }
    return c;
}

// The sum of a wave's values, in all lanes: four steps within rows of 16 lanes,
// two across them, no LDS.
__device__ inline int wave_sum(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return __builtin_amdgcn_readlane(v, 63);
}

// The same for values below 2^44.
__device__ inline uint64_t wave_sum(uint64_t v) {
    const uint32_t low = static_cast<uint32_t>(wave_sum(static_cast<int>(v & 0xfffff)));
    return (static_cast<uint64_t>(static_cast<uint32_t>(wave_sum(static_cast<int>(v >> 20)))) << 20) + low;
}

// floor(sqrt(v)) for 0 < v < 2^63: the rounded square root of the rounded v is
// off by less than one.
__device__ inline uint64_t floor_sqrt(uint64_t v) {
    uint64_t r = static_cast<uint64_t>(__builtin_sqrt(static_cast<double>(v)));
    if (r * r > v) --r;
    if ((r + 1) * (r + 1) <= v) ++r;
    return r;
}

// ---- norm -----------------------------------------------------------------------------
// h = sat(x + residual); S = sum h (0 for rms), V = n sum h^2 - S^2,
// R = floor(sqrt(V + eps)); y = sat(floor((2 (n h - S) gain + B) / 2B) + bias), B = R 2^shift.
//
// THREADS threads a row, KEPT pieces of eight elements each in registers (0: any
// length, read twice).  A wave that has rows to itself takes several in turn and
// keeps the gains.
//
// |n h - S| <= 2^32 and B < 2^47, so every value of the division is a whole number
// below 2^53: doubles hold it exactly.  The quotient is estimated a little high:
// where it is below 2^17 the estimate is off by less than 2^-34, so its floor is
// right or one too high, which the exact remainder's sign shows; where it is not,
// the result is clamped whatever it is.
//
// 16,384 rows of 768 with a residual, its sum kept (100 MB): 25 us, 4.0 TB/s
// (a copy reaches 5.0); a row a workgroup, elements one by one, took 57.
template <int THREADS, int KEPT>
__global__ __launch_bounds__(256) void fx_norm_kernel(FxNorm a) {
    constexpr int WAVES = THREADS / 64, ROWS = 256 / THREADS;
    __shared__ int64_t part[2][4];
    const int thread = threadIdx.x % THREADS;
    double gain[KEPT ? KEPT * 8 : 8];
    Eight bias[KEPT ? KEPT : 1];
    auto load_gain = [&](int at, double* g, Eight* b) {
        Eight u;
        u.v = load8(a.gain, at, a.cols);
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = 2.0 * u.e[e];
        b->v = a.bias ? load8(a.bias, at, a.cols) : v4i{0, 0, 0, 0};
    };
    if constexpr (KEPT > 0) {
#pragma unroll
        for (int i = 0; i < KEPT; ++i) {
            const int at = (i * THREADS + thread) * 8;
            if (at < a.cols) load_gain(at, gain + 8 * i, &bias[i]);
        }
    }
    for (size_t row = static_cast<size_t>(blockIdx.x) * ROWS + threadIdx.x / THREADS; row < a.rows;
         row += static_cast<size_t>(gridDim.x) * ROWS) {
        const int16_t* x = a.x + row * a.x_stride;
        const int16_t* res = a.residual ? a.residual + row * a.residual_stride : nullptr;
        auto piece = [&](int at) {
            const v4i v = load8(x, at, a.cols);
            return res ? add_sat(v, load8(res, at, a.cols)) : v;
        };
        int s = 0;  // at most 2^31 - 2^15, or -2^31, over a row
        uint64_t q = 0;
        auto count = [&](v4i v) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int pair = v[i];
                const v2s two = __builtin_bit_cast(v2s, pair);
                s = __builtin_amdgcn_sdot2(two, v2s{1, 1}, s, false);
                q += static_cast<uint32_t>(__builtin_amdgcn_sdot2(two, two, 0, false));  // at most 2^31
            }
        };
        v4i kept[KEPT ? KEPT : 1];
        if constexpr (KEPT > 0) {
#pragma unroll
            for (int i = 0; i < KEPT; ++i) {
                const int at = (i * THREADS + thread) * 8;
                kept[i] = at < a.cols ? piece(at) : v4i{0, 0, 0, 0};
                count(kept[i]);
            }
        } else {
            for (int at = thread * 8; at < a.cols; at += THREADS * 8) count(piece(at));
        }
        int64_t sum = wave_sum(s);
        q = wave_sum(q);
        if constexpr (WAVES > 1) {
            if (threadIdx.x / 64 * 64 == threadIdx.x) {
                part[0][threadIdx.x / 64] = sum;
                part[1][threadIdx.x / 64] = static_cast<int64_t>(q);
            }
            __syncthreads();
            sum = part[0][0] + part[0][1] + part[0][2] + part[0][3];
            q = static_cast<uint64_t>(part[1][0] + part[1][1] + part[1][2] + part[1][3]);
            __syncthreads();  // before the next row's
        }
        if (a.rms) sum = 0;
        const uint64_t v = static_cast<uint64_t>(a.cols) * q - static_cast<uint64_t>(sum * sum) + a.eps;
        const double below = 2.0 * static_cast<double>(floor_sqrt(v) << a.shift), inv = 1.0 / below, half = 0.5 * below;
        const double n = a.cols, away = -static_cast<double>(sum);
        auto finish = [&](int at, v4i h, const double* g, const Eight& b) {
            Eight hu, out;
            hu.v = h;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const double top = __builtin_fma(__builtin_fma(n, static_cast<double>(hu.e[e]), away), g[e], half);
                const double est = __builtin_floor(__builtin_fma(top, inv, 0x1p-34));
                const double rest = __builtin_fma(-est, below, top);
                const double est_in = __builtin_fmin(__builtin_fmax(est, -1048576.0), 1048576.0);
                int y = static_cast<int>(est_in) + (__builtin_bit_cast(int64_t, rest) < 0 ? -1 : 0) + b.e[e];
                out.e[e] = static_cast<int16_t>(min(max(y, -32768), 32767));
            }
            store8(a.out + row * a.out_stride, at, a.cols, out.v);
            if (a.sum) store8(a.sum + row * a.sum_stride, at, a.cols, h);
        };
        if constexpr (KEPT > 0) {
#pragma unroll
            for (int i = 0; i < KEPT; ++i) {
                const int at = (i * THREADS + thread) * 8;
                if (at < a.cols) finish(at, kept[i], gain + 8 * i, bias[i]);
            }
        } else {
            // a sum over x or the residual is written by the thread that has read it
            for (int at = thread * 8; at < a.cols; at += THREADS * 8) {
                load_gain(at, gain, bias);
                finish(at, piece(at), gain, bias[0]);
            }
        }
    }
}

// ---- embedding ------------------------------------------------------------------------
// out = sat(rs(table[token] scale, shift) + positions[position]); a token or
// position outside its table adds nothing.  A thread takes eight elements of a
// row; 16,384 rows of 768 (75 MB): 14 us, 5.4 TB/s (rows of the
// tables come twice and more, from the caches).
__global__ __launch_bounds__(256) void fx_embed_kernel(FxEmbed a, uint32_t pieces) {
    const size_t id = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x, row = id / pieces;
    if (row >= a.rows) return;
    const int at = static_cast<int>(id - row * pieces) * 8;
    const int64_t token = a.tokens[row], place = a.positions ? a.positions[row] : -1;
    Eight u;
    u.v = v4i{0, 0, 0, 0};
    if (token >= 0 && static_cast<size_t>(token) < a.vocab) {
        u.v = load8(a.table + token * a.table_stride, at, a.cols);
        if (a.scale != 1 || a.shift) {
            // the sum with the position is clamped once: outside 17 bits it is
            // clamped whatever the position holds
            Eight p;
            p.v = v4i{0, 0, 0, 0};
            if (place >= 0 && static_cast<size_t>(place) < a.position_rows)
                p.v = load8(a.position_table + place * a.position_stride, at, a.cols);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                u.e[e] = static_cast<int16_t>(sat16(rounded(static_cast<int64_t>(u.e[e]) * a.scale, a.shift) + p.e[e]));
            store8(a.out + row * a.out_stride, at, a.cols, u.v);
            return;
        }
    }
    if (place >= 0 && static_cast<size_t>(place) < a.position_rows)
        u.v = add_sat(u.v, load8(a.position_table + place * a.position_stride, at, a.cols));
    store8(a.out + row * a.out_stride, at, a.cols, u.v);
}

// ---- heads normed and rotated -------------------------------------------------------------
// For each head of n places: with a gain, V = n sum h^2 + eps, R = floor(sqrt(V)),
// B = R 2^gain_shift, h = sat(floor((2 n h gain + B) / 2B)): the norm's rounding to 16
// bits, so that this is the norm of each head followed by the rotation.  Then the
// places of pair i < pairs, (i, i + pairs) or (2 i, 2 i + 1), are turned by (c, s) =
// angles[position][i]; those after them stay, and so do all of a row whose position
// is outside the table.
//
// LANES lanes a head, four pairs of places each (what follows the pairs counts as
// pairs that stay): a head's sum takes log2 LANES steps between neighbours, and both
// places of a pair are in one lane, in one register.
//
// With gains, bound by vector instructions (f64: 0.70 of their issue) beside memory: 16,384 rows
// of 24 heads of 64 28.5 to 32.5 us where the last-level cache still holds a part of the rows, 36
// where it does not (101 MB at 3.5 to 2.8 TB/s).  Without them by memory: 4,095 rows of 40 heads
// of 128, 96 places of each turned, 16.5 and 21 us, 84 MB at 5.1 and 4.0 TB/s.
//
// KEPT heads a lane, in turn: the root and the reciprocal cost as much as eight places'
// quotients, and lane k of a head's lanes computes those of the k-th head for all.
//
// V is below 2^46, and a root that is no whole number at least 2^-24 below the next, far more
// than its rounding: its floor is R.  The estimate of a quotient (below 2^20 in size) is
// off by less than 2^-20, so that its floor with that much added is right or one too high, which
// the exact remainder's sign shows.  R is at least half the root of V >= n h^2, so that a
// quotient is below 2 sqrt(n) 2^15 in size and needs no bounds.  a c - b s = a c + (~b) s + s:
// a product of two pairs that saturates at 32 bits, which the sum's clamp to 16 does not show.
template <int LANES>
__device__ inline int group_sum(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0xb1, 0xf, 0xf, true);  // lanes 1 0 3 2
    v += __builtin_amdgcn_update_dpp(0, v, 0x4e, 0xf, 0xf, true);  // lanes 2 3 0 1
    if constexpr (LANES > 4) v += __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true);  // 7 - lane of 8
    if constexpr (LANES > 8) v += __builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, true);  // 15 - lane of 16
    return v;
}

template <int LANES, int KEPT>
__global__ __launch_bounds__(256, 8) void fx_rotate_kernel(FxRotate a, uint32_t items) {
    constexpr uint32_t HEADS = 64 / LANES;  // of a wave at a time
    const int lane = threadIdx.x & 63, part = lane % LANES, first = part * 4;  // pair
    const uint32_t item0 = (blockIdx.x * 4 + threadIdx.x / 64) * (HEADS * KEPT) + lane / LANES;
    // places of pair u: `one` and `two`
    auto one = [&](int u) { return a.adjacent || u >= a.pairs ? 2 * u : u; };
    auto two = [&](int u) { return a.adjacent || u >= a.pairs ? 2 * u + 1 : u + a.pairs; };
    // The lane's places are eight in a row, or four and four; a lane with pairs of both
    // kinds, or at the head's end, takes them one by one.
    const bool joint = a.adjacent || first >= a.pairs;
    const bool whole = joint ? 2 * first + 8 <= a.dim : first + 4 <= a.pairs;
    auto load = [&](const int16_t* p) {
        v4i h;
        if (whole && joint) {
            h = fx::load8(p + 2 * first);
        } else if (whole) {
            const uint2 lo = reinterpret_cast<const Row8*>(p + first)->v;
            const uint2 hi = reinterpret_cast<const Row8*>(p + first + a.pairs)->v;
            h[0] = static_cast<int>(__builtin_amdgcn_perm(hi.x, lo.x, 0x05040100u));
            h[1] = static_cast<int>(__builtin_amdgcn_perm(hi.x, lo.x, 0x07060302u));
            h[2] = static_cast<int>(__builtin_amdgcn_perm(hi.y, lo.y, 0x05040100u));
            h[3] = static_cast<int>(__builtin_amdgcn_perm(hi.y, lo.y, 0x07060302u));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint16_t x = static_cast<uint16_t>(one(first + i) < a.dim ? p[one(first + i)] : 0);
                const uint16_t y = static_cast<uint16_t>(two(first + i) < a.dim ? p[two(first + i)] : 0);
                h[i] = static_cast<int>(x | static_cast<uint32_t>(y) << 16);
            }
        }
        return h;
    };
    auto pair_of = [](int x, int y) { return static_cast<int>((static_cast<uint32_t>(x) & 0xffff) | static_cast<uint32_t>(y) << 16); };
    auto clamp = [](int y) { return min(max(y, -32768), 32767); };
    v4i kept[KEPT];
    uint32_t rows[KEPT], heads[KEPT];
#pragma unroll
    for (int k = 0; k < KEPT; ++k) {
        const uint32_t item = item0 + k * HEADS;
        rows[k] = item / a.all_heads;
        heads[k] = item - rows[k] * a.all_heads;
        kept[k] = v4i{0, 0, 0, 0};
        if (item < items) kept[k] = load(a.x + rows[k] * a.x_stride + static_cast<size_t>(heads[k]) * a.dim);
    }
    double below = 1.0, inv = 1.0;
    if (a.q_gain || a.k_gain) {
        uint64_t sum = 0;  // of this lane's head
#pragma unroll
        for (int k = 0; k < KEPT; ++k) {
            uint64_t q = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int pair = kept[k][i];
                const v2s two_places = __builtin_bit_cast(v2s, pair);
                q += static_cast<uint32_t>(__builtin_amdgcn_sdot2(two_places, two_places, 0, false));  // at most 2^31
            }
            // at most 2^33 a lane: in parts of 20 bits
            const uint32_t low = static_cast<uint32_t>(group_sum<LANES>(static_cast<int>(q & 0xfffff)));
            const uint32_t high = static_cast<uint32_t>(group_sum<LANES>(static_cast<int>(q >> 20)));
            if (KEPT == 1 || part == k) sum = (static_cast<uint64_t>(high) << 20) + low;
        }
        const uint64_t v = static_cast<uint64_t>(a.dim) * sum + a.eps;
        const double value = __builtin_fma(static_cast<double>(static_cast<uint32_t>(v >> 32)), 4294967296.0,
                                           static_cast<double>(static_cast<uint32_t>(v)));
        below = __builtin_floor(__builtin_sqrt(value)) * static_cast<double>(2u << a.gain_shift);
        inv = __builtin_amdgcn_rcp(below);
        inv = __builtin_fma(inv, __builtin_fma(-below, inv, 1.0), inv);
        inv = __builtin_fma(inv, __builtin_fma(-below, inv, 1.0), inv);
    }
    const double n2 = 2.0 * a.dim;
#pragma unroll
    for (int k = 0; k < KEPT; ++k) {
        // of the k-th head
        const int from = lane - part + k;
        const double b = KEPT == 1 ? below : __shfl(below, from), r = KEPT == 1 ? inv : __shfl(inv, from), half_b = 0.5 * b;
        if (item0 + k * HEADS >= items) break;
        v4i h = kept[k];
        const int16_t* gains = heads[k] < a.heads ? a.q_gain : a.k_gain;
        if (gains) {
            const v4i g = load(gains);
            auto normed = [&](int x, int gain) {
                const double top = __builtin_fma(n2, static_cast<double>(__mul24(x, gain)), half_b);
                const double est = __builtin_floor(__builtin_fma(top, r, 0x1p-20));
                const double rest = __builtin_fma(-est, b, top);
                return clamp(static_cast<int>(est) + (__builtin_bit_cast(int64_t, rest) < 0 ? -1 : 0));
            };
#pragma unroll
            for (int i = 0; i < 4; ++i)
                h[i] = pair_of(normed(static_cast<int16_t>(h[i]), static_cast<int16_t>(g[i])), normed(h[i] >> 16, g[i] >> 16));
        }
        if (first < a.pairs) {
            const int64_t place = a.positions[rows[k]];
            if (place >= 0 && static_cast<size_t>(place) < a.angle_rows) {
                const v4i turns = load8(a.angles + (static_cast<size_t>(place) * a.pairs + first) * 2, 0, 2 * (a.pairs - first));
                const int half = a.angle_shift ? 1 << (a.angle_shift - 1) : 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (first + i >= a.pairs) continue;
                    const int pair = h[i], less = pair ^ static_cast<int>(0xffff0000), cs = turns[i];
                    const int sc = static_cast<int>(__builtin_amdgcn_perm(cs, cs, 0x01000302u));
                    auto dot = [](int p, int q, int acc) {
                        return __builtin_amdgcn_sdot2(__builtin_bit_cast(v2s, p), __builtin_bit_cast(v2s, q), acc, true);
                    };
                    h[i] = pair_of(clamp(dot(less, cs, half + (cs >> 16)) >> a.angle_shift),
                                   clamp(dot(pair, sc, half) >> a.angle_shift));
                }
            }
        }
        int16_t* out = a.out + rows[k] * a.out_stride + static_cast<size_t>(heads[k]) * a.dim;
        if (whole && joint) {
            reinterpret_cast<Row16*>(out + 2 * first)->v = h;
        } else if (whole) {
            reinterpret_cast<Row8*>(out + first)->v =
                make_uint2(__builtin_amdgcn_perm(h[1], h[0], 0x05040100u), __builtin_amdgcn_perm(h[3], h[2], 0x05040100u));
            reinterpret_cast<Row8*>(out + first + a.pairs)->v =
                make_uint2(__builtin_amdgcn_perm(h[1], h[0], 0x07060302u), __builtin_amdgcn_perm(h[3], h[2], 0x07060302u));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (one(first + i) < a.dim) out[one(first + i)] = static_cast<int16_t>(h[i]);
                if (two(first + i) < a.dim) out[two(first + i)] = static_cast<int16_t>(h[i] >> 16);
            }
        }
    }
}

template <int LANES>
void launch_rotate(Context* c, const FxRotate& a) {
    const uint32_t items = static_cast<uint32_t>(a.rows) * a.all_heads;
    auto launch = [&](auto kernel, uint32_t each) {
        hipLaunchKernelGGL(kernel, dim3((items + each - 1) / each), dim3(256), 0, c->stream, a, items);
    };
    // Two heads a lane where they have norms and are many.  16,384 rows of 24 heads of 64, the same
    // each time, us with one, two and four: 30.5, 28.5, 32.1.
    if ((a.q_gain || a.k_gain) && items >= 512u / LANES * 4 * static_cast<uint32_t>(c->cu_count))
        launch(fx_rotate_kernel<LANES, 2>, 512 / LANES);
    else
        launch(fx_rotate_kernel<LANES, 1>, 256 / LANES);
}

template <int THREADS, int KEPT>
void launch_norm(Context* c, const FxNorm& a) {
    constexpr size_t rows = 256 / THREADS;
    // several rows a workgroup once there are eight workgroups a CU
    const size_t groups = std::min<size_t>((a.rows + rows - 1) / rows, 8 * static_cast<size_t>(c->cu_count));
    hipLaunchKernelGGL((fx_norm_kernel<THREADS, KEPT>), dim3(static_cast<unsigned>(groups)), dim3(256), 0, c->stream, a);
}

}  // namespace

// A row a wave while the wave can keep it: no barrier.  16,384 rows, us by a wave
// and by 256 threads a row: 512 columns 11.7 and 20.2, 768 18.2 and 26.9, 2,048 32.7
// and 38.5.  With 256 threads, kept and read twice: 4,096 columns 61.5 and 67.5,
// 8,192 131 and 151.  Pieces no row has cost too (768 columns in four pieces a
// thread 54.6), so there are widths in between.
int fx_norm(Context* c, const FxNorm& a) {
    if (a.cols <= 512)
        launch_norm<64, 1>(c, a);
    else if (a.cols <= 1024)
        launch_norm<64, 2>(c, a);
    else if (a.cols <= 2048)
        launch_norm<64, 4>(c, a);
    else if (a.cols <= 4096)
        launch_norm<256, 2>(c, a);
    else if (a.cols <= 8192)
        launch_norm<256, 4>(c, a);
    else
        launch_norm<256, 0>(c, a);
    VMX_HIP(c, hipGetLastError());
    return 0;
}

int fx_embed(Context* c, const FxEmbed& a) {
    const uint32_t pieces = static_cast<uint32_t>((a.cols + 7) / 8);
    // a launch holds less than 2^32 threads
    const size_t most = std::max<size_t>(1, (size_t{1} << 31) / pieces);
    FxEmbed part = a;
    for (size_t row = 0; row < a.rows; row += most) {
        part.tokens = a.tokens + row;
        part.positions = a.positions ? a.positions + row : nullptr;
        part.out = a.out + row * a.out_stride;
        part.rows = std::min(most, a.rows - row);
        hipLaunchKernelGGL(fx_embed_kernel, dim3(static_cast<unsigned>((part.rows * pieces + 255) / 256)), dim3(256), 0,
                           c->stream, part, pieces);
        VMX_HIP(c, hipGetLastError());
    }
    return 0;
}

int fx_rotate(Context* c, const FxRotate& a) {
    // a launch holds less than 2^32 threads, of 16 a head at most
    const size_t most = std::max<size_t>(1, (size_t{1} << 27) / a.all_heads);
    FxRotate part = a;
    for (size_t row = 0; row < a.rows; row += most) {
        part.x = a.x + row * a.x_stride;
        part.out = a.out + row * a.out_stride;
        part.positions = a.positions ? a.positions + row : nullptr;
        part.rows = std::min(most, a.rows - row);
        if (a.dim <= 32)
            launch_rotate<4>(c, part);
        else if (a.dim <= 64)
            launch_rotate<8>(c, part);
        else
            launch_rotate<16>(c, part);
        VMX_HIP(c, hipGetLastError());
    }
    return 0;
}

}  // namespace vmx
