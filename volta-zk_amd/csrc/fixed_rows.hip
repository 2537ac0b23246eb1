// fixed_rows.hip -- row operators of the fixed-point model: the norm with its
// residual addition, and the embedding of tokens and positions.  Both are bound
// by memory: eight elements a thread at a time, whatever the rows' alignment.
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

}  // namespace vmx
