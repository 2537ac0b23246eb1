// fixed_rows.hip -- row operators of the fixed-point model: the norm with its
// residual addition, and the embedding of tokens and positions.  Both are bound
// by memory: eight elements a thread at a time, whatever the rows' alignment.
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

__device__ inline int64_t wave_sum(int64_t v) {
    for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
    return v;
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
// length, read twice).  |n h - S| <= 2^32 and B < 2^47, so every value of the
// division is a whole number below 2^53: doubles hold it exactly.
//
// 16,384 rows of 768 with a residual, its sum kept (100 MB): a row a wave 28 us
// (3.6 TB/s), a row a workgroup and elements one by one 57 us.
template <int THREADS, int KEPT>
__global__ __launch_bounds__(256) void fx_norm_kernel(FxNorm a) {
    constexpr int WAVES = THREADS / 64;
    __shared__ int64_t part[2][4];
    const size_t row = static_cast<size_t>(blockIdx.x) * (256 / THREADS) + threadIdx.x / THREADS;
    const int thread = threadIdx.x % THREADS;
    if (WAVES == 1 && row >= a.rows) return;
    const int16_t* x = a.x + row * a.x_stride;
    const int16_t* res = a.residual ? a.residual + row * a.residual_stride : nullptr;
    auto piece = [&](int at) {
        const v4i v = load8(x, at, a.cols);
        return res ? add_sat(v, load8(res, at, a.cols)) : v;
    };
    int64_t s = 0;
    uint64_t q = 0;
    auto count = [&](v4i v) {
        int some = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int pair = v[i];
            const v2s two = __builtin_bit_cast(v2s, pair);
            some = __builtin_amdgcn_sdot2(two, v2s{1, 1}, some, false);
            q += static_cast<uint32_t>(__builtin_amdgcn_sdot2(two, two, 0, false));  // at most 2^31
        }
        s += some;
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
    s = wave_sum(s);
    q = static_cast<uint64_t>(wave_sum(static_cast<int64_t>(q)));
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) {
            part[0][threadIdx.x >> 6] = s;
            part[1][threadIdx.x >> 6] = static_cast<int64_t>(q);
        }
        __syncthreads();
        s = part[0][0] + part[0][1] + part[0][2] + part[0][3];
        q = static_cast<uint64_t>(part[1][0] + part[1][1] + part[1][2] + part[1][3]);
    }
    if (a.rms) s = 0;
    const uint64_t v = static_cast<uint64_t>(a.cols) * q - static_cast<uint64_t>(s * s) + a.eps;
    const double below = 2.0 * static_cast<double>(floor_sqrt(v) << a.shift), inv = 1.0 / below;
    const double n = a.cols, sum = static_cast<double>(s);
    auto finish = [&](int at, v4i h) {
        Eight hu, gu, bu, out;
        hu.v = h;
        gu.v = load8(a.gain, at, a.cols);
        bu.v = a.bias ? load8(a.bias, at, a.cols) : v4i{0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const double c = __builtin_fma(n, static_cast<double>(hu.e[e]), -sum);
            const double y = floor_div(__builtin_fma(c, 2.0 * gu.e[e], 0.5 * below), below, inv) + bu.e[e];
            out.e[e] = static_cast<int16_t>(__builtin_fmin(__builtin_fmax(y, -32768.0), 32767.0));
        }
        store8(a.out + row * a.out_stride, at, a.cols, out.v);
        if (a.sum) store8(a.sum + row * a.sum_stride, at, a.cols, h);
    };
    if constexpr (KEPT > 0) {
#pragma unroll
        for (int i = 0; i < KEPT; ++i) {
            const int at = (i * THREADS + thread) * 8;
            if (at < a.cols) finish(at, kept[i]);
        }
    } else {
        // a sum over x or the residual is written by the thread that has read it
        for (int at = thread * 8; at < a.cols; at += THREADS * 8) finish(at, piece(at));
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
    const size_t rows = 256 / THREADS;
    hipLaunchKernelGGL((fx_norm_kernel<THREADS, KEPT>), dim3(static_cast<unsigned>((a.rows + rows - 1) / rows)), dim3(256), 0,
                       c->stream, a);
}

}  // namespace

int fx_norm(Context* c, const FxNorm& a) {
    if (a.cols <= 512)
        launch_norm<64, 1>(c, a);
    else if (a.cols <= 1024)
        launch_norm<64, 2>(c, a);
    else if (a.cols <= 2048)
        launch_norm<256, 1>(c, a);
    else if (a.cols <= 8192)
        launch_norm<256, 4>(c, a);
    else
        launch_norm<256, 0>(c, a);
    VMX_HIP(c, hipGetLastError());
    return 0;
}

int fx_embed(Context* c, const FxEmbed& a) {
    const uint32_t pieces = static_cast<uint32_t>((a.cols + 7) / 8);
    hipLaunchKernelGGL(fx_embed_kernel, dim3(static_cast<unsigned>((a.rows * pieces + 255) / 256)), dim3(256), 0, c->stream, a,
                       pieces);
    VMX_HIP(c, hipGetLastError());
    return 0;
}

}  // namespace vmx
