// fixed_rows.hip -- row operators of the fixed-point model: the norm with its
// residual addition, and the embedding of tokens and positions.
#include "fixed.hpp"

namespace vmx {
namespace {

using namespace fx;

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
// One workgroup per row; the second pass reads the row again.
__global__ __launch_bounds__(256) void fx_norm_kernel(FxNorm a) {
    __shared__ int64_t part[2][4];
    const size_t row = blockIdx.x;
    const int16_t* x = a.x + row * a.x_stride;
    const int16_t* res = a.residual ? a.residual + row * a.residual_stride : nullptr;
    int64_t s = 0, q = 0;
    for (int j = threadIdx.x; j < a.cols; j += 256) {
        const int h = res ? sat16(x[j] + res[j]) : x[j];
        s += h;
        q += h * h;
    }
    s = wave_sum(s);
    q = wave_sum(q);
    if ((threadIdx.x & 63) == 0) {
        part[0][threadIdx.x >> 6] = s;
        part[1][threadIdx.x >> 6] = q;
    }
    __syncthreads();
    s = a.rms ? 0 : part[0][0] + part[0][1] + part[0][2] + part[0][3];
    q = part[1][0] + part[1][1] + part[1][2] + part[1][3];
    const uint64_t v = static_cast<uint64_t>(a.cols * q - s * s) + a.eps;
    const double below = 2.0 * static_cast<double>(floor_sqrt(v) << a.shift), inv = 1.0 / below;
    for (int j = threadIdx.x; j < a.cols; j += 256) {
        const int h = res ? sat16(x[j] + res[j]) : x[j];
        const double c = static_cast<double>(a.cols * static_cast<int64_t>(h) - s);
        double y = floor_div(2.0 * c * a.gain[j] + 0.5 * below, below, inv);
        if (a.bias) y += a.bias[j];
        a.out[row * a.out_stride + j] = static_cast<int16_t>(__builtin_fmin(__builtin_fmax(y, -32768.0), 32767.0));
        if (a.sum) a.sum[row * a.sum_stride + j] = static_cast<int16_t>(h);
    }
}

// ---- embedding ------------------------------------------------------------------------
// out = sat(rs(table[token] scale, shift) + positions[position]); a token or
// position outside its table adds nothing.
__global__ __launch_bounds__(256) void fx_embed_kernel(FxEmbed a) {
    const size_t row = blockIdx.x;
    const int64_t token = a.tokens[row], place = a.positions ? a.positions[row] : -1;
    const bool word = token >= 0 && static_cast<size_t>(token) < a.vocab;
    const bool where = place >= 0 && static_cast<size_t>(place) < a.position_rows;
    for (int j = threadIdx.x; j < a.cols; j += 256) {
        int64_t v = word ? rounded(static_cast<int64_t>(a.table[token * a.table_stride + j]) * a.scale, a.shift) : 0;
        if (where) v += a.position_table[place * a.position_stride + j];
        a.out[row * a.out_stride + j] = static_cast<int16_t>(sat16(v));
    }
}

}  // namespace

int fx_norm(Context* c, const FxNorm& a) {
    hipLaunchKernelGGL(fx_norm_kernel, dim3(static_cast<unsigned>(a.rows)), dim3(256), 0, c->stream, a);
    VMX_HIP(c, hipGetLastError());
    return 0;
}

int fx_embed(Context* c, const FxEmbed& a) {
    hipLaunchKernelGGL(fx_embed_kernel, dim3(static_cast<unsigned>(a.rows)), dim3(256), 0, c->stream, a);
    VMX_HIP(c, hipGetLastError());
    return 0;
}

}  // namespace vmx
