// fixed_linear.hip -- out = epilogue(x w): 16-bit integer matrix product on the
// i8 matrix cores (fixed.hpp has the identity) with bias, rounding shift,
// activation table and residual applied to the sums in registers.
#include "fixed.hpp"

namespace vmx {
namespace {

using namespace fx;

// ---- packing -------------------------------------------------------------------------
// One workgroup per 16 columns; its waves take the steps of 64 rows in turn.
__global__ __launch_bounds__(256) void fx_pack_weights_kernel(const int16_t* w, int k, int n, size_t stride,
                                                              bool transposed, unsigned char* out, size_t blocks) {
    __shared__ int part[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const size_t block = blockIdx.x;
    const int col = static_cast<int>(block * 16) + (lane & 15);
    const int steps = (k + 63) / 64;
    v4i* dst = reinterpret_cast<v4i*>(out + block * steps * 2048) + lane;
    int sum = 0;
    for (int s = wave; s < steps; s += 4) {
        const int at = s * 64 + 16 * (lane >> 4);
        union {
            v4i v[2];
            int16_t e[16];
        } u;
        u.v[0] = v4i{0, 0, 0, 0};
        u.v[1] = v4i{0, 0, 0, 0};
        if (col < n) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (at + i < k) u.e[i] = transposed ? w[col * stride + at + i] : w[(at + i) * stride + col];
        }
        sum = sum8(u.v[1], sum8(u.v[0], sum));
        v4i h, l;
        split16(u.v[0], u.v[1], &h, &l);
        dst[s * 128] = h;
        dst[s * 128 + 64] = l;
    }
    part[wave][lane] = sum;
    __syncthreads();
    if (threadIdx.x < 16) {
        int64_t total = 0;
        for (int g = 0; g < 4; ++g)
            for (int v = 0; v < 4; ++v) total += part[v][g * 16 + lane];
        int64_t* offs = reinterpret_cast<int64_t*>(out + blocks * steps * 2048);
        offs[block * 16 + lane] = 128 * (total - int64_t{128} * 64 * steps);
    }
}

// ---- epilogue ------------------------------------------------------------------------
__device__ inline void finish(const FxLinear& a, size_t row, int col, int64_t sum) {
    if (a.bias) sum += static_cast<int64_t>(a.bias[col]) << a.bias_shift;
    if (a.raw) {
        static_cast<int64_t*>(a.out)[row * a.out_stride + col] = sum;
        return;
    }
    int h = sat16(rounded(sum, a.shift));
    if (a.table) h = a.table[h + 32768];
    if (a.residual) h = sat16(h + a.residual[row * a.residual_stride + col]);
    static_cast<int16_t*>(a.out)[row * a.out_stride + col] = static_cast<int16_t>(h);
}

// ---- few rows ------------------------------------------------------------------------
// A workgroup computes MB * 16 rows of 16 columns; its waves take the steps of
// 64 along k in turn, each streaming its part of the packed weights once, and
// add their i64 sums in LDS.
template <int MB>
__global__ __launch_bounds__(1024) void fx_linear_rows_kernel(FxLinear a) {
    __shared__ unsigned long long total[MB * 256];
    __shared__ int x_sum[MB * 16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int steps = (a.k + 63) / 64, col0 = blockIdx.x * 16;
    const size_t row0 = static_cast<size_t>(blockIdx.y) * (MB * 16);
    for (int i = threadIdx.x; i < MB * 256; i += blockDim.x) total[i] = 0;
    for (int i = threadIdx.x; i < MB * 16; i += blockDim.x) x_sum[i] = 0;
    __syncthreads();
    const v4i* w = reinterpret_cast<const v4i*>(a.weights + static_cast<size_t>(blockIdx.x) * steps * 2048) + lane;
    v4i hh[MB] = {}, mid[MB] = {}, ll[MB] = {};
    int sums[MB] = {};
    for (int s = wave; s < steps; s += waves) {
        const v4i wh = w[s * 128], wl = w[s * 128 + 64];
#pragma unroll
        for (int b = 0; b < MB; ++b) {
            const size_t row = row0 + b * 16 + (lane & 15);
            v4i x0 = {}, x1 = {}, xh, xl;
            if (row < a.rows) load16(a.x + row * a.x_stride, s * 64 + 16 * (lane >> 4), a.k, &x0, &x1);
            sums[b] = sum8(x1, sum8(x0, sums[b]));
            split16(x0, x1, &xh, &xl);
            hh[b] = mfma(xh, wh, hh[b]);
            mid[b] = mfma(xh, wl, mid[b]);
            ll[b] = mfma(xl, wl, ll[b]);
            mid[b] = mfma(xl, wh, mid[b]);
        }
    }
#pragma unroll
    for (int b = 0; b < MB; ++b) {
        atomicAdd(&x_sum[b * 16 + (lane & 15)], sums[b]);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            atomicAdd(&total[b * 256 + (4 * (lane >> 4) + r) * 16 + (lane & 15)],
                      static_cast<unsigned long long>(join(hh[b][r], mid[b][r], ll[b][r])));
    }
    __syncthreads();
    const int64_t* offs =
        reinterpret_cast<const int64_t*>(a.weights + static_cast<size_t>(gridDim.x) * steps * 2048) + col0;
    for (int i = threadIdx.x; i < MB * 256; i += blockDim.x) {
        const size_t row = row0 + (i >> 4);
        const int col = col0 + (i & 15);
        if (row < a.rows && col < a.n)
            finish(a, row, col,
                   static_cast<int64_t>(total[i]) + offs[i & 15] + 128 * static_cast<int64_t>(x_sum[i >> 4]));
    }
}

}  // namespace

int fx_pack_weights(Context* c, const int16_t* w, size_t k, size_t n, size_t stride, bool transposed, void* out) {
    const size_t blocks = fx_blocks(n);
    hipLaunchKernelGGL(fx_pack_weights_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, c->stream, w,
                       static_cast<int>(k), static_cast<int>(n), stride, transposed, static_cast<unsigned char*>(out),
                       blocks);
    VMX_HIP(c, hipGetLastError());
    return 0;
}

int fx_linear(Context* c, const FxLinear& a) {
    const size_t blocks = fx_blocks(a.n), steps = fx_steps(a.k);
    const unsigned waves = static_cast<unsigned>(steps < 16 ? steps : 16);
    const int mb = a.rows <= 16 ? 1 : a.rows <= 32 ? 2 : 4;
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>((a.rows + 16 * mb - 1) / (16 * mb)));
    const dim3 threads(64 * waves);
    if (mb == 1)
        hipLaunchKernelGGL(fx_linear_rows_kernel<1>, grid, threads, 0, c->stream, a);
    else if (mb == 2)
        hipLaunchKernelGGL(fx_linear_rows_kernel<2>, grid, threads, 0, c->stream, a);
    else
        hipLaunchKernelGGL(fx_linear_rows_kernel<4>, grid, threads, 0, c->stream, a);
    VMX_HIP(c, hipGetLastError());
    return 0;
}

}  // namespace vmx
