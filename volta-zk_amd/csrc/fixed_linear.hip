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

// ---- many rows -----------------------------------------------------------------------
// A workgroup of 2 x 2 waves computes a tile of 32 I rows x 32 J columns, each
// wave I x J blocks of 16 x 16.  Along k it takes steps of 64: the step's x rows
// (raw i16) and packed weights go from memory to LDS without passing through
// registers, two steps deep, and a wave splits its x fragments into planes as
// it reads them.  Fragments lie in LDS in the order the lanes read them.
//
// x is copied in pieces of 8 elements when every piece is 16-byte aligned
// (`Aligned`), else through registers.  Places past k of a row's last piece may
// then hold anything: their weights are 0, and the identity of fixed.hpp holds
// for whatever x they have, as the same bytes feed products and sums.
// One 64-bit sum after its rounding shift (whose half is already in it), in 16 bits.
__device__ inline int shifted_sat(int64_t sum, uint32_t shift) {
    const int64_t v = sum >> shift;
    const int lo = static_cast<int>(v), hi = static_cast<int>(v >> 32);
    const int fit = hi == (lo >> 31) ? lo : (hi >> 31) ^ 0x7fffffff;
    return min(max(fit, -32768), 32767);
}

template <int I, int J, bool Aligned>
__global__ __launch_bounds__(256, 2) void fx_linear_tile_kernel(FxLinear a, unsigned row_tiles, unsigned col_tiles) {
    constexpr int BM = 32 * I, BN = 32 * J;
    constexpr int XP = BM / 8, WP = BN / 8;  // KiB pieces of a step
    constexpr int OUT_STRIDE = BN + 8;       // i16 of a row of finished values in LDS
    constexpr int STAGE = (XP + WP) * 1024;
    __shared__ __attribute__((aligned(1024)))
    unsigned char lds[2 * STAGE > BM * OUT_STRIDE * 2 ? 2 * STAGE : BM * OUT_STRIDE * 2];
    __shared__ int x_sum[BM];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave & 1, wn = wave >> 1;
    const int steps = (a.k + 63) / 64, blocks = (a.n + 15) / 16;
    // Workgroups go to the XCDs in turn: each XCD takes a run of neighbouring
    // tiles, so that their rows and columns meet in its L2.
    const unsigned tiles = row_tiles * col_tiles, per = (tiles + 7) / 8;
    const unsigned tile = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (tile >= tiles) return;
    const unsigned rt = tile / col_tiles, ct = tile % col_tiles;
    const size_t row0 = static_cast<size_t>(rt) * BM;
    const int rows = static_cast<int>(a.rows - row0 < BM ? a.rows - row0 : BM);
    const int block0 = static_cast<int>(ct) * (BN / 16);
    const int16_t* x = a.x + row0 * a.x_stride;

    // The pieces a wave copies: x piece p holds, of rows 16 (p >> 1) .., half p & 1
    // of each lane's 16 places; weight piece p is block p >> 1's plane p & 1.
    uint32_t x_at[XP / 4];
#pragma unroll
    for (int i = 0; i < XP / 4; ++i)
        x_at[i] = static_cast<uint32_t>(min(((i * 4 + wave) >> 1) * 16 + (lane & 15), rows - 1) * a.x_stride);
    const uint32_t k_at = 16 * (lane >> 4) + 8 * (wave & 1), k_last = (a.k - 1) & ~7;
    auto stage = [&](int s, unsigned char* to) {
        const uint32_t at = s * 64 + k_at;
#pragma unroll
        for (int i = 0; i < XP / 4; ++i) {
            unsigned char* place = to + (i * 4 + wave) * 1024;
            if constexpr (Aligned) {
                copy_to_lds(x, 2 * (x_at[i] + min(at, k_last)), place);
            } else {
                union {
                    v4i v;
                    int16_t e[8];
                } u;
                u.v = v4i{0, 0, 0, 0};
                const int16_t* from = x + min(((i * 4 + wave) >> 1) * 16 + (lane & 15), rows - 1) * a.x_stride + at;
                if (at + 8 <= static_cast<uint32_t>(a.k)) {
                    u.v = load8(from);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (at + e < static_cast<uint32_t>(a.k)) u.e[e] = from[e];
                }
                *reinterpret_cast<v4i*>(place + lane * 16) = u.v;
            }
        }
#pragma unroll
        for (int i = 0; i < WP / 4; ++i) {
            const int p = i * 4 + wave, b = min(block0 + (p >> 1), blocks - 1);
            copy_to_lds(a.weights + (static_cast<size_t>(b) * steps + s) * 2048 + (p & 1) * 1024, lane * 16,
                        to + (XP + p) * 1024);
        }
    };

    v4i hh[I][J] = {}, mid[I][J] = {}, ll[I][J] = {};
    int sums[I] = {};
    stage(0, lds);
    for (int s = 0; s < steps; ++s) {
        lds_copies_done();
        __syncthreads();  // this step's copies have landed for all waves, and all have left the other buffer
        if (s + 1 < steps) stage(s + 1, lds + ((s + 1) & 1) * STAGE);
        const unsigned char* now = lds + (s & 1) * STAGE;
        const v4i* xs = reinterpret_cast<const v4i*>(now) + wm * I * 128 + lane;
        const v4i* ws = reinterpret_cast<const v4i*>(now + XP * 1024) + wn * J * 128 + lane;
        v4i wh[J], wl[J];
#pragma unroll
        for (int j = 0; j < J; ++j) wh[j] = ws[j * 128], wl[j] = ws[j * 128 + 64];
#pragma unroll
        for (int i = 0; i < I; ++i) {
            const v4i x0 = xs[i * 128], x1 = xs[i * 128 + 64];
            sums[i] = sum8(x1, sum8(x0, sums[i]));
            v4i xh, xl;
            split16(x0, x1, &xh, &xl);
#pragma unroll
            for (int j = 0; j < J; ++j) {
                hh[i][j] = mfma(xh, wh[j], hh[i][j]);
                mid[i][j] = mfma(xh, wl[j], mid[i][j]);
                ll[i][j] = mfma(xl, wl[j], ll[i][j]);
            }
#pragma unroll
            for (int j = 0; j < J; ++j) mid[i][j] = mfma(xl, wh[j], mid[i][j]);
        }
    }
    if (wn == 0) {
#pragma unroll
        for (int i = 0; i < I; ++i) {
            int t = sums[i];
            t += __shfl_xor(t, 16);
            t += __shfl_xor(t, 32);
            if (lane < 16) x_sum[(wm * I + i) * 16 + lane] = t;
        }
    }
    __syncthreads();  // and the last step's buffer is free

    const int64_t* offs = reinterpret_cast<const int64_t*>(a.weights + static_cast<size_t>(blocks) * steps * 2048);
    int16_t* done = reinterpret_cast<int16_t*>(lds);
    // The sums of every place, with the column's constant and the row's.
    auto each = [&](auto&& use) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int col = (block0 + wn * J + j) * 16 + (lane & 15);
            int64_t off = col < a.n ? offs[col] : 0;
            if (a.bias && col < a.n) off += static_cast<int64_t>(a.bias[col]) << a.bias_shift;
            if (!a.raw && a.shift) off += int64_t{1} << (a.shift - 1);
#pragma unroll
            for (int i = 0; i < I; ++i) {
                const int at = (wm * I + i) * 16 + 4 * (lane >> 4);
                const v4i xs = *reinterpret_cast<const v4i*>(x_sum + at);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    use(at + r, (wn * J + j) * 16 + (lane & 15),
                        join(hh[i][j][r], mid[i][j][r], ll[i][j][r]) + off + (static_cast<int64_t>(xs[r]) << 7));
            }
        }
    };
    if (a.raw) {
        int64_t* out = static_cast<int64_t*>(a.out) + row0 * a.out_stride + block0 * 16;
        const int cols = a.n - block0 * 16;
        each([&](int row, int col, int64_t sum) {
            if (row < rows && col < cols) out[row * a.out_stride + col] = sum;
        });
        return;
    }
    each([&](int row, int col, int64_t sum) {
        done[row * OUT_STRIDE + col] = static_cast<int16_t>(shifted_sat(sum, a.shift));
    });
    __syncthreads();
    // Rows of finished values, eight columns a thread.
    for (int i = threadIdx.x; i < BM * (BN / 8); i += 256) {
        const int row = i / (BN / 8), at = i % (BN / 8) * 8, col = block0 * 16 + at;
        if (row >= rows || col >= a.n) continue;
        union {
            v4i v;
            int16_t e[8];
        } u, res;
        u.v = *reinterpret_cast<const v4i*>(done + row * OUT_STRIDE + at);
        const int live = min(a.n - col, 8);
        if (a.table) {
#pragma unroll
            for (int e = 0; e < 8; ++e) u.e[e] = a.table[u.e[e] + 32768];
        }
        int16_t* out = static_cast<int16_t*>(a.out) + (row0 + row) * a.out_stride + col;
        const int16_t* from = a.residual + (row0 + row) * a.residual_stride + col;
        if (live == 8) {
            if (a.residual) {
                res.v = load8(from);
#pragma unroll
                for (int e = 0; e < 8; ++e) u.e[e] = static_cast<int16_t>(min(max(u.e[e] + res.e[e], -32768), 32767));
            }
            reinterpret_cast<Row16*>(out)->v = u.v;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < live)
                    out[e] = static_cast<int16_t>(a.residual ? min(max(u.e[e] + from[e], -32768), 32767) : u.e[e]);
        }
    }
}

template <int I, int J>
void launch_tile(Context* c, const FxLinear& a) {
    // Aligned also needs a tile's offsets to fit 32 bits.
    const bool aligned =
        reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.x_stride % 8 == 0 && a.x_stride < (size_t{1} << 23);
    const unsigned rt = static_cast<unsigned>((a.rows + 32 * I - 1) / (32 * I));
    const unsigned ct = static_cast<unsigned>((a.n + 32 * J - 1) / (32 * J));
    const dim3 grid((rt * ct + 7) / 8 * 8);
    if (aligned)
        hipLaunchKernelGGL((fx_linear_tile_kernel<I, J, true>), grid, dim3(256), 0, c->stream, a, rt, ct);
    else
        hipLaunchKernelGGL((fx_linear_tile_kernel<I, J, false>), grid, dim3(256), 0, c->stream, a, rt, ct);
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
    if (a.rows > 64) {
        launch_tile<4, 4>(c, a);
        VMX_HIP(c, hipGetLastError());
        return 0;
    }
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
