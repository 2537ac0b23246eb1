// fixed_linear.hip -- out = epilogue(x w): 16-bit integer matrix product on the
// i8 matrix cores (fixed.hpp has the identity) with bias, rounding shift,
// activation table and residual applied to the sums in registers.
#include <algorithm>

#include "fixed.hpp"

namespace vmx {
namespace {

using namespace fx;

// ---- packing -------------------------------------------------------------------------
// One workgroup per 16 columns: once for their largest value, then its waves
// take the steps of 64 rows in turn.  Done once for a model's weights; bound by
// latency where columns are few: 3,072 x 768 (4.7 MB) 27 us on 48 workgroups (17 in
// a loop, from the caches), 768 x 50,257 (77 MB) 110 us, 1.4 TB/s read plus written.
// Transposed weights are read two bytes a lane, rows apart: 45 us in a loop and 144.
__global__ __launch_bounds__(1024) void fx_pack_weights_kernel(const int16_t* w, int k, int n, size_t stride,
                                                               bool transposed, unsigned char* out, size_t blocks) {
    __shared__ int most;
    __shared__ unsigned long long sums[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const size_t block = blockIdx.x;
    const int col = static_cast<int>(block * 16) + (lane & 15);
    const int steps = (k + 63) / 64;
    auto at = [&](int row) -> int {
        return col < n && row < k ? (transposed ? w[col * stride + row] : w[row * stride + col]) : 0;
    };
    if (threadIdx.x == 0) most = 0;
    if (threadIdx.x < 16) sums[threadIdx.x] = 0;
    __syncthreads();
    int largest = 0;
    for (int row = threadIdx.x >> 4; row < k; row += 64) largest = max(largest, at(row));
    for (int m = 32; m; m >>= 1) largest = max(largest, __shfl_xor(largest, m));
    if (lane == 0) atomicMax(&most, largest);
    __syncthreads();
    const int off = most > HALVES_MAX ? 128 : 0;
    unsigned char* dst = out + block * steps * 2048 + lane * 16;
    int sum = 0;
    for (int s = wave; s < steps; s += 16) {
        union {
            v4i v;
            uint8_t b[16];
        } h, l;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int v = at(s * 64 + 16 * (lane >> 4) + i) - off, p = halves(v);
            sum += v;
            h.b[i] = static_cast<uint8_t>(p >> 8);
            l.b[i] = static_cast<uint8_t>(p);
        }
        *reinterpret_cast<v4i*>(dst + s * 2048) = h.v;
        *reinterpret_cast<v4i*>(dst + s * 2048 + 1024) = l.v;
    }
    atomicAdd(&sums[lane & 15], static_cast<unsigned long long>(static_cast<int64_t>(sum)));
    __syncthreads();
    if (threadIdx.x < 16) {
        int64_t* columns = reinterpret_cast<int64_t*>(out + blocks * steps * 2048);
        columns[block * 16 + lane] = 128 * static_cast<int64_t>(sums[lane]);
        if (threadIdx.x == 0) reinterpret_cast<int*>(columns + blocks * 16)[block] = off;
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
// A workgroup computes 16 rows of 16 columns; its waves take the steps of 64
// along k in turn, each streaming its part of the packed weights once, and add
// their i64 sums in LDS.  Bound by the weights: 7 rows of 768 x 50,257 (77 MB, and
// 2.8 MB of sums) 13.8 us, 5.8 TB/s, as the weights stay in the last-level cache;
// one row of 3,072 x 768 4.6 us, a launch and one trip to memory a step.
__global__ __launch_bounds__(1024) void fx_linear_rows_kernel(FxLinear a) {
    __shared__ unsigned long long total[256];
    __shared__ int x_sum[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int steps = (a.k + 63) / 64, col0 = blockIdx.x * 16;
    const size_t row0 = static_cast<size_t>(blockIdx.y) * 16, row = row0 + (lane & 15);
    for (int i = threadIdx.x; i < 256; i += blockDim.x) total[i] = 0;
    if (threadIdx.x < 16) x_sum[threadIdx.x] = 0;
    __syncthreads();
    const v4i* w = reinterpret_cast<const v4i*>(a.weights + static_cast<size_t>(blockIdx.x) * steps * 2048) + lane;
    v4i hh = {}, mid = {}, ll = {};
    int sum = 0;
    for (int s = wave; s < steps; s += waves) {
        const v4i wh = w[s * 128], wl = w[s * 128 + 64];
        v4i x0 = {}, x1 = {}, xh, xl;
        if (row < a.rows) load16(a.x + row * a.x_stride, s * 64 + 16 * (lane >> 4), a.k, &x0, &x1);
        sum = sum8(x1, sum8(x0, sum));
        split16(x0, x1, &xh, &xl);
        hh = mfma(xh, wh, hh);
        mid = mfma(xh, wl, mid);
        ll = mfma(xl, wl, ll);
        mid = mfma(xl, wh, mid);
    }
    atomicAdd(&x_sum[lane & 15], sum);
#pragma unroll
    for (int r = 0; r < 4; ++r)
        atomicAdd(&total[(4 * (lane >> 4) + r) * 16 + (lane & 15)],
                  static_cast<unsigned long long>(join(hh[r], mid[r], ll[r])));
    __syncthreads();
    const int64_t* offs = reinterpret_cast<const int64_t*>(a.weights + static_cast<size_t>(gridDim.x) * steps * 2048);
    const int64_t off = reinterpret_cast<const int*>(offs + static_cast<size_t>(gridDim.x) * 16)[blockIdx.x];
    for (int i = threadIdx.x; i < 256; i += blockDim.x) {
        const int col = col0 + (i & 15);
        if (row0 + (i >> 4) < a.rows && col < a.n)
            finish(a, row0 + (i >> 4), col, static_cast<int64_t>(total[i]) + offs[col] + off * x_sum[i >> 4]);
    }
}

// ---- rows that are not aligned ---------------------------------------------------------
// x with rows of whole 16-byte pieces, a piece a thread.  What a row's last piece
// holds past k is 0.
__global__ __launch_bounds__(256) void fx_align_rows_kernel(const int16_t* x, size_t stride, size_t rows, int k,
                                                            uint32_t pieces, v4i* out) {
    const size_t id = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x, row = id / pieces;
    if (row >= rows) return;
    const int at = static_cast<int>(id - row * pieces) * 8;
    const int16_t* from = x + row * stride + at;
    union {
        v4i v;
        int16_t e[8];
    } u;
    u.v = v4i{0, 0, 0, 0};
    if (at + 8 <= k) {
        u.v = load8(from);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (at + e < k) u.e[e] = from[e];
    }
    out[id] = u.v;
}

// ---- many rows -----------------------------------------------------------------------
// A workgroup of WM x WN waves computes a tile of 32 WM I rows x 32 WN J
// columns, each wave I x J blocks of 32 x 32.  Along k it takes steps of 64: the
// step's x rows (raw i16) and packed weights go from memory to LDS without
// passing through registers, STAGES - 1 steps ahead, and a wave splits its x
// fragments into planes as it reads them.  Fragments lie in LDS in the order the
// lanes read them.
//
// Large products: 16,384 x 768 x 4,096 takes 202 to 220 us, 1.9 to 2.0 POP/s of i8
// work (a library i8 product of 16,384^3 reaches 2.33).  Matrix cores are busy 0.46 of
// its cycles; a tile a CU takes 13 us, of which 4.7 are its start and end (the estimate
// in launch_product; the other workgroup of the CU hides part of both), and within the
// steps waves wait for one another and for copies.  The clock falls with the data: 2.06 GHz here, and on weights of zero
// 186 of then 235 us.  Weights over 32,639, whose row sums of x are taken in every step:
// one in a tile 210 and one in each block 224 us where 203 without, seven rows of 768 x
// 50,257 14.0 with and without.
// At one tile a CU the steps' waits bound it: 1,023 x 768 x 3,072 17.7 us, 20.8 with a
// table, whose lookups are bound by their rate (four times as many under way together
// took as long); matrix cores busy 0.14.
//
// x is copied in pieces of 8 elements when every piece is 16-byte aligned
// (`Aligned`), else through registers.  Places past k of a row's last piece may
// then hold anything: their weights are 0, and the identity of fixed.hpp holds
// for whatever x they have, as the same bytes feed products and sums.
template <int WM, int WN, int I, int J, int STAGES, bool Aligned>
__global__ __launch_bounds__(64 * WM * WN, 2) void fx_linear_tile_kernel(FxLinear a, unsigned row_tiles,
                                                                         unsigned col_tiles) {
    constexpr int BM = 32 * WM * I, BN = 32 * WN * J, WAVES = WM * WN;
    constexpr int XP = BM / 8, WP = BN / 8;  // KiB pieces of a step
    static_assert(XP % WAVES == 0 && WP % WAVES == 0 && WAVES % 2 == 0, "equal shares of copies");
    constexpr int OUT_STRIDE = BN + 8;       // i16 of a row of finished values in LDS
    constexpr int STAGE = (XP + WP) * 1024;
    __shared__ __attribute__((aligned(1024)))
    unsigned char lds[STAGES * STAGE > BM * OUT_STRIDE * 2 ? STAGES * STAGE : BM * OUT_STRIDE * 2];
    __shared__ int x_sum[BM];
    __shared__ int64_t column[BN];
    static_assert(BN <= 64 * WAVES, "a column a thread");
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave % WM, wn = wave / WM;
    const int steps = (a.k + 63) / 64, blocks = (a.n + 15) / 16;
    // Workgroups go to the XCDs in turn: each XCD takes a run of tiles, which go
    // down panels of 1,024 columns, so that what its CUs work on at one time shares
    // rows and columns in its L2 (16,384 x 768 x 4,096 by whole rows of tiles, whose
    // 6.3 MB of weights an L2 does not hold: 212 us, by panels 202).
    constexpr unsigned PANEL = 1024 / BN;
    const unsigned tiles = row_tiles * col_tiles, per = (tiles + 7) / 8;
    const unsigned tile = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (tile >= tiles) return;
    const unsigned panel = tile / (PANEL * row_tiles), place = tile - panel * PANEL * row_tiles;
    const unsigned across = min(PANEL, col_tiles - panel * PANEL);
    const unsigned rt = place / across, ct = panel * PANEL + place % across;
    const size_t row0 = static_cast<size_t>(rt) * BM;
    const int rows = static_cast<int>(a.rows - row0 < BM ? a.rows - row0 : BM);
    const int block0 = static_cast<int>(ct) * (BN / 16);
    const int16_t* x = a.x + row0 * a.x_stride;

    // The pieces a wave copies: x piece p holds, of rows 16 (p >> 1) .., half p & 1
    // of each lane's 16 places; weight piece p is block p >> 1's plane p & 1.
    uint32_t x_at[XP / WAVES];
#pragma unroll
    for (int i = 0; i < XP / WAVES; ++i)
        x_at[i] = static_cast<uint32_t>(min(((i * WAVES + wave) >> 1) * 16 + (lane & 15), rows - 1) * a.x_stride);
    const uint32_t k_at = 16 * (lane >> 4) + 8 * (wave & 1), k_last = (a.k - 1) & ~7;
    auto stage = [&](int s, unsigned char* to) {
        const uint32_t at = s * 64 + k_at;
#pragma unroll
        for (int i = 0; i < XP / WAVES; ++i) {
            unsigned char* place = to + (i * WAVES + wave) * 1024;
            if constexpr (Aligned) {
                copy_to_lds(x, 2 * (x_at[i] + min(at, k_last)), place);
            } else {
                union {
                    v4i v;
                    int16_t e[8];
                } u;
                u.v = v4i{0, 0, 0, 0};
                const int16_t* from = x + min(((i * WAVES + wave) >> 1) * 16 + (lane & 15), rows - 1) * a.x_stride + at;
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
        for (int i = 0; i < WP / WAVES; ++i) {
            const int p = i * WAVES + wave, b = min(block0 + (p >> 1), blocks - 1);
            copy_to_lds(a.weights + (static_cast<size_t>(b) * steps + s) * 2048 + (p & 1) * 1024, lane * 16,
                        to + (XP + p) * 1024);
        }
    };

    const int64_t* offs = reinterpret_cast<const int64_t*>(a.weights + static_cast<size_t>(blocks) * steps * 2048);
    const int* o = reinterpret_cast<const int*>(offs + static_cast<size_t>(blocks) * 16);
    // On their way before the first copies, awaited after them: whether a weight of
    // the tile needed its offset, and the columns' constants.
    const int lane_o = lane < BN / 16 && block0 + lane < blocks ? o[block0 + lane] : 0;
    const int my_col = block0 * 16 + static_cast<int>(threadIdx.x);
    int64_t mine = 0;
    int bias = 0;
    if (threadIdx.x < BN && my_col < a.n) {
        mine = offs[my_col];
        if (a.bias) bias = a.bias[my_col];
    }

    // A lane's fragment of 32 rows (or columns) and half u of the step: its row is
    // lane & 31, its 16 places start at 32 u + 16 (lane >> 5).
    const int in_block = ((lane >> 4) & 1) * 128 + (lane >> 5) * 16 + (lane & 15);
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s)
        if (s < steps) stage(s, lds + s * STAGE);
    const bool offset = __any(lane_o);  // then row sums of x are needed
    if (threadIdx.x < BN) {
        mine += static_cast<int64_t>(bias) << a.bias_shift;
        column[threadIdx.x] = !a.raw && a.shift ? mine + (int64_t{1} << (a.shift - 1)) : mine;
    }
    v16i hh[I][J] = {}, mid[I][J] = {}, ll[I][J] = {};
    int sums[I] = {};
    int now_at = 0, next_at = (STAGES - 1) * STAGE;
    for (int s = 0; s < steps; ++s) {
        // This step's copies have landed for all waves, and all have left the
        // buffer of the step before.
        if (Aligned && s + STAGES - 2 < steps)
            lds_copies_done<(STAGES - 2) * (XP + WP) / WAVES>();
        else
            lds_copies_done<0>();
        __syncthreads();
        if (s + STAGES - 1 < steps) stage(s + STAGES - 1, lds + next_at);
        const unsigned char* now = lds + now_at;
        next_at = now_at;
        now_at = now_at + STAGE == STAGES * STAGE ? 0 : now_at + STAGE;
        const v4i* xs = reinterpret_cast<const v4i*>(now) + wm * I * 256 + in_block;
        const v4i* ws = reinterpret_cast<const v4i*>(now + XP * 1024) + wn * J * 256 + in_block;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            v4i wh[J], wl[J];
#pragma unroll
            for (int j = 0; j < J; ++j) wh[j] = ws[j * 256 + u * 32], wl[j] = ws[j * 256 + 64 + u * 32];
#pragma unroll
            for (int i = 0; i < I; ++i) {
                const v4i x0 = xs[i * 256 + u * 32], x1 = xs[i * 256 + 64 + u * 32];
                if (offset) sums[i] = sum8(x1, sum8(x0, sums[i]));
                v4i xh, xl;
                split16(x0, x1, &xh, &xl);
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    hh[i][j] = mfma32(xh, wh[j], hh[i][j]);
                    mid[i][j] = mfma32(xh, wl[j], mid[i][j]);
                    ll[i][j] = mfma32(xl, wl[j], ll[i][j]);
                }
#pragma unroll
                for (int j = 0; j < J; ++j) mid[i][j] = mfma32(xl, wh[j], mid[i][j]);
            }
        }
    }
    if (wn == 0) {
#pragma unroll
        for (int i = 0; i < I; ++i) {
            const int t = sums[i] + __shfl_xor(sums[i], 32);
            if (lane < 32) x_sum[(wm * I + i) * 32 + lane] = t;
        }
    }
    __syncthreads();  // and the last step's buffer is free

    int16_t* done = reinterpret_cast<int16_t*>(lds);
    if (offset) {
        // 128 sum x, as 2^16 (sum >> 9) + 2^7 (sum & 511), joins the outer sums
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int col = block0 * 16 + (wn * J + j) * 32 + (lane & 31), mask = col < a.n && o[col >> 4] ? -1 : 0;
#pragma unroll
            for (int i = 0; i < I; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int sum = x_sum[(wm * I + i) * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)] & mask;
                    hh[i][j][r] += sum >> 9;
                    ll[i][j][r] += (sum & 511) << 7;
                }
        }
    }
    // Every place with its three sums and its column's constant.
    auto each = [&](auto&& use) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int place = (wn * J + j) * 32 + (lane & 31);
            if (block0 * 16 + place >= a.n) continue;
            const int64_t off = column[place];
#pragma unroll
            for (int i = 0; i < I; ++i) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int row = (wm * I + i) * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
                    use(row, place, hh[i][j][r], mid[i][j][r], ll[i][j][r], off);
                }
            }
        }
    };
    if (a.raw) {
        int64_t* out = static_cast<int64_t*>(a.out) + row0 * a.out_stride + block0 * 16;
        const int cols = a.n - block0 * 16;
        each([&](int row, int col, int h, int m, int l, int64_t off) {
            if (row < rows && col < cols) out[row * a.out_stride + col] = join(h, m, l) + off;
        });
        return;
    }
    if (a.shift <= 45 && a.bias_shift <= 29) {
        // Constants below 2^45 + 2^39 (bias, half of the shift's step, 128 sum W): with
        // off = 2^16 A + B the sum is 2^16 high + low, 0 <= low < 2^16 and high, below
        // 2^30 + 2^29 + 2^25 in size, in 32 bits, and its shift needs no 64-bit
        // arithmetic (under a shift below 16, high is clamped first: past 15 bits
        // the result is clamped whatever they are).
        auto put = [&](int row, int col, int v) {
            done[row * OUT_STRIDE + col] = static_cast<int16_t>(min(max(v, -32768), 32767));
        };
        auto low = [](int m, int l, int64_t off) { return ((m & 255) << 8) + l + static_cast<int>(off & 0xffff); };
        auto high = [](int h, int m, int t, int64_t off) {
            return h + (m >> 8) + static_cast<int>(off >> 16) + (t >> 16);
        };
        if (a.shift >= 16) {
            const uint32_t more = a.shift - 16;
            each([&](int row, int col, int h, int m, int l, int64_t off) {
                put(row, col, high(h, m, low(m, l, off), off) >> more);
            });
        } else {
            const uint32_t up = 16 - a.shift;
            each([&](int row, int col, int h, int m, int l, int64_t off) {
                const int t = low(m, l, off);
                put(row, col, (min(max(high(h, m, t, off), -32768), 32767) << up) + ((t & 0xffff) >> a.shift));
            });
        }
    } else {
        each([&](int row, int col, int h, int m, int l, int64_t off) {
            done[row * OUT_STRIDE + col] = static_cast<int16_t>(sat16((join(h, m, l) + off) >> a.shift));
        });
    }
    __syncthreads();
    // Rows of finished values, eight columns a thread.
    for (int i = threadIdx.x; i < BM * (BN / 8); i += 64 * WAVES) {
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

// Whether the tile kernel may copy x in pieces; a tile's offsets have to fit 32 bits.
bool aligned_rows(const FxLinear& a) {
    return reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.x_stride % 8 == 0 && a.x_stride < (size_t{1} << 22);
}

template <int WM, int WN, int I, int J, int STAGES>
void launch_tile(Context* c, const FxLinear& a) {
    const bool aligned = aligned_rows(a);
    constexpr int BM = 32 * WM * I, BN = 32 * WN * J;
    const unsigned rt = static_cast<unsigned>((a.rows + BM - 1) / BM), ct = static_cast<unsigned>((a.n + BN - 1) / BN);
    const dim3 grid((rt * ct + 7) / 8 * 8), threads(64 * WM * WN);
    if (aligned)
        hipLaunchKernelGGL((fx_linear_tile_kernel<WM, WN, I, J, STAGES, true>), grid, threads, 0, c->stream, a, rt, ct);
    else
        hipLaunchKernelGGL((fx_linear_tile_kernel<WM, WN, I, J, STAGES, false>), grid, threads, 0, c->stream, a, rt, ct);
}

// Which kernel.  us for k x n on the rows given, in a loop (5 us of them the call):
//                          16-row    64 x 64,  64 x 64,  128 x 128,  128 x 128,
//                                    4 stages  2 stages  8 waves, 4  4 waves, 2
//   768 x 4096, 48 rows    6.2       8.4       8.4       14.0        16.1
//   3072 x 768, 200        13.8      21.4      23.4      40.6        52.9
//   768 x 4096, 200        16.0      9.1       9.5       15.4        17.6
//   3072 x 768, 800        39.2      23.0      32.8      40.5        53.2
//   768 x 50257, 48        38.8      21.8      19.6      30.3        25.9
//   768 x 4096, 800        51.2      22.3      20.8      17.8        19.8
//   3072 x 768, 3,200      133       51.9      48.1      43.8        54.3
//   768 x 768, 6,000       70.6      28.7      26.2      32.1        27.0
//   3072 x 768, 6,000      238       81.5      84.8      86.9        76.5
//   768 x 3072, 6,000      255       86.7      75.8      77.6        64.8
//   768 x 4096, 16,384               310       261       231         201
// The 16-row kernel reads the packed weights once for 16 rows and splits k over
// its waves: it wins up to about 1,400 workgroups, and always for 16 rows.  A
// small tile a CU wants depth of prefetch, a large one eight waves on it, and past
// that two workgroups a CU hide each other's waits.  The estimates, in ns from the
// calls above, are a start and an end plus so much a step, by tiles on each CU.
int launch_product(Context* c, const FxLinear& a) {
    const size_t blocks = fx_blocks(a.n), steps = fx_steps(a.k), row_blocks = (a.rows + 15) / 16;
    const size_t cus = c->cu_count;
    const size_t small = ((blocks + 3) / 4) * ((row_blocks + 3) / 4), large = ((blocks + 7) / 8) * ((row_blocks + 7) / 8);
    const size_t turns = (large + cus - 1) / cus;
    const size_t deep = small <= cus ? 5000 + 325 * steps : SIZE_MAX;
    const size_t pairs = 6000 + std::max<size_t>(600, 350 * small / cus) * steps;
    const size_t waves8 = turns == 1 ? 7500 + 710 * steps : turns * (6500 + 780 * steps);
    const size_t two = turns == 1 ? 5700 + 960 * steps : turns * (4700 + 690 * steps) + turns % 2 * 350 * steps;
    const size_t least = std::min(std::min(deep, pairs), std::min(waves8, two));
    if (row_blocks == 1 || blocks * row_blocks <= 1400) {
        // 1 x 3,072 x 768: 6.3 us with 4 waves, 5.7 with 16; 1 x 768 x 50,257: 13.6 and 14.9
        const unsigned waves = static_cast<unsigned>(std::min<size_t>(steps, blocks * row_blocks < cus ? 16 : 4));
        hipLaunchKernelGGL(fx_linear_rows_kernel, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(row_blocks)),
                           dim3(64 * waves), 0, c->stream, a);
    } else if (deep == least) {
        launch_tile<2, 2, 1, 1, 4>(c, a);
    } else if (pairs == least) {
        launch_tile<2, 2, 1, 1, 2>(c, a);
    } else if (waves8 == least) {
        launch_tile<4, 2, 1, 2, 4>(c, a);
    } else {
        launch_tile<2, 2, 2, 2, 2>(c, a);
    }
    VMX_HIP(c, hipGetLastError());
    return 0;
}

// Space for aligned rows.
constexpr size_t ALIGNED_MAX = size_t{128} << 20;

// Rows from .. from + count of a.
FxLinear rows_of(FxLinear a, size_t from, size_t count) {
    a.x += from * a.x_stride;
    if (a.residual) a.residual += from * a.residual_stride;
    a.out = static_cast<unsigned char*>(a.out) + from * a.out_stride * (a.raw ? 8 : 2);
    a.rows = count;
    return a;
}

}  // namespace

int fx_pack_weights(Context* c, const int16_t* w, size_t k, size_t n, size_t stride, bool transposed, void* out) {
    const size_t blocks = fx_blocks(n);
    hipLaunchKernelGGL(fx_pack_weights_kernel, dim3(static_cast<unsigned>(blocks)), dim3(1024), 0, c->stream, w,
                       static_cast<int>(k), static_cast<int>(n), stride, transposed, static_cast<unsigned char*>(out),
                       blocks);
    VMX_HIP(c, hipGetLastError());
    return 0;
}

// Rows that are not aligned are aligned in a workspace, as many at a time as it may
// hold, where it may grow: copies through registers wait for memory in each step, and
// rows of other alignment take twice the accesses (us without and with, the aligning
// included: 1,337 x 961 x 5,203 68 and 43, 16,384 x 767 x 4,096 412 and 232, 1,023 x
// 767 x 3,072 34 and 22).  A launch to align rows costs about 3 us: 100 x 767 x 768
// (4,032 steps of 16 x 16) 9.3 us without and 10.7 with, 20 x 3,001 x 768 (4,512) 11.9
// and 9.9, 100 x 767 x 3,072 (16,128) 18.1 and 12.4.
int fx_linear(Context* c, const FxLinear& a) {
    const size_t pieces = (a.k + 7) / 8, row_bytes = pieces * 16;
    const size_t row_blocks = (a.rows + 15) / 16;
    const bool align = row_blocks > 1 && fx_blocks(a.n) * row_blocks * fx_steps(a.k) >= 4400 && !aligned_rows(a);
    // whole tiles, of 1,024 rows at least (k is below 2^16)
    const size_t most = ALIGNED_MAX / row_bytes / 128 * 128;
    if (!align || !try_ws(c, WS_FIXED, workspace_step(std::min(a.rows, most) * row_bytes, ALIGNED_MAX)))
        return launch_product(c, a);
    v4i* to = ws<v4i>(c, WS_FIXED);
    for (size_t row = 0; row < a.rows; row += most) {
        FxLinear part = rows_of(a, row, std::min(most, a.rows - row));
        hipLaunchKernelGGL(fx_align_rows_kernel, dim3(static_cast<unsigned>((part.rows * pieces + 255) / 256)), dim3(256), 0,
                           c->stream, part.x, part.x_stride, part.rows, a.k, static_cast<uint32_t>(pieces), to);
        part.x = reinterpret_cast<const int16_t*>(to);
        part.x_stride = pieces * 8;
        if (launch_product(c, part)) return -1;
    }
    return 0;
}

}  // namespace vmx
