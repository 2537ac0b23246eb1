// fixed.hpp -- fixed-point model operators over resident i16 tensors: shared
// device arithmetic, the packed layouts and the launchers.
//
// Every operator is exact integer arithmetic with a defined rounding, so its
// result does not depend on how sums are split or in which order they are
// joined: split axes and atomic additions give the same bits every time.
//
// 16-bit products on the matrix cores.  A 16-bit x is 256 h + l + 128 with
// h = x >> 8 and l = (x & 255) - 128, both signed bytes.  A w of at most 32,639
// is 256 h + l with signed bytes itself (l the low byte's own sign, h the rest);
// larger ones need the 128 as well.  So with X = x - 128 and W = w - o, o = 0 or
// 128, a product of 16-bit vectors is four products of 8-bit ones:
//   sum X W = 2^16 sum xh wh + 2^8 (sum xh wl + sum xl wh) + sum xl wl,
//   sum x w = sum X W + 128 sum_k W + o sum_k x.
// The two middle products share an accumulator: three i32 sums per result,
// which hold rows of 2^16 - 1 elements (2 * 2^14 a place in the middle one).
// Padding places hold x = 0 and w = 0, which the same identity covers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <cstddef>

#include "context.hpp"

namespace vmx {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));
typedef short v2s __attribute__((ext_vector_type(2)));

namespace fx {

// Rows of tensors may start at any element: global loads and stores of 16
// bytes need no more than the element's alignment on this target.
struct __attribute__((packed, aligned(2))) Row16 {
    v4i v;
};
struct __attribute__((packed, aligned(2))) Row8 {
    uint2 v;
};

__device__ inline v4i load8(const int16_t* p) { return reinterpret_cast<const Row16*>(p)->v; }

// Sixteen i16 (lo: the first eight) as their high and their offset low bytes.
__device__ inline void split16(v4i lo, v4i hi, v4i* h, v4i* l) {
    const uint32_t top = 0x07050301u, bottom = 0x06040200u, off = 0x80808080u;
    (*h)[0] = __builtin_amdgcn_perm(lo[1], lo[0], top);
    (*h)[1] = __builtin_amdgcn_perm(lo[3], lo[2], top);
    (*h)[2] = __builtin_amdgcn_perm(hi[1], hi[0], top);
    (*h)[3] = __builtin_amdgcn_perm(hi[3], hi[2], top);
    (*l)[0] = __builtin_amdgcn_perm(lo[1], lo[0], bottom) ^ off;
    (*l)[1] = __builtin_amdgcn_perm(lo[3], lo[2], bottom) ^ off;
    (*l)[2] = __builtin_amdgcn_perm(hi[1], hi[0], bottom) ^ off;
    (*l)[3] = __builtin_amdgcn_perm(hi[3], hi[2], bottom) ^ off;
}

// acc + the sum of the eight i16 of v (mod 2^32).
__device__ inline int sum8(v4i v, int acc) {
    const v2s one = {1, 1};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int pair = v[i];  // a bit cast of the vector's element itself reads element 0
        acc = __builtin_amdgcn_sdot2(__builtin_bit_cast(v2s, pair), one, acc, false);
    }
    return acc;
}

// Elements at .. at + 15 of a row of `len` starting at p, zero from len on.
__device__ inline void load16(const int16_t* p, int at, int len, v4i* lo, v4i* hi) {
    if (at + 16 <= len) {
        *lo = load8(p + at);
        *hi = load8(p + at + 8);
        return;
    }
    union {
        v4i v[2];
        int16_t e[16];
    } u;
    u.v[0] = v4i{0, 0, 0, 0};
    u.v[1] = v4i{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (at + i < len) u.e[i] = p[at + i];
    *lo = u.v[0];
    *hi = u.v[1];
}

// Sixteen bytes a lane from base + off (off a lane's own, base the wave's) to
// LDS at `to` (the wave's) + 16 lane, without registers between.  The compiler
// does not see the copy: lds_copies_done waits for a wave's own ones, and a
// barrier after it covers the workgroup's.  (Through the builtin it would wait
// for all of them before every read of LDS, the buffers in use among them.)
__device__ inline void copy_to_lds(const void* base, uint32_t off, void* to) {
    const uint32_t at = static_cast<uint32_t>(
        reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)to));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(at)), "v"(off), "s"(base)
                 : "memory", "m0");
}
// Waits until at most `Left` of the wave's copies are under way.
template <int Left>
__device__ inline void lds_copies_done() {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(Left) : "memory");
}

// Both shapes take 16 places of one row (column) per lane, in the same order on
// both sides; results: row 4 (lane >> 4) + r, column lane & 15 of 16 x 16, and
// row 8 (r >> 2) + 4 (lane >> 5) + (r & 3), column lane & 31 of 32 x 32.
__device__ inline v4i mfma(v4i a, v4i b, v4i c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
__device__ inline v16i mfma32(v4i a, v4i b, v16i c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
}

// A 16-bit w, less its offset, as its two signed bytes (high in bits 15..8 of the result).
__device__ inline int halves(int w) {
    const int l = static_cast<int8_t>(w);
    return ((w - l) & 0xff00) | (l & 0xff);
}
constexpr int HALVES_MAX = 32639;  // the largest w that needs no offset

__device__ inline int64_t join(int hh, int mid, int ll) {
    return (static_cast<int64_t>(hh) << 16) + (static_cast<int64_t>(mid) << 8) + ll;
}

__device__ inline int64_t rounded(int64_t a, uint32_t shift) {
    return shift ? (a + (int64_t{1} << (shift - 1))) >> shift : a;
}

__device__ inline int sat16(int64_t a) {
    return static_cast<int>(a < -32768 ? -32768 : a > 32767 ? 32767 : a);
}

// floor(a / b) for |a|, b < 2^52, b > 0, whole numbers held in doubles; inv = 1 / b.
// The estimate is off by at most one, and the remainder is exact in one fma.
__device__ inline double floor_div(double a, double b, double inv) {
    double q = __builtin_floor(a * inv);
    const double r = __builtin_fma(-q, b, a);
    return r < 0 ? q - 1 : r >= b ? q + 1 : q;
}

}  // namespace fx

// Workspace to ask for where `bytes` are needed: sizes double from 1 MiB up to `most`
// (a power of two) and are its multiples from there, so that needs that grow a little
// at a time (a tile of tokens, a row) are met by few allocations.
inline size_t workspace_step(size_t bytes, size_t most) {
    size_t step = size_t{1} << 20;
    while (step < bytes && step < most) step *= 2;
    return (bytes + step - 1) / step * step;
}

// ---- matrix product --------------------------------------------------------------
// Packed weights: for each block of 16 columns, each step of 64 rows of w, the
// high and the low plane in the order a wave's lanes read them (lane l: column
// l & 15, rows 16 (l >> 4) .. + 15), 1 KiB each; then 128 sum_k W of every
// column, i64; then o of every block, i32.
constexpr size_t FX_K_MAX = 65535;
inline size_t fx_blocks(size_t n) { return (n + 15) / 16; }
inline size_t fx_steps(size_t k) { return (k + 63) / 64; }
inline size_t fx_weight_bytes(size_t k, size_t n) { return fx_blocks(n) * (fx_steps(k) * 2048 + 128 + 4); }

struct FxLinear {
    const int16_t* x;
    size_t x_stride;
    const unsigned char* weights;
    const int16_t* bias;      // null: none
    const int16_t* table;     // null: none; 65,536 entries
    const int16_t* residual;  // null: none
    size_t residual_stride;
    void* out;  // i16, or the i64 sums (raw)
    size_t out_stride;
    size_t rows;
    int k, n;
    uint32_t bias_shift, shift;
    bool raw;
};

int fx_pack_weights(Context* c, const int16_t* w, size_t k, size_t n, size_t stride, bool transposed, void* out);
int fx_linear(Context* c, const FxLinear& a);

// ---- attention over a cache ---------------------------------------------------------
// One record per (slot, key head, 64 tokens), heads padded to 64 or 128 places,
// in pieces of 1 KiB in the order a wave reads them:
//   keys    32-token block x 32 places x plane (lane l: token l & 31, places
//           16 (l >> 5) .. + 15), split as weights are, with an offset for
//           tokens that hold a value over 32,639
//   values  32-token block x 32 places x plane (lane l: place l & 31, byte
//           4 q + r of token 8 q + 4 (l >> 5) + r: the order in which a wave holds
//           the scores of 32 tokens), split with the offset always
//   extras  256 sum_d k + the key's offset, of each token, i32
constexpr int FX_TILE = 64;
constexpr size_t FX_HEAD_MAX = 128;
constexpr size_t FX_CACHE_MAX = 65536;  // tokens a slot: the i32 sums of e v hold 87,000
constexpr size_t FX_TABLE_MAX = 8192;
constexpr int FX_SEQS = 64;             // sequences a launch
inline size_t fx_head_pad(size_t dim) { return dim <= 64 ? 64 : 128; }
inline size_t fx_tiles(size_t capacity) { return (capacity + FX_TILE - 1) / FX_TILE; }
inline size_t fx_record_bytes(size_t dim) { return fx_head_pad(dim) * 256 + 256; }

struct FxCache {
    unsigned char* data;
    size_t slots, kv_heads, dim, capacity;
};

// Rows row .. row + count of the packed tensors are the last `count` tokens of
// the `length` in `slot`.
struct FxSeq {
    uint32_t slot, row, count, length;
};

struct FxAttention {
    const int16_t* q;
    size_t q_stride;
    int16_t* out;
    size_t out_stride;
    const uint16_t* table;
    uint32_t entries, heads, shift;
    bool causal;
};

int fx_kv_append(Context* c, const FxCache& cache, const int16_t* k, size_t k_stride, const int16_t* v, size_t v_stride,
                 const FxSeq* seqs, size_t count);
int fx_attention(Context* c, const FxCache& cache, const FxAttention& a, const FxSeq* seqs, size_t count);

// ---- rows -----------------------------------------------------------------------------
struct FxNorm {
    const int16_t* x;
    size_t x_stride;
    const int16_t* residual;  // null: none
    size_t residual_stride;
    int16_t* sum;  // null: not kept
    size_t sum_stride;
    const int16_t* gain;
    const int16_t* bias;  // null: none
    int16_t* out;
    size_t out_stride;
    size_t rows;
    int cols;
    uint32_t shift;
    uint64_t eps;
    bool rms;
};

struct FxEmbed {
    const int32_t* tokens;
    const int16_t* table;
    size_t table_stride, vocab;
    const int32_t* positions;        // null: none
    const int16_t* position_table;
    size_t position_stride, position_rows;
    int16_t* out;
    size_t out_stride;
    size_t rows;
    int cols;
    int32_t scale;
    uint32_t shift;
};

int fx_norm(Context* c, const FxNorm& a);
int fx_embed(Context* c, const FxEmbed& a);

}  // namespace vmx
