// abi_fixed.cpp -- entry points of the fixed-point model operators
// (include/volta_cuda_abi.h, "Fixed-point model operators"): checks of
// arguments, regions and overlaps; the kernels are in fixed_*.hip.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <exception>
#include <string>
#include <vector>

#include "fixed.hpp"
#include "volta_cuda_abi.h"

using namespace vmx;

namespace {

template <class F>
int guarded(Context* c, const char* what, F&& f) noexcept {
    try {
        return f();
    } catch (...) {
        try {
            return fail_msg(c, (std::string(what) + " threw a C++ exception").c_str());
        } catch (...) {
            return fail_msg(c, "C++ exception");
        }
    }
}

// Sizes that a launch's 32-bit indices hold.
constexpr size_t MAX_ROWS = size_t{1} << 24;
constexpr size_t MAX_COLS = size_t{1} << 24;

struct Span {
    const unsigned char* at = nullptr;
    size_t bytes = 0;
};

// A rows x cols matrix of `elem`-byte elements, `stride` elements from row to row.
int matrix(Context* c, uint64_t id, size_t off, size_t stride, size_t rows, size_t cols, size_t elem, void** out,
           Span* span, bool read_only) {
    size_t before = 0, count = 0;
    if (stride < cols) return fail_msg(c, "row stride is shorter than a row");
    if (!mul_ok(rows - 1, stride, &before) || !add_ok(before, cols, &count))
        return fail_msg(c, "resident matrix geometry overflows size_t");
    if (region_elems(c, id, off, count, elem, out, read_only)) return -1;
    if (reinterpret_cast<uintptr_t>(*out) % elem) return fail_msg(c, "misaligned resident matrix");
    *span = Span{static_cast<const unsigned char*>(*out), count * elem};
    return 0;
}

bool overlap(const Span& a, const Span& b) { return a.at < b.at + b.bytes && b.at < a.at + a.bytes; }

// Timing record around a launch.
template <class F>
int counted(Context* c, F&& launch) {
    if (begin_op(c) || mark_op(c, 1)) return -1;
    if (launch()) return -1;
    if (mark_op(c, 2)) return -1;
    return finish_op(c, OP_GEMM, 0, 0);
}

bool cache_ok(size_t slots, size_t kv_heads, size_t dim, size_t capacity, size_t* bytes) {
    size_t heads = 0;
    return slots && kv_heads && dim && dim <= FX_HEAD_MAX && capacity && capacity <= FX_CACHE_MAX &&
           kv_heads <= 65535 && slots <= UINT32_MAX && mul_ok(slots, kv_heads, &heads) &&
           mul3_ok(heads, fx_tiles(capacity), fx_record_bytes(dim), bytes);
}

int resolve_cache(Context* c, const VoltaFixedCache* cache, FxCache* out, Span* span, bool read_only) {
    size_t bytes = 0;
    if (!cache || !cache_ok(cache->slots, cache->kv_heads, cache->dim, cache->capacity, &bytes))
        return fail_msg(c, "invalid fixed-point cache geometry");
    void* p = nullptr;
    if (region(c, cache->id, cache->off_bytes, bytes, &p, read_only)) return -1;
    if (reinterpret_cast<uintptr_t>(p) % 16) return fail_msg(c, "misaligned fixed-point cache");
    *out = FxCache{static_cast<unsigned char*>(p), cache->slots, cache->kv_heads, cache->dim, cache->capacity};
    *span = Span{static_cast<const unsigned char*>(p), bytes};
    return 0;
}

// Checked sequences without the empty ones; *rows is one past their last row.
// `append` asks for slots that occur once, `inside` for count <= length.
int resolve_sequences(Context* c, const FxCache& cache, const VoltaFixedSequence* seqs, size_t count, bool append,
                      bool inside, std::vector<FxSeq>* out, size_t* rows) {
    *rows = 0;
    if (count && !seqs) return fail_msg(c, "missing sequences");
    for (size_t i = 0; i < count; ++i) {
        const VoltaFixedSequence& s = seqs[i];
        if (s.slot >= cache.slots) return fail_msg(c, "sequence slot is outside the cache");
        if (s.length > cache.capacity) return fail_msg(c, "sequence is longer than the cache's capacity");
        if (inside && s.count > s.length) return fail_msg(c, "sequence has more new tokens than tokens");
        if (s.count > MAX_ROWS || s.row > MAX_ROWS) return fail_msg(c, "sequence rows are out of range");
        if (!s.count) continue;
        out->push_back(FxSeq{static_cast<uint32_t>(s.slot), static_cast<uint32_t>(s.row),
                             static_cast<uint32_t>(s.count), static_cast<uint32_t>(s.length)});
        *rows = std::max<size_t>(*rows, s.row + s.count);
    }
    std::vector<FxSeq> sorted(*out);
    if (append) {
        std::sort(sorted.begin(), sorted.end(), [](const FxSeq& a, const FxSeq& b) { return a.slot < b.slot; });
        for (size_t i = 1; i < sorted.size(); ++i)
            if (sorted[i].slot == sorted[i - 1].slot) return fail_msg(c, "a slot occurs twice in one append");
    } else {
        std::sort(sorted.begin(), sorted.end(), [](const FxSeq& a, const FxSeq& b) { return a.row < b.row; });
        for (size_t i = 1; i < sorted.size(); ++i)
            if (sorted[i].row < sorted[i - 1].row + sorted[i - 1].count)
                return fail_msg(c, "rows of two sequences overlap");
    }
    return 0;
}

}  // namespace

VMX_API size_t volta_mi355x_fixed_weights_bytes(size_t k, size_t n) {
    return k && k <= FX_K_MAX && n && n <= MAX_COLS ? fx_weight_bytes(k, n) : 0;
}

VMX_API int volta_mi355x_fixed_weights_device(void* raw, uint64_t w_id, size_t w_off, size_t k, size_t n, size_t stride,
                                              int transposed, uint64_t out_id, size_t out_off) {
    Context* c = static_cast<Context*>(raw);
    const size_t bytes = volta_mi355x_fixed_weights_bytes(k, n);
    if (!c || !bytes) return fail_msg(c, "invalid fixed-point weight geometry");
    return guarded(c, "fixed-point weights", [&] {
        void *w = nullptr, *out = nullptr;
        Span ws, os;
        if (matrix(c, w_id, w_off, stride, transposed ? n : k, transposed ? k : n, 2, &w, &ws, true) ||
            region(c, out_id, out_off, bytes, &out))
            return -1;
        if (reinterpret_cast<uintptr_t>(out) % 16) return fail_msg(c, "misaligned packed weights");
        os = Span{static_cast<const unsigned char*>(out), bytes};
        if (overlap(ws, os)) return fail_msg(c, "fixed-point weights and their packed form overlap");
        return counted(c, [&] {
            return fx_pack_weights(c, static_cast<const int16_t*>(w), k, n, stride, transposed != 0, out);
        });
    });
}

VMX_API int volta_mi355x_fixed_linear_device(void* raw, const VoltaFixedLinear* a) {
    Context* c = static_cast<Context*>(raw);
    if (!c || !a || !a->rows || a->rows > MAX_ROWS) return fail_msg(c, "invalid fixed-point linear geometry");
    const size_t bytes = volta_mi355x_fixed_weights_bytes(a->k, a->n);
    if (!bytes || a->bias_shift > 46 || (!a->raw && a->shift > 62))
        return fail_msg(c, "invalid fixed-point linear geometry");
    if (a->raw && (a->table_id || a->residual_id))
        return fail_msg(c, "raw fixed-point sums take neither a table nor a residual");
    return guarded(c, "fixed-point linear", [&] {
        void *x = nullptr, *w = nullptr, *bias = nullptr, *table = nullptr, *res = nullptr, *out = nullptr;
        Span xs, ws, bs, ts, rs, os;
        if (matrix(c, a->x_id, a->x_off, a->x_stride, a->rows, a->k, 2, &x, &xs, true) ||
            region(c, a->weights_id, a->weights_off_bytes, bytes, &w, true) ||
            (a->bias_id && matrix(c, a->bias_id, a->bias_off, a->n, 1, a->n, 2, &bias, &bs, true)) ||
            (a->table_id && matrix(c, a->table_id, a->table_off, 65536, 1, 65536, 2, &table, &ts, true)) ||
            (a->residual_id && matrix(c, a->residual_id, a->residual_off, a->residual_stride, a->rows, a->n, 2, &res,
                                      &rs, true)) ||
            matrix(c, a->out_id, a->out_off, a->out_stride, a->rows, a->n, a->raw ? 8 : 2, &out, &os, false))
            return -1;
        if (reinterpret_cast<uintptr_t>(w) % 16) return fail_msg(c, "misaligned packed weights");
        ws = Span{static_cast<const unsigned char*>(w), bytes};
        const bool in_place = res == out && a->residual_stride == a->out_stride;
        if (overlap(os, xs) || overlap(os, ws) || overlap(os, bs) || overlap(os, ts) || (!in_place && overlap(os, rs)))
            return fail_msg(c, "fixed-point linear output overlaps an input");
        FxLinear l{};
        l.x = static_cast<const int16_t*>(x);
        l.x_stride = a->x_stride;
        l.weights = static_cast<const unsigned char*>(w);
        l.bias = static_cast<const int16_t*>(bias);
        l.table = static_cast<const int16_t*>(table);
        l.residual = static_cast<const int16_t*>(res);
        l.residual_stride = a->residual_stride;
        l.out = out;
        l.out_stride = a->out_stride;
        l.rows = a->rows;
        l.k = static_cast<int>(a->k);
        l.n = static_cast<int>(a->n);
        l.bias_shift = a->bias_shift;
        l.shift = a->shift;
        l.raw = a->raw != 0;
        return counted(c, [&] { return fx_linear(c, l); });
    });
}

VMX_API size_t volta_mi355x_fixed_cache_bytes(size_t slots, size_t kv_heads, size_t dim, size_t capacity) {
    size_t bytes = 0;
    return cache_ok(slots, kv_heads, dim, capacity, &bytes) ? bytes : 0;
}

VMX_API int volta_mi355x_fixed_kv_append_device(void* raw, const VoltaFixedCache* cache, uint64_t k_id, size_t k_off,
                                                size_t k_stride, uint64_t v_id, size_t v_off, size_t v_stride,
                                                const VoltaFixedSequence* sequences, size_t count) {
    Context* c = static_cast<Context*>(raw);
    if (!c) return fail_msg(c, "missing context");
    return guarded(c, "fixed-point cache append", [&] {
        FxCache kv{};
        Span cs, ks, vs;
        std::vector<FxSeq> seqs;
        size_t rows = 0;
        if (resolve_cache(c, cache, &kv, &cs, false) ||
            resolve_sequences(c, kv, sequences, count, true, true, &seqs, &rows))
            return -1;
        if (!rows) return empty_op(c, OP_GEMM);
        const size_t cols = kv.kv_heads * kv.dim;
        void *k = nullptr, *v = nullptr;
        if (matrix(c, k_id, k_off, k_stride, rows, cols, 2, &k, &ks, true) ||
            matrix(c, v_id, v_off, v_stride, rows, cols, 2, &v, &vs, true))
            return -1;
        if (overlap(cs, ks) || overlap(cs, vs)) return fail_msg(c, "keys or values overlap the cache");
        return counted(c, [&] {
            return fx_kv_append(c, kv, static_cast<const int16_t*>(k), k_stride, static_cast<const int16_t*>(v), v_stride,
                                seqs.data(), seqs.size());
        });
    });
}

namespace {

// What a row sees of the keys: all up to its own, or a window with sinks, or a prefix before its sequence.
struct Seen {
    size_t window = 0, sinks = 0;
    uint64_t prefix_slot = 0, prefix = 0;
};

int attention(Context* c, const VoltaFixedCache* cache, const VoltaFixedAttention* a, const Seen& seen,
              const VoltaFixedSequence* sequences, size_t count) {
    if (!c || !a) return fail_msg(c, "invalid fixed-point attention geometry");
    if (a->shift < 8 || a->shift > 24 || !a->entries || a->entries > FX_TABLE_MAX)
        return fail_msg(c, "invalid fixed-point attention shift or table");
    return guarded(c, "fixed-point attention", [&] {
        FxCache kv{};
        Span cs, qs, ts, os;
        std::vector<FxSeq> seqs;
        size_t rows = 0;
        if (resolve_cache(c, cache, &kv, &cs, true)) return -1;
        if (!a->heads || a->heads % kv.kv_heads || a->heads > 65535)
            return fail_msg(c, "attention heads are not a multiple of the cache's");
        if (resolve_sequences(c, kv, sequences, count, false, a->causal != 0, &seqs, &rows)) return -1;
        if (seen.prefix && (seen.prefix_slot >= kv.slots || seen.prefix > kv.capacity))
            return fail_msg(c, "prefix is outside the cache");
        for (const FxSeq& s : seqs) {
            if (seen.prefix && s.slot == seen.prefix_slot) return fail_msg(c, "a sequence is in the prefix's slot");
            if (seen.prefix + s.length > FX_CACHE_MAX) return fail_msg(c, "prefix and sequence are longer than 65,536 tokens");
            // a launch's 32-bit rows: tokens x query heads of a key head, in blocks of 128
            if (s.count * (a->heads / kv.kv_heads) > INT32_MAX - 127)
                return fail_msg(c, "a sequence has more rows than 32 bits hold");
        }
        if (!rows) return empty_op(c, OP_GEMM);
        const size_t cols = a->heads * kv.dim;
        size_t places = 0;
        if (!mul_ok(rows, a->heads, &places) || places > INT32_MAX)
            return fail_msg(c, "fixed-point attention has too many rows");
        void *q = nullptr, *table = nullptr, *out = nullptr;
        if (matrix(c, a->q_id, a->q_off, a->q_stride, rows, cols, 2, &q, &qs, true) ||
            matrix(c, a->table_id, a->table_off, a->entries, 1, a->entries, 2, &table, &ts, true) ||
            matrix(c, a->out_id, a->out_off, a->out_stride, rows, cols, 2, &out, &os, false))
            return -1;
        if (overlap(os, qs) || overlap(os, ts) || overlap(os, cs))
            return fail_msg(c, "fixed-point attention output overlaps an input");
        const FxAttention t{static_cast<const int16_t*>(q),
                            a->q_stride,
                            static_cast<int16_t*>(out),
                            a->out_stride,
                            static_cast<const uint16_t*>(table),
                            static_cast<uint32_t>(a->entries),
                            static_cast<uint32_t>(a->heads),
                            a->shift,
                            a->causal != 0,
                            seen.window,
                            seen.sinks,
                            static_cast<uint32_t>(seen.prefix_slot),
                            static_cast<uint32_t>(seen.prefix)};
        return counted(c, [&] { return fx_attention(c, kv, t, seqs.data(), seqs.size()); });
    });
}

}  // namespace

VMX_API int volta_mi355x_fixed_attention_device(void* raw, const VoltaFixedCache* cache, const VoltaFixedAttention* a,
                                                const VoltaFixedSequence* sequences, size_t count) {
    return attention(static_cast<Context*>(raw), cache, a, Seen{}, sequences, count);
}

VMX_API int volta_mi355x_fixed_window_attention_device(void* raw, const VoltaFixedCache* cache,
                                                       const VoltaFixedAttention* a, size_t window, size_t sinks,
                                                       const VoltaFixedSequence* sequences, size_t count) {
    Context* c = static_cast<Context*>(raw);
    if (!c || !a || !window || !a->causal) return fail_msg(c, "a window of at least one key needs causal attention");
    return attention(c, cache, a, Seen{window, sinks, 0, 0}, sequences, count);
}

VMX_API int volta_mi355x_fixed_prefix_attention_device(void* raw, const VoltaFixedCache* cache,
                                                       const VoltaFixedAttention* a, uint64_t prefix_slot,
                                                       uint64_t prefix_length, const VoltaFixedSequence* sequences,
                                                       size_t count) {
    return attention(static_cast<Context*>(raw), cache, a, Seen{0, 0, prefix_slot, prefix_length}, sequences, count);
}

VMX_API int volta_mi355x_fixed_norm_device(void* raw, const VoltaFixedNorm* a) {
    Context* c = static_cast<Context*>(raw);
    if (!c || !a || !a->rows || a->rows > MAX_ROWS || !a->cols || a->cols > 65536 || a->shift > 15 || !a->eps ||
        a->eps > uint64_t{1} << 40)
        return fail_msg(c, "invalid fixed-point norm geometry");
    return guarded(c, "fixed-point norm", [&] {
        void *x = nullptr, *res = nullptr, *sum = nullptr, *gain = nullptr, *bias = nullptr, *out = nullptr;
        Span xs, rs, ss, gs, bs, os;
        if (matrix(c, a->x_id, a->x_off, a->x_stride, a->rows, a->cols, 2, &x, &xs, true) ||
            (a->residual_id && matrix(c, a->residual_id, a->residual_off, a->residual_stride, a->rows, a->cols, 2, &res,
                                      &rs, true)) ||
            matrix(c, a->gain_id, a->gain_off, a->cols, 1, a->cols, 2, &gain, &gs, true) ||
            (a->bias_id && matrix(c, a->bias_id, a->bias_off, a->cols, 1, a->cols, 2, &bias, &bs, true)) ||
            (a->sum_id && matrix(c, a->sum_id, a->sum_off, a->sum_stride, a->rows, a->cols, 2, &sum, &ss, false)) ||
            matrix(c, a->out_id, a->out_off, a->out_stride, a->rows, a->cols, 2, &out, &os, false))
            return -1;
        const bool over_x = sum == x && a->sum_stride == a->x_stride;
        const bool over_res = sum == res && a->sum_stride == a->residual_stride;
        if (overlap(os, xs) || overlap(os, rs) || overlap(os, gs) || overlap(os, bs) || overlap(os, ss) ||
            (!over_x && overlap(ss, xs)) || (!over_res && overlap(ss, rs)) || overlap(ss, gs) || overlap(ss, bs))
            return fail_msg(c, "fixed-point norm output overlaps another tensor");
        FxNorm n{};
        n.x = static_cast<const int16_t*>(x);
        n.x_stride = a->x_stride;
        n.residual = static_cast<const int16_t*>(res);
        n.residual_stride = a->residual_stride;
        n.sum = static_cast<int16_t*>(sum);
        n.sum_stride = a->sum_stride;
        n.gain = static_cast<const int16_t*>(gain);
        n.bias = static_cast<const int16_t*>(bias);
        n.out = static_cast<int16_t*>(out);
        n.out_stride = a->out_stride;
        n.rows = a->rows;
        n.cols = static_cast<int>(a->cols);
        n.shift = a->shift;
        n.eps = a->eps;
        n.rms = a->rms != 0;
        return counted(c, [&] { return fx_norm(c, n); });
    });
}

VMX_API int volta_mi355x_fixed_embed_device(void* raw, const VoltaFixedEmbed* a) {
    Context* c = static_cast<Context*>(raw);
    if (!c || !a || !a->rows || a->rows > MAX_ROWS || !a->cols || a->cols > MAX_COLS || !a->vocab || a->shift > 46 ||
        (!a->positions_id != !a->position_table_id) || (a->positions_id && !a->position_rows))
        return fail_msg(c, "invalid fixed-point embedding geometry");
    return guarded(c, "fixed-point embedding", [&] {
        void *tokens = nullptr, *table = nullptr, *places = nullptr, *where = nullptr, *out = nullptr;
        Span ns, ts, ps, ws, os;
        if (matrix(c, a->tokens_id, a->tokens_off, a->rows, 1, a->rows, 4, &tokens, &ns, true) ||
            matrix(c, a->table_id, a->table_off, a->table_stride, a->vocab, a->cols, 2, &table, &ts, true) ||
            (a->positions_id &&
             (matrix(c, a->positions_id, a->positions_off, a->rows, 1, a->rows, 4, &places, &ps, true) ||
              matrix(c, a->position_table_id, a->position_table_off, a->position_stride, a->position_rows, a->cols, 2,
                     &where, &ws, true))) ||
            matrix(c, a->out_id, a->out_off, a->out_stride, a->rows, a->cols, 2, &out, &os, false))
            return -1;
        if (overlap(os, ns) || overlap(os, ts) || overlap(os, ps) || overlap(os, ws))
            return fail_msg(c, "fixed-point embedding output overlaps an input");
        FxEmbed e{};
        e.tokens = static_cast<const int32_t*>(tokens);
        e.table = static_cast<const int16_t*>(table);
        e.table_stride = a->table_stride;
        e.vocab = a->vocab;
        e.positions = static_cast<const int32_t*>(places);
        e.position_table = static_cast<const int16_t*>(where);
        e.position_stride = a->position_stride;
        e.position_rows = a->position_rows;
        e.out = static_cast<int16_t*>(out);
        e.out_stride = a->out_stride;
        e.rows = a->rows;
        e.cols = static_cast<int>(a->cols);
        e.scale = a->scale;
        e.shift = a->shift;
        return counted(c, [&] { return fx_embed(c, e); });
    });
}

VMX_API int volta_mi355x_fixed_rotate_device(void* raw, const VoltaFixedRotate* a) {
    Context* c = static_cast<Context*>(raw);
    if (!c || !a || !a->rows || a->rows > MAX_ROWS || !a->dim || a->dim > FX_HEAD_MAX || a->heads > 65535 ||
        a->kv_heads > 65535 || !(a->heads + a->kv_heads) || a->rotated > a->dim || a->rotated % 2 || a->gain_shift > 15 ||
        a->angle_shift > 15 || !a->eps || a->eps > uint64_t{1} << 40)
        return fail_msg(c, "invalid fixed-point rotation geometry");
    if (!a->rotated != !a->angles_id || !a->rotated != !a->positions_id || (a->rotated && !a->angle_rows))
        return fail_msg(c, "rotated places, angles and positions come together");
    return guarded(c, "fixed-point rotation", [&] {
        void *x = nullptr, *qg = nullptr, *kg = nullptr, *angles = nullptr, *places = nullptr, *out = nullptr;
        Span xs, qs, ks, as, ps, os;
        const size_t cols = (a->heads + a->kv_heads) * a->dim;
        if (matrix(c, a->x_id, a->x_off, a->x_stride, a->rows, cols, 2, &x, &xs, true) ||
            (a->q_gain_id && matrix(c, a->q_gain_id, a->q_gain_off, a->dim, 1, a->dim, 2, &qg, &qs, true)) ||
            (a->k_gain_id && matrix(c, a->k_gain_id, a->k_gain_off, a->dim, 1, a->dim, 2, &kg, &ks, true)) ||
            (a->rotated && (matrix(c, a->angles_id, a->angles_off, a->rotated, a->angle_rows, a->rotated, 2, &angles,
                                   &as, true) ||
                            matrix(c, a->positions_id, a->positions_off, a->rows, 1, a->rows, 4, &places, &ps, true))) ||
            matrix(c, a->out_id, a->out_off, a->out_stride, a->rows, cols, 2, &out, &os, false))
            return -1;
        const bool in_place = out == x && a->out_stride == a->x_stride;
        if ((!in_place && overlap(os, xs)) || overlap(os, qs) || overlap(os, ks) || overlap(os, as) || overlap(os, ps))
            return fail_msg(c, "fixed-point rotation output overlaps an input");
        FxRotate r{};
        r.x = static_cast<const int16_t*>(x);
        r.x_stride = a->x_stride;
        r.q_gain = static_cast<const int16_t*>(qg);
        r.k_gain = static_cast<const int16_t*>(kg);
        r.angles = static_cast<const int16_t*>(angles);
        r.angle_rows = a->angle_rows;
        r.positions = static_cast<const int32_t*>(places);
        r.out = static_cast<int16_t*>(out);
        r.out_stride = a->out_stride;
        r.rows = a->rows;
        r.heads = static_cast<uint32_t>(a->heads);
        r.all_heads = static_cast<uint32_t>(a->heads + a->kv_heads);
        r.dim = static_cast<int>(a->dim);
        r.pairs = static_cast<int>(a->rotated / 2);
        r.eps = a->eps;
        r.gain_shift = a->gain_shift;
        r.angle_shift = a->angle_shift;
        r.adjacent = a->adjacent != 0;
        return counted(c, [&] { return fx_rotate(c, r); });
    });
}

VMX_API int volta_mi355x_fixed_choose_device(void* raw, const VoltaFixedChoose* a, const VoltaFixedChoice* choices,
                                             size_t count) {
    Context* c = static_cast<Context*>(raw);
    if (!c || !a || !count || count > MAX_ROWS || !choices || !a->vocab || a->vocab > MAX_COLS || a->bias_shift > 46)
        return fail_msg(c, "invalid fixed-point choice geometry");
    return guarded(c, "fixed-point choice", [&] {
        const size_t words = (a->vocab + 31) / 32;
        if (a->allowed_id && a->allowed_stride < words) return fail_msg(c, "row stride is shorter than a row");
        std::vector<FxChoice> rows;
        rows.reserve(count);
        // ends of the lists and of the masks that the rows read
        size_t history = 0, biases = 0, masks = 0;
        for (size_t i = 0; i < count; ++i) {
            const VoltaFixedChoice& s = choices[i];
            size_t end = 0;
            if (!s.repetition) return fail_msg(c, "repetition is zero");
            if (s.history_count > MAX_ROWS || s.bias_count > MAX_ROWS)
                return fail_msg(c, "a row's history or biases are too long");
            if ((s.history_count && !a->history_id) || (s.bias_count && (!a->bias_tokens_id || !a->bias_values_id)) ||
                (s.mask >= 0 && !a->allowed_id))
                return fail_msg(c, "a row reads a list that is missing");
            FxChoice r{};
            r.mask = -1;
            r.frequency = s.frequency;
            r.presence = s.presence;
            r.repetition = s.repetition;
            if (s.history_count) {
                if (!add_ok(s.history_first, s.history_count, &end)) return fail_msg(c, "a row's history is out of range");
                history = std::max(history, end);
                r.history = s.history_first;
                r.history_count = static_cast<uint32_t>(s.history_count);
            }
            if (s.bias_count) {
                if (!add_ok(s.bias_first, s.bias_count, &end)) return fail_msg(c, "a row's biases are out of range");
                biases = std::max(biases, end);
                r.bias = s.bias_first;
                r.bias_count = static_cast<uint32_t>(s.bias_count);
            }
            if (s.mask >= 0) {
                size_t at = 0;
                if (!mul_ok(static_cast<size_t>(s.mask), a->allowed_stride, &at) || at > INT64_MAX)
                    return fail_msg(c, "a row's mask is out of range");
                masks = std::max(masks, static_cast<size_t>(s.mask) + 1);
                r.mask = static_cast<int64_t>(at);
            }
            rows.push_back(r);
        }
        void *logits = nullptr, *past = nullptr, *tokens = nullptr, *values = nullptr, *allowed = nullptr,
             *adjusted = nullptr, *out = nullptr;
        Span ls, hs, bs, vs, ms, as, os;
        if (matrix(c, a->logits_id, a->logits_off, a->logits_stride, count, a->vocab, 8, &logits, &ls, true) ||
            (history && matrix(c, a->history_id, a->history_off, history, 1, history, 4, &past, &hs, true)) ||
            (biases && (matrix(c, a->bias_tokens_id, a->bias_tokens_off, biases, 1, biases, 4, &tokens, &bs, true) ||
                        matrix(c, a->bias_values_id, a->bias_values_off, biases, 1, biases, 4, &values, &vs, true))) ||
            (masks && matrix(c, a->allowed_id, a->allowed_off, a->allowed_stride, masks, words, 4, &allowed, &ms, true)) ||
            (a->adjusted_id && matrix(c, a->adjusted_id, a->adjusted_off, a->adjusted_stride, count, a->vocab, 8, &adjusted,
                                      &as, false)) ||
            matrix(c, a->out_id, a->out_off, count, 1, count, 4, &out, &os, false))
            return -1;
        const bool in_place = adjusted == logits && a->adjusted_stride == a->logits_stride;
        for (const Span& in : {hs, bs, vs, ms})
            if (overlap(os, in) || overlap(as, in)) return fail_msg(c, "fixed-point choice output overlaps an input");
        if (overlap(os, ls) || overlap(os, as) || (!in_place && overlap(as, ls)))
            return fail_msg(c, "fixed-point choice output overlaps an input");
        FxChoose f{};
        f.logits = static_cast<const int64_t*>(logits);
        f.logits_stride = a->logits_stride;
        f.history = static_cast<const int32_t*>(past);
        f.bias_tokens = static_cast<const int32_t*>(tokens);
        f.bias_values = static_cast<const int32_t*>(values);
        f.allowed = static_cast<const uint32_t*>(allowed);
        f.adjusted = static_cast<int64_t*>(adjusted);
        f.adjusted_stride = a->adjusted_stride;
        f.tokens = static_cast<int32_t*>(out);
        f.vocab = static_cast<uint32_t>(a->vocab);
        f.bias_shift = a->bias_shift;
        return counted(c, [&] { return fx_choose(c, f, rows.data(), rows.size()); });
    });
}
