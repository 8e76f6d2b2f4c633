// sc_ops_capi.cpp - the extern "C" layer of include/sc_ops.h: every request is checked whole on the host before the first
// launch, so a refusal (SC_EINVAL / SC_ERANGE) has enqueued nothing.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <exception>
#include <string>

#include "sc_ops.h"
#include "sc_ops.hpp"

namespace {

int bad(const char* op, const char* why) { return sc::record_error(SC_EINVAL, std::string("sc_ops: ") + op + ": " + why); }
int beyond(const char* op, const char* why) { return sc::record_error(SC_ERANGE, std::string("sc_ops: ") + op + ": " + why); }

template <class F>
int guarded(F&& f) {
    try {
        return f();
    } catch (const std::exception& e) {
        return sc::record_error(SC_EINVAL, std::string("sc_ops: ") + e.what());
    } catch (...) {
        return sc::record_error(SC_EINVAL, "sc_ops: unknown failure");
    }
}

int launched(hipError_t e, const char* op) {
    if (e == hipSuccess) return sc::record_ok();
    return sc::record_error(SC_EHIP, std::string("sc_ops: ") + op + ": " + hipGetErrorString(e));
}

bool off(const void* p, uintptr_t align) { return (reinterpret_cast<uintptr_t>(p) & (align - 1)) != 0; }

// The row stride of an activation tensor: whole 16 bytes from row to row, at least a row, at most 2^22 values (the rows
// of a chunk of 64 lie within 2^31 bytes).
bool row_stride(int64_t ld, int64_t row, int32_t dtype) {
    return ld >= row && ld <= (int64_t(1) << 22) && ld % (dtype == SC_DTYPE_F16 ? 8 : 4) == 0;
}
constexpr int64_t most_floats = int64_t(1) << 40;   // of a stride
int64_t value_bytes(int32_t dtype) { return dtype == SC_DTYPE_F16 ? 2 : 4; }

// Whether two tensors of `rows` rows have a byte in common, rows [p + t * ld, + row).  Rows side by side in one buffer, such
// as the parts of a fused projection, have one stride and none in common.
bool share_bytes(const void* a, int64_t a_ld, int64_t a_row, const void* b, int64_t b_ld, int64_t b_row, int64_t rows) {
    if (rows == 0) return false;
    const uint64_t p = reinterpret_cast<uintptr_t>(a), q = reinterpret_cast<uintptr_t>(b);
    if (p <= q ? q - p >= uint64_t((rows - 1) * a_ld + a_row) : p - q >= uint64_t((rows - 1) * b_ld + b_row)) return false;
    if (a_ld != b_ld) return true;
    const int64_t into = p <= q ? int64_t((q - p) % a_ld) : (a_ld - int64_t((p - q) % a_ld)) % a_ld;   // b's rows into a's
    return into < a_row || into + b_row > a_ld;
}

// Checks a cache and lays it out for the kernels; an SC_ status.
int cache_args(const char* op, const sc_kv_cache* c, int64_t n_seqs, sc::CacheArgs& o) {
    if (!c) return bad(op, "missing cache");
    if (c->format != SC_KV_F16 && c->format != SC_KV_INT8) return bad(op, "the cache's format must be f16 or int8");
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return bad(op, "head_dim must be 64, 128 or 256");
    if (c->n_head_kv < 1 || c->n_head_kv > 256) return bad(op, "n_head_kv must be 1 .. 256");
    if (c->page_size < 1 || c->page_size > 65536) return bad(op, "page_size must be 1 .. 65536");
    if (c->n_pages < 1 || c->n_pages > INT32_MAX) return bad(op, "n_pages must be 1 .. 2^31 - 1");
    if (c->table_ld < 1 || c->table_ld > INT32_MAX / c->page_size) return bad(op, "table_ld * page_size must be 1 .. 2^31 - 1");
    if (c->n_pages > INT32_MAX / (c->n_head_kv * c->page_size)) return beyond(op, "a pool of 2^31 rows or more");
    if (!c->table && n_seqs > INT32_MAX / c->table_ld) return beyond(op, "an identity table past 2^31 pages");
    if (!c->k || !c->v || off(c->k, 16) || off(c->v, 16)) return bad(op, "the cache's pools must be given, 16-byte aligned");
    if (c->format == SC_KV_INT8 && (!c->k_scale || !c->v_scale || off(c->k_scale, 8) || off(c->v_scale, 8)))
        return bad(op, "an int8 cache's scale pools must be given, 8-byte aligned");
    if (off(c->table, 4)) return bad(op, "the page table must be 4-byte aligned");
    o.k = static_cast<uint8_t*>(c->k);
    o.v = static_cast<uint8_t*>(c->v);
    o.k_scale = c->k_scale;
    o.v_scale = c->v_scale;
    o.table = c->table;
    o.table_ld = c->table_ld;
    o.cells = uint32_t(c->table_ld * c->page_size);
    o.n_pages = uint32_t(c->n_pages);
    o.H = uint32_t(c->n_head_kv);
    o.ps = sc::make_fastdiv(uint32_t(c->page_size));
    return SC_OK;
}

int attn_args(const sc_kv_cache* cache, const sc_attn_decode* d, sc::AttnArgs& a, uint64_t& ws_bytes) {
    const char* op = "attn_decode";
    if (!d) return bad(op, "missing request");
    if (d->n_seqs < 1 || d->n_seqs > SC_ATTN_MAX_SEQS) return bad(op, "n_seqs must be 1 .. SC_ATTN_MAX_SEQS");
    if (const int e = cache_args(op, cache, d->n_seqs, a.c)) return e;
    if (d->max_len < 0 || d->max_len > int64_t(a.c.cells)) return bad(op, "max_len must be 0 .. table_ld * page_size");
    if (d->window < 0) return bad(op, "window must not be negative");
    if (d->dtype != SC_DTYPE_F16 && d->dtype != SC_DTYPE_F32) return bad(op, "dtype must be f16 or f32");
    if (d->n_head < 1 || d->n_head > 4096 || d->n_head % cache->n_head_kv)
        return bad(op, "n_head must be a multiple of n_head_kv, at most 4096");
    if (!d->lens || off(d->lens, 8)) return bad(op, "lens must be given, 8-byte aligned");
    if (!d->q || !d->out || off(d->q, 16) || off(d->out, 16)) return bad(op, "q and out must be given, 16-byte aligned");
    const int64_t row = d->n_head * cache->head_dim;
    if (!row_stride(d->q_ld, row, d->dtype) || !row_stride(d->out_ld, row, d->dtype))
        return bad(op, "q_ld and out_ld must be whole 16 bytes and hold n_head * head_dim values");
    if (off(d->lse, 4)) return bad(op, "lse must be 4-byte aligned");
    a.lens = d->lens;
    a.q = static_cast<const uint8_t*>(d->q);
    a.out = static_cast<uint8_t*>(d->out);
    a.lse = d->lse;
    a.q_ld = d->q_ld * value_bytes(d->dtype);
    a.out_ld = d->out_ld * value_bytes(d->dtype);
    a.n_seqs = uint32_t(d->n_seqs);
    a.n_head = uint32_t(d->n_head);
    a.max_len = uint32_t(d->max_len);
    a.window = d->window >= d->max_len ? 0 : uint32_t(d->window);
    a.scale = d->scale;
    a.ws = nullptr;
    ws_bytes = sc::plan_attn(a, int(cache->head_dim));
    return SC_OK;
}

int mass_args(const sc_kv_cache* cache, const sc_attn_mass* d, sc::MassArgs& a) {
    const char* op = "attn_mass";
    if (!d) return bad(op, "missing request");
    if (d->n_seqs < 1 || d->n_seqs > SC_ATTN_MAX_SEQS) return bad(op, "n_seqs must be 1 .. SC_ATTN_MAX_SEQS");
    if (const int e = cache_args(op, cache, d->n_seqs, a.c)) return e;
    if (d->max_len < 0 || d->max_len > int64_t(a.c.cells)) return bad(op, "max_len must be 0 .. table_ld * page_size");
    if (d->window < 0) return bad(op, "window must not be negative");
    if (d->dtype != SC_DTYPE_F16 && d->dtype != SC_DTYPE_F32) return bad(op, "dtype must be f16 or f32");
    if (d->n_head < 1 || d->n_head > 4096 || d->n_head % cache->n_head_kv)
        return bad(op, "n_head must be a multiple of n_head_kv, at most 4096");
    const int64_t G = d->n_head / cache->n_head_kv;
    if (d->rows < 1 || d->rows > 1024 / G) return bad(op, "rows must be at least 1, rows * n_head / n_head_kv at most 1024");
    if (!d->lens || off(d->lens, 8)) return bad(op, "lens must be given, 8-byte aligned");
    if (!d->q || off(d->q, 16)) return bad(op, "q must be given, 16-byte aligned");
    if (!row_stride(d->q_ld, d->n_head * cache->head_dim, d->dtype))
        return bad(op, "q_ld must be whole 16 bytes and hold n_head * head_dim values");
    if (off(d->lse, 4)) return bad(op, "lse must be 4-byte aligned");
    if (!(d->decay - d->decay == 0)) return bad(op, "decay must be a finite number");
    if (!d->mass || off(d->mass, 4)) return bad(op, "mass must be given, 4-byte aligned");
    if (d->mass_ld < d->max_len || d->mass_ld < 1 || d->mass_ld > INT32_MAX) return bad(op, "mass_ld must be at least max_len, 1 .. 2^31 - 1");
    a.lens = d->lens;
    a.q = static_cast<const uint8_t*>(d->q);
    a.lse = d->lse;
    a.mass = d->mass;
    a.q_ld = d->q_ld * value_bytes(d->dtype);
    a.mass_ld = uint64_t(d->mass_ld);
    a.n_seqs = uint32_t(d->n_seqs);
    a.n_head = uint32_t(d->n_head);
    a.rows = uint32_t(d->rows);
    a.cols = uint32_t(d->rows * G);
    a.max_len = uint32_t(d->max_len);
    a.window = d->window >= d->max_len ? 0 : uint32_t(d->window);
    a.G = sc::make_fastdiv(uint32_t(G));
    a.scale = d->scale;
    a.decay = d->decay;
    return SC_OK;
}

// Whether two ranges of as many bytes meet without being the same one.
bool half_over(const void* a, const void* b, uint64_t bytes) {
    const uint64_t p = reinterpret_cast<uintptr_t>(a), q = reinterpret_cast<uintptr_t>(b);
    return p != q && (p < q ? q - p : p - q) < bytes;
}

int evict_args(const sc_kv_cache* cache, const sc_kv_evict* d, sc::EvictArgs& a) {
    const char* op = "kv_evict";
    if (!d) return bad(op, "missing request");
    if (d->n_seqs < 1 || d->n_seqs > SC_ATTN_MAX_SEQS) return bad(op, "n_seqs must be 1 .. SC_ATTN_MAX_SEQS");
    if (const int e = cache_args(op, cache, d->n_seqs, a.c)) return e;
    if (d->max_len < 0 || d->max_len > int64_t(a.c.cells)) return bad(op, "max_len must be 0 .. table_ld * page_size");
    if (d->keep < 1 || d->keep > INT32_MAX) return bad(op, "keep must be 1 .. 2^31 - 1");
    if (d->sinks < 0 || d->recent < 0 || d->sinks > d->keep || d->recent > d->keep - d->sinks)
        return bad(op, "sinks and recent must not be negative, nor more than keep together");
    if (!d->lens || off(d->lens, 8) || !d->lens_out || off(d->lens_out, 8)) return bad(op, "lens and lens_out must be given, 8-byte aligned");
    if (off(d->known, 8) || off(d->total, 8)) return bad(op, "known and total must be 8-byte aligned");
    if (!d->mass || off(d->mass, 4) || !d->mass_out || off(d->mass_out, 4)) return bad(op, "mass and mass_out must be given, 4-byte aligned");
    if (off(d->born, 4) || off(d->born_out, 4)) return bad(op, "born and born_out must be 4-byte aligned");
    if (!d->born != !d->known) return bad(op, "born and known are given together");
    if (d->ld < d->max_len || d->ld < 1 || d->ld > INT32_MAX) return bad(op, "ld must be at least max_len, 1 .. 2^31 - 1");
    const uint64_t bytes = uint64_t(d->n_seqs) * uint64_t(cache->n_head_kv) * uint64_t(d->ld) * 4;
    if (half_over(d->mass, d->mass_out, bytes) || (d->born && d->born_out && half_over(d->born, d->born_out, bytes)))
        return bad(op, "mass_out and born_out must be mass and born or share no byte with them");
    a.lens = d->lens;
    a.known = d->known;
    a.total = d->total;
    a.lens_out = d->lens_out;
    a.mass = d->mass;
    a.mass_out = d->mass_out;
    a.born = d->born;
    a.born_out = d->born_out;
    a.ld = uint64_t(d->ld);
    a.n_seqs = uint32_t(d->n_seqs);
    a.max_len = uint32_t(d->max_len);
    a.keep = uint32_t(d->keep);
    a.sinks = uint32_t(d->sinks);
    a.recent = uint32_t(d->recent);
    return SC_OK;
}

int gdn_args(const char* op, const sc_gdn* d, bool step, sc::GdnArgs& a) {
    if (!d) return bad(op, "missing request");
    if (d->state_size != 32 && d->state_size != 64 && d->state_size != 128) return bad(op, "state_size must be 32, 64 or 128");
    if (d->k_heads < 1 || d->v_heads < 1 || d->v_heads > 1024 || d->v_heads % d->k_heads)
        return bad(op, "v_heads must be a multiple of k_heads, at most 1024");
    if (d->n_seqs < 1 || d->n_seqs > 4096) return bad(op, "n_seqs must be 1 .. 4096");
    if (d->tokens < 0 || d->tokens > (int64_t(1) << 23)) return bad(op, "tokens must be 0 .. 2^23");
    if (step ? d->cu || d->tokens != d->n_seqs : !d->cu || off(d->cu, 8))
        return bad(op, step ? "a step has one row a sequence and no cu" : "cu must be given, 8-byte aligned");
    if (d->dtype != SC_DTYPE_F16 && d->dtype != SC_DTYPE_F32) return bad(op, "dtype must be f16 or f32");
    if (!d->q || !d->k || !d->v || !d->out || off(d->q, 16) || off(d->k, 16) || off(d->v, 16) || off(d->out, 16))
        return bad(op, "q, k, v and out must be given, 16-byte aligned");
    const int64_t S = d->state_size;
    if (!row_stride(d->q_ld, d->k_heads * S, d->dtype) || !row_stride(d->k_ld, d->k_heads * S, d->dtype) ||
        !row_stride(d->v_ld, d->v_heads * S, d->dtype) || !row_stride(d->out_ld, d->v_heads * S, d->dtype))
        return bad(op, "row strides must be whole 16 bytes and hold a row");
    if (!d->g || !d->beta || off(d->g, 4) || off(d->beta, 4) || d->gate_ld < d->v_heads || d->gate_ld > (int64_t(1) << 22))
        return bad(op, "g and beta must be given, 4-byte aligned, gate_ld at least v_heads");
    if (!d->state || off(d->state, 8)) return bad(op, "state must be given, 8-byte aligned");
    if (d->state_offset < 0 || d->state_offset % 4 || d->state_head_ld < S || d->state_head_ld % 4 || d->state_key_ld < S ||
        d->state_key_ld % 4)
        return bad(op, "state strides must be multiples of 4 floats and hold a row");
    if (d->state_offset > most_floats || d->state_head_ld > most_floats || d->state_key_ld > most_floats) return bad(op, "state strides must be at most 2^40 floats");
    // the heads' rows inside a key's, or the keys' inside a head's block: anything else puts two values in one place
    if (d->state_key_ld < (d->v_heads - 1) * d->state_head_ld + S && d->state_head_ld < (S - 1) * d->state_key_ld + S)
        return bad(op, "state strides overlap");
    if (!(d->eps >= 0)) return bad(op, "eps must not be negative");
    const int64_t b = value_bytes(d->dtype);
    a.q = static_cast<const uint8_t*>(d->q);
    a.k = static_cast<const uint8_t*>(d->k);
    a.v = static_cast<const uint8_t*>(d->v);
    a.out = static_cast<uint8_t*>(d->out);
    a.q_ld = d->q_ld * b;
    a.k_ld = d->k_ld * b;
    a.v_ld = d->v_ld * b;
    a.out_ld = d->out_ld * b;
    a.g = d->g;
    a.beta = d->beta;
    a.gate_ld = d->gate_ld;
    a.state = d->state;
    a.state_offset = d->state_offset;
    a.head_ld = d->state_head_ld;
    a.key_ld = d->state_key_ld;
    a.cu = d->cu;
    a.n_seqs = uint32_t(d->n_seqs);
    a.tokens = uint32_t(d->tokens);
    a.v_heads = uint32_t(d->v_heads);
    a.l2norm = d->l2norm != 0;
    a.share = sc::make_fastdiv(uint32_t(d->v_heads / d->k_heads));
    a.scale = d->scale;
    a.eps = d->eps;
    return SC_OK;
}

// Workgroups of other columns read queries and keys of rows that one has written the outputs of; a row's values are read by
// the one that writes its outputs, before it does, so those may lie in one place.
bool outputs_apart(const sc_gdn* d) {
    const int64_t b = value_bytes(d->dtype), row = d->v_heads * d->state_size * b, key_row = d->k_heads * d->state_size * b;
    auto meets = [&](const void* x, int64_t ld, int64_t x_row) {
        return share_bytes(d->out, d->out_ld * b, row, x, ld * b, x_row, d->tokens);
    };
    return !meets(d->q, d->q_ld, key_row) && !meets(d->k, d->k_ld, key_row) &&
           ((d->out == d->v && d->out_ld == d->v_ld) || !meets(d->v, d->v_ld, row));
}
constexpr const char* kOutputsMeet = "out must not overlap q or k, nor v unless it is v";

// Checks an append, by one position a token or by several axes', and enqueues it.
int rope_append(const char* op, const sc_kv_cache* cache, const sc_rope_append* d, const sc_rope_axes* x, bool axes, void* stream) {
    if (!d || (axes && !x)) return bad(op, "missing request");
    if (d->n_seqs < 1 || d->n_seqs > 4096) return bad(op, "n_seqs must be 1 .. 4096");
    sc::RopeArgs a{};
    if (const int e = cache_args(op, cache, d->n_seqs, a.c)) return e;
    if (d->tokens < 0 || d->tokens > (int64_t(1) << 23)) return bad(op, "tokens must be 0 .. 2^23");
    if (!d->cu && d->tokens != d->n_seqs) return bad(op, "without cu there is one row a sequence");
    if (off(d->cu, 8) || !d->pos0 || off(d->pos0, 8)) return bad(op, "cu and pos0 must be 8-byte aligned, pos0 given");
    if (d->dtype != SC_DTYPE_F16 && d->dtype != SC_DTYPE_F32) return bad(op, "dtype must be f16 or f32");
    if (!d->k || !d->v || off(d->k, 16) || off(d->v, 16)) return bad(op, "k and v must be given, 16-byte aligned");
    const int64_t row = cache->n_head_kv * cache->head_dim;
    if (!row_stride(d->k_ld, row, d->dtype) || !row_stride(d->v_ld, row, d->dtype))
        return bad(op, "k_ld and v_ld must be whole 16 bytes and hold n_head_kv * head_dim values");
    if (!d->q ? d->n_head != 0 : d->n_head < 1 || d->n_head > 4096) return bad(op, "n_head must be 1 .. 4096 with q, 0 without");
    if (d->q) {
        if (!d->q_out || off(d->q, 16) || off(d->q_out, 16)) return bad(op, "q and q_out must be given, 16-byte aligned");
        if (!row_stride(d->q_ld, d->n_head * cache->head_dim, d->dtype) ||
            !row_stride(d->q_out_ld, d->n_head * cache->head_dim, d->dtype))
            return bad(op, "q_ld and q_out_ld must be whole 16 bytes and hold n_head * head_dim values");
        if (d->q == d->q_out && d->q_ld != d->q_out_ld) return bad(op, "queries rotated in place need one stride");
    }
    if (d->pairing != SC_ROPE_HALVES && d->pairing != SC_ROPE_NEIGHBOURS) return bad(op, "unknown pairing");
    if (d->rot_dim < 0 || d->rot_dim > cache->head_dim || d->rot_dim % 8) return bad(op, "rot_dim must be a multiple of 8, 0 .. head_dim");
    if (d->rot_dim && (!d->inv_freq || off(d->inv_freq, 4))) return bad(op, "inv_freq must be given, 4-byte aligned");
    if (axes) {
        if (x->n_axes < 1 || x->n_axes > 4) return bad(op, "n_axes must be 1 .. 4");
        if (!x->pos || off(x->pos, 8) || x->pos_ld < d->tokens || x->pos_ld > most_floats)
            return bad(op, "pos must be given, 8-byte aligned, pos_ld at least tokens");
        if (d->rot_dim && !x->host_axis) return bad(op, "host_axis must be given");
        for (int64_t i = 0; i < d->rot_dim / 2; ++i) {
            if (x->host_axis[i] >= x->n_axes) return bad(op, "an entry of host_axis is not below n_axes");
            a.axis[i / 16] |= uint32_t(x->host_axis[i]) << (i % 16 * 2);
        }
        a.axes = uint32_t(x->n_axes);
        a.pos = x->pos;
        a.pos_ld = x->pos_ld;
    }
    if (d->tokens == 0) return sc::record_ok();
    const int64_t b = value_bytes(d->dtype);
    a.k = static_cast<const uint8_t*>(d->k);
    a.v = static_cast<const uint8_t*>(d->v);
    a.q = static_cast<const uint8_t*>(d->q);
    a.q_out = static_cast<uint8_t*>(d->q_out);
    a.k_ld = d->k_ld * b;
    a.v_ld = d->v_ld * b;
    a.q_ld = d->q_ld * b;
    a.q_out_ld = d->q_out_ld * b;
    a.cu = d->cu;
    a.pos0 = d->pos0;
    a.inv_freq = d->inv_freq;
    a.tokens = uint32_t(d->tokens);
    a.n_seqs = uint32_t(d->n_seqs);
    a.n_head = uint32_t(d->n_head);
    a.rot = uint32_t(d->rot_dim);
    a.neighbours = d->pairing == SC_ROPE_NEIGHBOURS;
    return launched(sc::launch_rope(a, int(cache->head_dim), cache->format, d->dtype == SC_DTYPE_F16,
                                    static_cast<hipStream_t>(stream)), op);
}

}  // namespace

int sc_rope_append_async(const sc_kv_cache* cache, const sc_rope_append* d, void* stream) {
    return guarded([&] { return rope_append("rope_append", cache, d, nullptr, false, stream); });
}

int sc_rope_axes_append_async(const sc_kv_cache* cache, const sc_rope_append* d, const sc_rope_axes* axes, void* stream) {
    return guarded([&] { return rope_append("rope_axes_append", cache, d, axes, true, stream); });
}

uint64_t sc_attn_decode_workspace_bytes(const sc_kv_cache* cache, const sc_attn_decode* d) {
    sc::AttnArgs a{};
    uint64_t need = 0;
    return guarded([&] { return attn_args(cache, d, a, need); }) == SC_OK ? need : 0;
}

int sc_attn_decode_async(const sc_kv_cache* cache, const sc_attn_decode* d, void* workspace, uint64_t workspace_bytes,
                         void* stream) {
    return guarded([&] {
        const char* op = "attn_decode";
        sc::AttnArgs a{};
        uint64_t need = 0;
        if (const int e = attn_args(cache, d, a, need)) return e;
        if (!workspace || off(workspace, 16) || workspace_bytes < need)
            return bad(op, "workspace missing, not 16-byte aligned or below sc_attn_decode_workspace_bytes");
        sc::place_attn(a, workspace, need);
        return launched(sc::launch_attn(a, int(cache->head_dim), cache->format, d->dtype == SC_DTYPE_F16,
                                        static_cast<hipStream_t>(stream)), op);
    });
}

uint64_t sc_attn_mass_workspace_bytes(const sc_kv_cache* cache, const sc_attn_mass* d) {
    sc::MassArgs a{};
    return guarded([&] { return mass_args(cache, d, a); }) == SC_OK
               ? sc::plan_mass(a, int(cache->head_dim), d->dtype == SC_DTYPE_F16, nullptr) : 0;
}

int sc_attn_mass_async(const sc_kv_cache* cache, const sc_attn_mass* d, void* workspace, uint64_t workspace_bytes, void* stream) {
    return guarded([&] {
        const char* op = "attn_mass";
        sc::MassArgs a{};
        if (const int e = mass_args(cache, d, a)) return e;
        const bool f16 = d->dtype == SC_DTYPE_F16;
        if (!workspace || off(workspace, 16) || workspace_bytes < sc::plan_mass(a, int(cache->head_dim), f16, workspace))
            return bad(op, "workspace missing, not 16-byte aligned or below sc_attn_mass_workspace_bytes");
        if (d->max_len == 0) return sc::record_ok();
        return launched(sc::launch_mass(a, int(cache->head_dim), cache->format, f16, static_cast<hipStream_t>(stream)), op);
    });
}

uint64_t sc_kv_evict_workspace_bytes(const sc_kv_cache* cache, const sc_kv_evict* d) {
    sc::EvictArgs a{};
    return guarded([&] { return evict_args(cache, d, a); }) == SC_OK ? sc::plan_evict(a, nullptr) : 0;
}

int sc_kv_evict_async(const sc_kv_cache* cache, const sc_kv_evict* d, void* workspace, uint64_t workspace_bytes, void* stream) {
    return guarded([&] {
        const char* op = "kv_evict";
        sc::EvictArgs a{};
        if (const int e = evict_args(cache, d, a)) return e;
        if (!workspace || off(workspace, 16) || workspace_bytes < sc::plan_evict(a, workspace))
            return bad(op, "workspace missing, not 16-byte aligned or below sc_kv_evict_workspace_bytes");
        return launched(sc::launch_evict(a, int(cache->head_dim), cache->format, static_cast<hipStream_t>(stream)), op);
    });
}

int sc_conv_async(const sc_conv* d, void* stream) {
    return guarded([&] {
        const char* op = "conv";
        if (!d) return bad(op, "missing request");
        if (d->channels < 8 || d->channels > (int64_t(1) << 20) || d->channels % 8) return bad(op, "channels must be a multiple of 8, 8 .. 2^20");
        if (d->taps < 2 || d->taps > 5) return bad(op, "taps must be 2 .. 5");
        if (d->n_seqs < 1 || d->n_seqs > 4096) return bad(op, "n_seqs must be 1 .. 4096");
        if (d->tokens < 0 || d->tokens > (int64_t(1) << 23)) return bad(op, "tokens must be 0 .. 2^23");
        if (!d->cu && d->tokens != d->n_seqs) return bad(op, "without cu there is one row a sequence");
        if (off(d->cu, 8)) return bad(op, "cu must be 8-byte aligned");
        if (d->dtype != SC_DTYPE_F16 && d->dtype != SC_DTYPE_F32) return bad(op, "dtype must be f16 or f32");
        if (!d->x || !d->out || off(d->x, 16) || off(d->out, 16)) return bad(op, "x and out must be given, 16-byte aligned");
        if (!row_stride(d->x_ld, d->channels, d->dtype) || !row_stride(d->out_ld, d->channels, d->dtype))
            return bad(op, "x_ld and out_ld must be whole 16 bytes and hold a row");
        if (!d->weight || off(d->weight, 16) || off(d->bias, 16)) return bad(op, "weight must be given, weight and bias 16-byte aligned");
        if (d->activation != SC_CONV_NONE && d->activation != SC_CONV_SILU) return bad(op, "unknown activation");
        if (!d->state || off(d->state, 8)) return bad(op, "state must be given, 8-byte aligned");
        if (d->state_offset < 0 || d->state_offset % 4 || d->state_offset > most_floats) return bad(op, "state_offset must be a multiple of 4, 0 .. 2^40");
        if (d->state_layout != SC_CONV_SLOT && d->state_layout != SC_CONV_ROWS) return bad(op, "unknown state_layout");
        if (d->state_layout == SC_CONV_ROWS && (d->state_ld < d->channels || d->state_ld % 4 || d->state_ld > most_floats))
            return bad(op, "state_ld must be a multiple of 4, channels .. 2^40");
        // a prompt's rows are read by the workgroups of the rows after them; a single row by the lane that writes it
        const int64_t b = value_bytes(d->dtype);
        if ((d->cu || d->out != d->x || d->out_ld != d->x_ld) &&
            share_bytes(d->out, d->out_ld * b, d->channels * b, d->x, d->x_ld * b, d->channels * b, d->tokens))
            return bad(op, "out must not overlap x, unless it is x and there is no cu");
        if (d->tokens == 0) return sc::record_ok();
        sc::ConvArgs a{};
        a.x = static_cast<const uint8_t*>(d->x);
        a.out = static_cast<uint8_t*>(d->out);
        a.x_ld = d->x_ld * b;
        a.out_ld = d->out_ld * b;
        a.weight = d->weight;
        a.bias = d->bias;
        a.state = d->state;
        a.state_offset = d->state_offset;
        a.state_ld = d->state_ld;
        a.cu = d->cu;
        a.n_seqs = uint32_t(d->n_seqs);
        a.tokens = uint32_t(d->tokens);
        a.channels = uint32_t(d->channels);
        a.silu = d->activation == SC_CONV_SILU;
        return launched(sc::launch_conv(a, d->taps, d->dtype == SC_DTYPE_F16, d->state_layout == SC_CONV_SLOT,
                                        static_cast<hipStream_t>(stream)), op);
    });
}

int sc_gdn_step_async(const sc_gdn* d, void* stream) {
    return guarded([&] {
        sc::GdnArgs a{};
        if (const int e = gdn_args("gdn_step", d, true, a)) return e;
        if (!outputs_apart(d)) return bad("gdn_step", kOutputsMeet);
        return launched(sc::launch_gdn_step(a, int(d->state_size), d->dtype == SC_DTYPE_F16, static_cast<hipStream_t>(stream)),
                        "gdn_step");
    });
}

uint64_t sc_gdn_chunk_workspace_bytes(const sc_gdn* d) {
    sc::GdnArgs a{};
    if (guarded([&] { return gdn_args("gdn_chunk", d, false, a); }) != SC_OK) return 0;
    sc::ChunkArgs c;
    return sc::plan_gdn_chunks(a, int(d->state_size), d->dtype == SC_DTYPE_F16, c);
}

int sc_gdn_chunk_async(const sc_gdn* d, void* workspace, uint64_t workspace_bytes, void* stream) {
    return guarded([&] {
        const char* op = "gdn_chunk";
        sc::GdnArgs a{};
        if (const int e = gdn_args(op, d, false, a)) return e;
        if (!workspace || off(workspace, 256) || workspace_bytes < sc_gdn_chunk_workspace_bytes(d))
            return bad(op, "workspace missing, not 256-byte aligned or below sc_gdn_chunk_workspace_bytes");
        if (!outputs_apart(d)) return bad(op, kOutputsMeet);
        if (d->tokens == 0) return sc::record_ok();
        return launched(sc::launch_gdn_chunk(a, int(d->state_size), d->dtype == SC_DTYPE_F16, workspace,
                                             static_cast<hipStream_t>(stream)), op);
    });
}
