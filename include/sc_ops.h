/* sc_ops.h - the operators that run on a decode slot between two hand-offs, in libsc_handoff.so.
 *
 * A hand-off (sc_handoff.h) puts a sequence's paged K/V and its Gated-DeltaNet state into a decode slot.  These entry
 * points compute on such slots: new tokens' keys and values appended with the position rotation on the way (by one position a
 * token, or by several axes'), attention of one new token a sequence over its paged cache, the cells that attention has use for
 * kept and the others evicted, and the short convolution and the gated delta rule by single tokens and by whole prompts.
 *
 * Like every entry point of the library they take plain pointers, return a status of sc_handoff.h (the message in
 * sc_last_error()), let no exception out, check a request before anything is enqueued (SC_EINVAL / SC_ERANGE: nothing
 * launched, nothing written), allocate nothing and only enqueue kernels on `stream` (a hipStream_t; NULL is the null
 * stream), so a call can be captured into a graph.  Pointers are device pointers unless a name says host.
 * Lengths, positions, page tables and state pointers lie in device memory and are read when the kernels run; the host
 * gets bounds only.  What they say is bounded there: a row, cell or page outside its buffers is left out, never touched.
 */
#ifndef SC_OPS_H
#define SC_OPS_H

#include <stddef.h>
#include <stdint.h>

#include "sc_handoff.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- paged caches ------------------------------------------------------------------------------------------------- */

/* One layer's K and V cache of many sequences, in the decode layout: the row of cell t and kv head h is
 * (page * n_head_kv + h) * page_size + t % page_size of either pool, page = table[s * table_ld + t / page_size] for
 * sequence s.  Rows are head_dim f16 values (SC_KV_F16) or head_dim int8 codes with one f16 scale per 64 values in the
 * scale pools (SC_KV_INT8, the rule of sc_kv_append_async).  A page that is negative or not below n_pages is not
 * resident: a write to its cells is skipped, a read leaves them out.  Slots in q4_0 or K8V4
 * are not taken. */
typedef struct sc_kv_cache {
    int32_t format;           /* SC_KV_F16 or SC_KV_INT8 */
    int64_t n_head_kv;        /* 1 .. 256 */
    int64_t head_dim;         /* 64, 128 or 256 */
    int64_t page_size;        /* cells in a page, 1 .. 65536 */
    int64_t n_pages;          /* physical pages of each pool; n_pages * n_head_kv * page_size < 2^31 rows */
    void* k;                  /* [n_pages][n_head_kv][page_size][head_dim], 16-byte aligned */
    void* v;
    uint16_t* k_scale;        /* [n_pages][n_head_kv][page_size][head_dim / 64], 8-byte aligned; NULL for f16 */
    uint16_t* v_scale;
    const int32_t* table;     /* [n_seqs][table_ld] logical -> physical page; NULL: sequence s's logical page p is
                                 physical page s * table_ld + p (one sequence: the identity table) */
    int64_t table_ld;         /* logical pages of a sequence: it has at most table_ld * page_size cells, < 2^31 */
} sc_kv_cache;

/* ---- rotated append ------------------------------------------------------------------------------------------------ */

/* Which values of a head turn together. */
enum { SC_ROPE_HALVES = 0,       /* value i with value i + rot_dim / 2 */
       SC_ROPE_NEIGHBOURS = 1 }; /* value 2 i with value 2 i + 1 */

typedef struct sc_rope_append {
    int64_t tokens;           /* rows in k, v and q, of all sequences together, at most 2^23 */
    int32_t n_seqs;           /* 1 .. 4096 */
    const int64_t* cu;        /* [n_seqs + 1] ascending from 0: rows [cu[s], cu[s + 1]) are sequence s's; a row past
                                 cu[n_seqs] belongs to none and is left out.  NULL: row s is sequence s's (tokens ==
                                 n_seqs) */
    const int64_t* pos0;      /* [n_seqs] the cell of sequence s's first row, which is its position */
    int32_t dtype;            /* SC_DTYPE_F16 or SC_DTYPE_F32: k, v, q and q_out */
    const void* k;            /* [tokens][n_head_kv][head_dim], k_ld values from token to token */
    const void* v;
    const void* q;            /* [tokens][n_head][head_dim], or NULL: no queries */
    void* q_out;              /* the rotated queries; may be q itself (then q_out_ld == q_ld) */
    int64_t k_ld, v_ld, q_ld, q_out_ld;  /* multiples of 4 (f32) or 8 (f16) values, at most 2^22 */
    int64_t n_head;           /* query heads, 0 without q, at most 4096 */
    int32_t pairing;          /* SC_ROPE_* */
    int64_t rot_dim;          /* the first rot_dim values of a head are rotated: a multiple of 8, 0 .. head_dim */
    const float* inv_freq;    /* [rot_dim / 2] radians a position; angles are formed in 64 bits */
} sc_rope_append;

/* For each row: the first rot_dim values of every key and query head are rotated by position * inv_freq[i] (a, b ->
 * a cos - b sin, a sin + b cos), keys and values are written to the cache in its format (f16 by round to nearest even,
 * int8 by sc_kv_append_async's rule), queries to q_out.  A position before 0 or past the table is not written.  One
 * launch. */
int sc_rope_append_async(const sc_kv_cache* cache, const sc_rope_append* a, void* stream);

/* Positions of several axes (time, height, width): a pair of a head turns by the position that its row has on the pair's axis. */
typedef struct sc_rope_axes {
    int32_t n_axes;           /* 1 .. 4 */
    const uint8_t* host_axis; /* host [rot_dim / 2]: the axis of pair i, below n_axes; read before the call returns */
    const int64_t* pos;       /* [n_axes][pos_ld]: the position of every row on every axis, 8-byte aligned */
    int64_t pos_ld;           /* at least `tokens` */
} sc_rope_axes;

/* sc_rope_append_async with these positions: a->pos0 is only the cell of a sequence's first row, so a cell need not be its
 * token's position (after a picture, whose tokens share positions, or after an eviction).  Angles are formed in 64 bits from
 * positions of any sign.  One launch. */
int sc_rope_axes_append_async(const sc_kv_cache* cache, const sc_rope_append* a, const sc_rope_axes* axes, void* stream);

/* ---- paged attention of one new token ------------------------------------------------------------------------------- */

typedef struct sc_attn_decode {
    int32_t n_seqs;           /* 1 .. SC_ATTN_MAX_SEQS */
    const int64_t* lens;      /* [n_seqs] cells each sequence attends over, its new token's among them; < 0 counts as 0,
                                 more than max_len as max_len */
    int64_t max_len;          /* host bound on every length, at most table_ld * page_size; sizes the launch and workspace */
    int64_t window;           /* 0: every cell; else the last `window` cells of each sequence */
    int32_t dtype;            /* SC_DTYPE_F16 or SC_DTYPE_F32: q and out */
    int64_t n_head;           /* query heads, a multiple of n_head_kv: head i reads kv head i / (n_head / n_head_kv) */
    const void* q;            /* [n_seqs][n_head][head_dim], q_ld values from sequence to sequence, 16-byte aligned */
    void* out;                /* likewise with out_ld; must not overlap q */
    int64_t q_ld, out_ld;     /* multiples of 4 (f32) or 8 (f16) values, at most 2^22 */
    float* lse;               /* [n_seqs][n_head], or NULL */
    float scale;              /* scores are scale * q . k */
} sc_attn_decode;
#define SC_ATTN_MAX_SEQS 1024

/* out = softmax(scale * q . K) V over the resident cells of the window, and lse = log of the sum of the exponentials
 * (natural), which joins the result with one over other cells.  Sums and softmax statistics in 32 bits; f16 queries are
 * exact, weights and f32 queries are carried as two f16 parts in units of their own size, so f32 results keep f32 accuracy,
 * also where one cell outweighs the rest by up to 2^80.  Infinite values that are attended make what the formula makes of
 * them.  A sequence with no cell left (or whose every score is -inf) gets zeros and lse = -inf.  What lies in cells outside
 * the sequence does not matter.  The cache's length is split over the chip on the device from the lengths and the parts are joined by
 * a second kernel; the result does not depend on timing. */
uint64_t sc_attn_decode_workspace_bytes(const sc_kv_cache* cache, const sc_attn_decode* a);
int sc_attn_decode_async(const sc_kv_cache* cache, const sc_attn_decode* a, void* workspace, uint64_t workspace_bytes,
                         void* stream);

/* ---- what attention has use for ------------------------------------------------------------------------------------------ */

typedef struct sc_attn_mass {
    int32_t n_seqs;           /* 1 .. SC_ATTN_MAX_SEQS */
    const int64_t* lens;      /* [n_seqs] cells of each sequence, its latest rows' among them; < 0 counts as 0, more than
                                 max_len as max_len */
    int64_t max_len;          /* host bound on every length, at most table_ld * page_size */
    int64_t window;           /* 0, or the attention's window: a row sees the last `window` of its cells */
    int64_t rows;             /* R: the latest queries of each sequence, at least 1; rows * n_head / n_head_kv <= 1024 */
    int32_t dtype;            /* SC_DTYPE_F16 or SC_DTYPE_F32: q */
    int64_t n_head;           /* query heads, a multiple of n_head_kv, at most 4096 */
    const void* q;            /* [n_seqs * R][n_head][head_dim], the rotated queries, q_ld values from row to row, 16-byte
                                 aligned: row r of a sequence is the query of its cell len - R + r, and sees the cells up to it */
    int64_t q_ld;             /* a multiple of 4 (f32) or 8 (f16) values, at most 2^22 */
    const float* lse;         /* [n_seqs * R][n_head] the log of each query's sum of exponentials as the attention left it
                                 (sc_attn_decode's lse), or NULL: formed here, from the same cells */
    float scale;              /* scores are scale * q . k */
    float decay;              /* what the mass that is there is multiplied by; 0: it is overwritten, whatever it is */
    float* mass;              /* [n_seqs][n_head_kv][mass_ld], 4-byte aligned */
    int64_t mass_ld;          /* at least max_len, at most 2^31 - 1 */
} sc_attn_mass;

/* mass[s][h][c] = decay * mass[s][h][c] + sum over the rows and the query heads of kv head h of exp(scale * q . k_c - lse), for
 * the cells below each sequence's length; the rest of `mass` is left as it is.  A cell that a row does not see, or that is not
 * resident, gets nothing from it; a row that sees no cell, or whose every score is -inf, gives none, nor does a query whose
 * `lse` is -inf, whatever it holds.  A score of +inf weighs inf under a finite `lse`, and NaN under one of +inf, under which the
 * query's finite scores weigh nothing; where the sum is formed here, a query with a score of +inf or NaN makes NaN of every cell that
 * it sees.  f16 queries are exact, f32 ones two f16 parts of 22 bits or more together, sums in 32 bits; the result does not depend on
 * timing.  Reads the keys only, once with `lse` and twice without; one to four launches, or for more than 16 columns of max_len
 * beyond 2^29 up to four for each time.  A mass that begins at 0 and is never decayed sums to the number of queries so far times heads. */
uint64_t sc_attn_mass_workspace_bytes(const sc_kv_cache* cache, const sc_attn_mass* a);
int sc_attn_mass_async(const sc_kv_cache* cache, const sc_attn_mass* a, void* workspace, uint64_t workspace_bytes, void* stream);

typedef struct sc_kv_evict {
    int32_t n_seqs;           /* 1 .. SC_ATTN_MAX_SEQS */
    const int64_t* lens;      /* [n_seqs] cells of each sequence; < 0 counts as 0, more than max_len as max_len */
    int64_t max_len;          /* host bound on every length, at most table_ld * page_size */
    int64_t keep;             /* cells that a sequence may keep, at least 1: one that has no more is left as it is */
    int64_t sinks;            /* its first tokens and its latest ones are kept whatever their mass: sinks + recent <= keep */
    int64_t recent;
    const float* mass;        /* [n_seqs][n_head_kv][ld], 4-byte aligned */
    float* mass_out;          /* likewise, or `mass` itself: the mass of the cells that are kept, at their new places, and 0 in the
                                 rest of the old length */
    const int32_t* born;      /* [n_seqs][n_head_kv][ld] the number of the token that each cell holds (0 the first), or NULL */
    int32_t* born_out;        /* likewise, or `born` itself, or NULL: the numbers of the cells that are kept */
    int64_t ld;               /* of all four: at least max_len, 1 .. 2^31 - 1 */
    const int64_t* known;     /* [n_seqs] cells whose number `born` holds, the last eviction's lens_out: later cells are the latest
                                 tokens in order.  Given with `born`; NULL: no cell's */
    const int64_t* total;     /* [n_seqs] tokens so far, evicted ones too, below 2^31; NULL: the lengths, nothing was evicted */
    int64_t* lens_out;        /* [n_seqs] the new lengths, min(length, keep); may be lens, known or total */
} sc_kv_evict;

/* Of each kv head of each sequence with more than `keep` cells, keeps `keep`: the first `sinks` tokens, the `recent` latest, then
 * those with the largest mass (equal ones from the lowest cell on, NaN last).  A kept cell below `keep` stays; the others' rows (keys,
 * values, scales) move to the places below `keep` that have become free, in ascending order both.  Cells from `keep` on keep
 * what they hold and are no longer the sequence's: their pages can be given to others.  So a cache is in no order after this:
 * attention over it needs none, but a window by cells means nothing there, and positions are given to the next append apart from its
 * cells (sc_rope_axes_append_async).  Each kv head keeps cells of its own.  Nothing else that is kept by cell moves along (an
 * indexer's pooled rows, sc_slot_layers).  The pages below a length are to be resident and the
 * sequence's own: a row is neither read from nor written to a page that is not resident.  One launch where a head can
 * move 128 cells at most and lens_out shares nothing with what it is made from, else two, or five for long heads that several
 * workgroups share; the result does not depend on timing.  Layers that share an array of lengths need lens_out apart from it. */
uint64_t sc_kv_evict_workspace_bytes(const sc_kv_cache* cache, const sc_kv_evict* a);
int sc_kv_evict_async(const sc_kv_cache* cache, const sc_kv_evict* a, void* workspace, uint64_t workspace_bytes, void* stream);

/* ---- the short convolution before a recurrent layer --------------------------------------------------------------------- */

enum { SC_CONV_NONE = 0, SC_CONV_SILU = 1 };             /* what is applied to the sums */
enum { SC_CONV_SLOT = 0,       /* history [channels][taps - 1], a slot's GDN row from S * HV * S floats on */
       SC_CONV_ROWS = 1 };     /* history [taps - 1][state_ld], the last rows of a prefill's convolution inputs */

typedef struct sc_conv {
    int64_t channels;         /* C: a multiple of 8, 8 .. 2^20 */
    int32_t taps;             /* W: 2 .. 5 */
    int32_t n_seqs;           /* 1 .. 4096 */
    int64_t tokens;           /* rows of x and out, at most 2^23 */
    const int64_t* cu;        /* [n_seqs + 1] as in sc_rope_append, a sequence's rows in order; NULL: row s is sequence s's one
                                 new token (tokens == n_seqs) */
    int32_t dtype;            /* SC_DTYPE_F16 or SC_DTYPE_F32: x and out */
    const void* x;            /* [tokens][C], x_ld values from row to row, 16-byte aligned */
    void* out;                /* [tokens][C]; shares no byte with x, but may be x itself without cu (then out_ld == x_ld) */
    int64_t x_ld, out_ld;     /* multiples of 4 (f32) or 8 (f16) values, at most 2^22 */
    const float* weight;      /* [C][W], 16-byte aligned: weight[c][W - 1] meets the row itself */
    const float* bias;        /* [C], 16-byte aligned, or NULL */
    int32_t activation;       /* SC_CONV_NONE or SC_CONV_SILU */
    float* const* state;      /* device [n_seqs]: each sequence's base, 16-byte aligned, none of them twice; a NULL entry is a
                                 sequence without a slot: its out rows are zeros.  A history shares no byte with x or out */
    int64_t state_offset;     /* floats from the base to this layer's history, a multiple of 4 (e.g. layer * sc_gdn_row_floats +
                                 S * HV * S), at most 2^40 */
    int32_t state_layout;     /* SC_CONV_SLOT or SC_CONV_ROWS; the oldest row first in both */
    int64_t state_ld;         /* SC_CONV_ROWS: floats from row to row, a multiple of 4, C .. 2^40 */
} sc_conv;

/* out[t][c] = f(bias[c] + sum over j of weight[c][j] * x[t - (W - 1) + j][c]), the rows before a sequence's first being its
 * history, and the history becomes the last W - 1 rows of both together.  Sums in 32 bits; f is v / (1 + exp(-v)) for
 * SC_CONV_SILU.  A sequence without rows keeps its history; rows past cu[n_seqs] are left out.  One launch. */
int sc_conv_async(const sc_conv* a, void* stream);

/* ---- the gated delta rule --------------------------------------------------------------------------------------------- */

/* For each value head, with its state M [key][value] in f32, and per token its key k, query q, value v, log decay g and
 * write strength beta:
 *     M <- exp(g) M;   u = beta (v - M^T k);   M <- M + k u^T;   out = scale * M^T q
 * with k and q divided by sqrt(sum of squares + eps) first when l2norm is set.  Value head h takes key head
 * h / (v_heads / k_heads).  The layout of the GDN rows the hand-off moves. */
typedef struct sc_gdn {
    int64_t k_heads, v_heads; /* v_heads a multiple of k_heads; at most 1024 */
    int64_t state_size;       /* S: values of a head, 32, 64 or 128 */
    int32_t n_seqs;           /* 1 .. 4096 */
    int64_t tokens;           /* rows of q, k, v, g, beta and out, at most 2^23 */
    const int64_t* cu;        /* chunk form: [n_seqs + 1] as in sc_rope_append; step form: NULL (row s is sequence s's) */
    int32_t dtype;            /* SC_DTYPE_F16 or SC_DTYPE_F32: q, k, v and out */
    const void* q;            /* [tokens][k_heads][S], q_ld values from token to token, 16-byte aligned */
    const void* k;
    const void* v;            /* [tokens][v_heads][S] */
    void* out;                /* [tokens][v_heads][S]; may be v itself (then out_ld == v_ld), and shares no byte with q, k or
                                 the rest of v: refused by the calls that enqueue */
    int64_t q_ld, k_ld, v_ld, out_ld;   /* multiples of 4 (f32) or 8 (f16) values, at most 2^22 */
    const float* g;           /* [tokens][v_heads], <= 0 (below -200 counts as -200, whose decay is 0 as well) */
    const float* beta;        /* [tokens][v_heads] */
    int64_t gate_ld;          /* values from token to token of g and beta, at most 2^22 */
    float scale;
    int32_t l2norm;
    float eps;
    float* const* state;      /* device [n_seqs]: each sequence's base, 16-byte aligned; a NULL entry is a sequence without
                                 a slot: its out rows are zeros */
    int64_t state_offset;     /* floats from the base to this layer's state (e.g. a multiple of sc_gdn_row_floats) */
    int64_t state_head_ld;    /* floats between heads: S in a slot's (S, HV, S) row, S * S in the prefill layout */
    int64_t state_key_ld;     /* floats between keys: HV * S in a slot's row, S in the prefill layout.  All three multiples of 4, at
                                 most 2^40; the heads lie inside a key's row or the keys inside a head's block */
} sc_gdn;

/* One token of every sequence (tokens == n_seqs): state read, updated in place, one launch. */
int sc_gdn_step_async(const sc_gdn* a, void* stream);
/* Every sequence's tokens in order (a prompt, or a piece of one: the state goes on from what it holds).  A sequence
 * without tokens keeps its state; rows past cu[n_seqs] are left out.  Sums, states and the products of a chunk's rows with each
 * other in 32 bits; products with the state run on the matrix cores in two f16 parts of each column's own size, which keep f32
 * accuracy.  Infinities and NaN stay in the heads that they belong to, and reach no output before the 16 tokens (of a chunk of 64,
 * from the sequence's first) that they are among.  The result does not depend on timing. */
uint64_t sc_gdn_chunk_workspace_bytes(const sc_gdn* a);
int sc_gdn_chunk_async(const sc_gdn* a, void* workspace, uint64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* SC_OPS_H */
