/* z2b_ops.h — operators on device buffers around a decode step over a shared prompt
 * (libz2b.so, need a GPU).
 *
 * z2b_step runs these three steps inside its own graph, over the library's own KV pages and
 * one row or prompt per stream. The entry points here offer them for a caller's own model
 * code and caches, in the forms that streams sharing a prompt and carrying drafted tokens
 * need:
 *   z2b_rope_append       rotate the new rows' queries and keys, append keys and values to a
 *                         paged cache (beside the step's fixed interleaved full-head form)
 *   z2b_prefix_attention  attention of every stream over one shared prefix, read once for
 *                         all of them, and over its own paged rows
 *   z2b_verify_drafts     accept or replace drafted tokens against the target's
 *                         probabilities, from given random numbers (beside the step's sampler)
 *
 * Conventions, as in z2b.h: plain pointers and sizes, Z2B_OK or an error code, and
 * z2b_last_error() for the last failure of the calling thread. Every array is device memory
 * of `device`; the work is queued on `stream` (cudaStream_t of that device, NULL: its
 * default stream) and nothing is allocated, copied to the host or synchronised, so calls can
 * be captured into a CUDA graph. The calling thread's current device is left as it was.
 * Strides count elements. `err`, when not NULL, is a uint32 word on the device that the
 * kernels OR their findings into, never clearing it: Z2B_OPS_BAD_INDEX for offsets, lengths
 * or token ids out of range (the row is skipped, the token refused; offsets that descend:
 * z2b_prefix_attention skips every row) and for u_draw outside [0, 1), Z2B_OPS_BAD_PAGE for a
 * page id outside the cache (its keys read as zeros, its rows are not stored),
 * Z2B_OPS_TIMEOUT for a bounded wait that ran out (the results that needed it are not
 * numbers, with or without `err`). No input is dereferenced before it is
 * checked, with or without `err`.
 *
 * Rows: stream b of n_seq owns the packed rows [row_off[b], row_off[b+1]) of the n_rows rows
 * of q (row_off[0] >= 0, ascending, row_off[n_seq] <= n_rows; rows ahead of row_off[0] and behind
 * row_off[n_seq] are padding, which no call writes or lets into a result). seq_len[b] counts the
 * cached rows of the stream's own pages, its new rows included: new row i of n is cache row
 * seq_len[b] - n + i, which lives in row (that % page_len) of page
 * page_table[b * table_stride + that / page_len], and its position is prefix_len + that.
 */
#ifndef Z2B_OPS_H
#define Z2B_OPS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ggml type ids of the element types. */
#define Z2B_TYPE_F32 0
#define Z2B_TYPE_F16 1
#define Z2B_TYPE_BF16 30

#define Z2B_OPS_TIMEOUT 1u
#define Z2B_OPS_BAD_INDEX 2u
#define Z2B_OPS_BAD_PAGE 4u

/* ---- rotary position table ---------------------------------------------------------- */
#define Z2B_ROPE_MAX_DIM 256           /* rotated dims at most */
#define Z2B_ROPE_INTERLEAVED 0         /* pairs (2i, 2i + 1): ggml's normal layout */
#define Z2B_ROPE_HALF 1                /* pairs (i, i + rot_dim / 2) */
#define Z2B_ROPE_SCALE_NONE 0
#define Z2B_ROPE_SCALE_LINEAR 1        /* positions / factor */
#define Z2B_ROPE_SCALE_NTK 2           /* base * factor^(d / (d - 2)) */
#define Z2B_ROPE_SCALE_BY_PARTS 3      /* NTK-by-parts (Peng et al. 2023): pairs turning >= 32 times
                                          within orig_ctx keep their frequency, those turning <= 1
                                          time are divided by factor, linear in between; cos and sin
                                          times 0.1 ln(factor) + 1 */

/* Host-side plan of a rotation; plain data, usable on any device and thread. step[i] is pair
 * i's advance per position in turns, as a 64-bit fraction: position * step wraps modulo one
 * turn without rounding, so far positions lose nothing. */
typedef struct z2b_rope {
    int32_t rot_dim, layout;
    float mag;                         /* factor on cos and sin */
    int32_t reserved;
    uint64_t step[Z2B_ROPE_MAX_DIM / 2];
} z2b_rope;

/* Fill `out`. rot_dim even, 2..Z2B_ROPE_MAX_DIM (the first rot_dim dims of a head turn, the
 * others pass); base > 1; factor > 0, and 1 with SCALE_NONE; orig_ctx > 0 is read with
 * SCALE_BY_PARTS only; SCALE_NTK needs rot_dim > 2. The scaled base and frequencies have to be
 * finite and the factor on cos and sin positive. Host only. */
int z2b_rope_init(z2b_rope* out, int rot_dim, int layout, double base, int scaling, double factor, int orig_ctx);

/* ---- paged cache --------------------------------------------------------------------- */
/* A view of the caller's K and V pages of one layer: element d of head h of row r of page p
 * at k[p * page_stride + r * row_stride + h * head_stride + d]; v has the same strides. */
typedef struct z2b_paged_kv {
    void* k;
    void* v;
    int32_t type;                      /* Z2B_TYPE_F16 or Z2B_TYPE_BF16 */
    int32_t n_pages, page_len, n_head_kv, head_dim;
    int64_t page_stride, row_stride, head_stride;
} z2b_paged_kv;

/* ---- rotate and append ---------------------------------------------------------------- */
typedef struct z2b_rope_append_args {
    int32_t device;
    int32_t type;                      /* of q, q_out, k, v: F32, F16 or BF16 */
    int32_t n_rows, n_seq, n_head;     /* head_dim and n_head_kv are the cache's */
    int32_t prefix_len;
    const z2b_rope* rope;              /* host; NULL: no rotation */
    const z2b_paged_kv* kv;            /* host */
    const void* q;                     /* [n_rows][n_head][head_dim], or NULL with n_head 0 */
    void* q_out;                       /* rotated queries; may be q itself */
    const void* k;                     /* [n_rows][n_head_kv][head_dim], or NULL (with v) to only rotate q */
    const void* v;
    int64_t q_row, q_head, o_row, o_head, k_row, k_head, v_row, v_head;   /* strides */
    const int32_t* row_off;            /* [n_seq + 1] */
    const int32_t* seq_len;            /* [n_seq] */
    const int32_t* page_table;         /* [n_seq][table_stride], max_pages entries each */
    int64_t table_stride;
    int32_t max_pages;
    const int32_t* pos;                /* [n_rows] positions in place of prefix_len + cache row, or NULL */
    uint32_t* err;
} z2b_rope_append_args;

/* Rotate q into q_out and k into the cache, and store v, in one launch. Angles are exact to
 * f32 at any 32-bit position; the products are f32 and rounded once to their destination's
 * type. Of rows that name the same cache row parts of any stay. q_out is q itself or apart from q, k and
 * v, and no two places of q_out, or of the cache that is stored to, share memory. With k NULL only q turns: the
 * pages are not looked at, and max_pages may be 0. */
int z2b_rope_append(const z2b_rope_append_args* args, void* stream);

/* ---- attention over a shared prefix ---------------------------------------------------- */
typedef struct z2b_prefix_attn_args {
    int32_t device;
    int32_t n_rows, n_seq, n_head;     /* n_head a multiple of the cache's n_head_kv */
    int32_t prefix_len;                /* shared rows, >= 0 */
    float scale;                       /* on q . k, usually 1 / sqrt(head_dim); any sign, twice it finite */
    const z2b_paged_kv* kv;            /* host; head_dim 16, 32, 64 or 128; page_len a multiple of 8;
                                          k, v 16-byte aligned, strides multiples of 8 */
    const void* q;                     /* [n_rows][n_head][head_dim], the cache's type */
    void* out;                         /* the same shape and type */
    float* lse;                        /* [n_rows][n_head] natural log of the sum of exponentials, or NULL */
    int64_t q_row, q_head, o_row, o_head;   /* even */
    const int32_t* row_off;
    const int32_t* seq_len;
    const int32_t* page_table;
    int64_t table_stride;
    int32_t max_pages;
    const int32_t* prefix_pages;       /* [ceil(prefix_len / page_len)] */
    void* workspace;                   /* 16-byte aligned; contents before and after are of no meaning, so
                                          calls that do not run at the same time may share it */
    size_t workspace_bytes;            /* >= z2b_prefix_attention_workspace(args) */
    uint32_t* err;
} z2b_prefix_attn_args;

/* out[t] = softmax(scale q[t] . K) V over the prefix_len shared rows and the rows of the
 * stream's own pages up to the row's own; a row that sees none gives zeros and an lse of
 * -infinity. No two rows or heads of out share memory; it may lie across q. Products of 16-bit operands, sums and softmax statistics in f32, the
 * probabilities rounded to the cache's type for their product with V. Cache rows at or
 * behind seq_len and prefix_len may hold anything; those before and the scores must be finite,
 * and bf16 values of V below 2^80 (probabilities are held up to 2^15 ahead of their sum, so that
 * small ones keep their bits). A query that is not a number has a result that is not. The result
 * does not depend on timing: the same call gives the same bits. */
int z2b_prefix_attention(const z2b_prefix_attn_args* args, void* stream);
/* Workspace bytes of a call with these sizes and this cache (no other pointer is looked at); 0 for
 * bad ones. */
size_t z2b_prefix_attention_workspace(const z2b_prefix_attn_args* args);

/* ---- verification of drafts ------------------------------------------------------------ */
typedef struct z2b_verify_args {
    int32_t device;
    int32_t type;                      /* of p and q: F32, F16 or BF16 */
    int32_t n_seq, max_draft, n_codebooks, vocab;
    const void* p;                     /* target: [n_seq][max_draft + 1][n_codebooks][vocab] */
    const void* q;                     /* draft:  [n_seq][max_draft][n_codebooks][vocab], or NULL: the draft put
                                          all its probability on the drafted token */
    const int32_t* draft;              /* [n_seq][max_draft][n_codebooks] token ids */
    const int32_t* n_draft;            /* [n_seq] drafted frames, 0..max_draft, or NULL: max_draft each */
    const double* u_accept;            /* [n_seq][max_draft][n_codebooks] uniforms in [0, 1) */
    const double* u_draw;              /* [n_seq][max_draft + 1][n_codebooks], in [0, 1) too */
    int32_t* tokens;                   /* [n_seq][max_draft + 1][n_codebooks]: accepted frames, one more frame, -1 behind */
    int32_t* n_accepted;               /* [n_seq] */
    int64_t p_seq, p_frame, p_book, q_seq, q_frame, q_book;   /* strides; vocab is contiguous */
    uint32_t* err;
} z2b_verify_args;

/* Speculative sampling over frames of n_codebooks independent tokens. A drafted token x is
 * kept when u_accept * q(x) < p(x); the first frame with a refused token ends the run, and
 * each refused token of it is replaced by a draw from max(p - q, 0) (from p where that is
 * zero everywhere); when all drafts are kept, one frame more is drawn from p. Frames then
 * follow the target's distribution exactly. A draw takes the first token whose running sum
 * (64 bits) exceeds u_draw * total; a u_draw below 0 counts as 0, any other outside [0, 1) draws
 * the last token with mass; a row of p without any mass gives -1. A p(x) or q(x) that is
 * not a number refuses its token, a difference that is not a number counts as zero in a draw. */
int z2b_verify_drafts(const z2b_verify_args* args, void* stream);

#ifdef __cplusplus
}
#endif
#endif
