/* lm_head.h: the C ABI of the LM head's pick and of its losses on MI355X (gfx950), in libdense_reader.so beside
 * dense_reader.h.
 *
 * An LM head run as dense_reader matmuls with top-k records (dr_matmul's dr_topk, bf16 keys) leaves, per row, the
 * best candidates of every 32-column tile of the vocabulary. These entry points turn the records into token ids on the
 * device, with nothing read back: per row an output page of 32 uint32 words, [token, the device's own best id, the
 * valid candidates' count, 0 ...].
 *
 * Reference interfaces replaced (XylolabsInc/tensix-kernels, paths relative to its root):
 *   dr_head_pick         <- lm_head_topk/head_pick.py:101-220 pick() and its kernels head_pick_reader.cpp,
 *                           head_pick_compute.cpp, head_pick_writer.cpp (the best `top` candidates by key, their exact
 *                           logits from the bf16 head rows, the pick of lmhead.py:40-46 pick_token)
 *   dr_head_pick_records <- lm_head_topk/head_pick.py:241-329 pick_records() and head_pick_records.cpp (the best
 *                           record by the device's own logit, through a token map)
 *
 * Both take plain device pointers and a hipStream_t (as void*), allocate nothing, and return DR_OK or a DR_E* status
 * of dense_reader.h. Many records are selected by several workgroups a row that meet in a workspace of
 * dr_topk_merge_workspace_bytes(n_records, rows, k) bytes (dense_reader.h; zeroed once by the caller, its counters
 * left at zero by every launch; launches sharing one must not overlap in time).
 */
#ifndef LM_HEAD_H
#define LM_HEAD_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* records [n_records][2 * rows * k] uint32 (dr_topk's bf16 records: keys, then ids); row r of x [rows][ldx] bf16
 * and the head table head [>= vocab][ld_head] bf16 (one row a token, dim columns used). Per row r < rows: the best
 * `top` (1 .. 32) valid slots by key, the earlier slot (record by record, slot by slot) first among equal keys; a slot
 * is valid when its key is not 0 and its id is below vocab. Their logits x[r] . head[id] summed in float32 (rounded to
 * bf16 with round_bf16), and the token is the lowest id among the largest logits, a NaN counting as the largest.
 * out [32][32] uint32: row r = [token (0 when no slot is valid), the first candidate's id (0xFFFFFFFF when none), the
 * candidates' count, 0 ...]. ids_out (or NULL): row 0's token also into ids_out[0]. rows <= 32; dim a multiple of 8;
 * x, head 16-byte aligned with ldx, ld_head multiples of 8. */
int dr_head_pick(const void* records, int n_records, int rows, int k, int top, int round_bf16, const void* x, int ldx,
                 int dim, const void* head, int64_t ld_head, int64_t vocab, void* out, void* ids_out, void* workspace,
                 int64_t workspace_bytes, void* stream);

/* The records' pick with no rescore: per row r < rows, the valid slot of the largest key (a NaN's key above all, -0's
 * equal to +0's), the earliest among equals; its id mapped through token_map (int32 [>= vocab], or NULL: the id).
 * out [32][32] uint32: row r = [token, the id, the valid slots' count, 0 ...] ([0, 0xFFFFFFFF, 0] when none).
 * ids_out (or NULL): row 0's token also into ids_out[0]. */
int dr_head_pick_records(const void* records, int n_records, int rows, int k, int64_t vocab, const void* token_map,
                         void* out, void* ids_out, void* workspace, int64_t workspace_bytes, void* stream);

/* The losses. A head [vocab][dim] bf16 (one row a token, as dr_head_pick reads it) against rows x [rows][dim] bf16:
 * z = x . head^T, float32 sums, of which no call has more than 2 GiB in memory (a call of both directions may keep that
 * much in its workspace, beside up to 1 GiB of their gradient). Per row, with lse = log(sum over v < valid of
 * exp(z[v] / T)):
 *   tokens (vals NULL, k 1, T 1): loss = lse - z[id];
 *   a teacher's best k logits (vals): over the entries held, q = softmax(vals / T),
 *     loss = sum q (log q - z[id] / T + lse), the divergence of the row's softmax at temperature T from the teacher's
 *     over its entries. An id that comes twice counts twice.
 * An entry is held when its id lies in 0 .. valid - 1 and (teacher) its value is not -inf. A row with no entry held is
 * left out: loss, lse, logits and dx 0, nothing into dhead, whatever x, g or vals hold there.
 *
 * Gradients of sum over rows of g[row] * loss[row]: dz[v] = g / T (p[v] - sum of q over entries of id v), p = exp(z / T -
 * lse); dx = dz . head, dhead = dz^T . x (rows valid .. vocab - 1 zeros). Piece by piece of the vocabulary (dz to 1 GiB)
 * z is computed again; a call of one piece may keep it in its workspace instead. dz is rounded to
 * bf16 (divided by the largest |g| of the rows that count, which the float32 sums get back, unless their weights lie
 * further apart than 2^40; up to 32 rows and one piece, what that leaves is rounded and summed too), the sums are
 * float32, dx and dhead rounded once.
 *
 * No counterpart in the reference, which has no training: the head and the teacher's records are its
 * lm_head_topk/head_pick.py:43-52 and dense_reader/linear.py:747-768.
 */
#define DR_LOSS_MAX_K 64
#define DR_LOSS_MAX_LD (1 << 21) /* ldx and ld_head at most */

/* what a call computes */
#define DR_LOSS_FORWARD 1  /* loss, lse, logits */
#define DR_LOSS_BACKWARD 2 /* dx, dhead, from lse and logits (a forward call's, of the same inputs) */

typedef struct dr_head_loss {
    const void* x;        /* [rows][ldx] bf16, 16-byte aligned, ldx a multiple of 8, to DR_LOSS_MAX_LD */
    int64_t ldx;
    const void* head;     /* [vocab][ld_head] bf16, the same */
    int64_t ld_head;
    int32_t rows, dim;    /* rows to 2^20, dim a multiple of 8; rows * valid to about 2^39 */
    int32_t vocab, valid; /* 1 <= valid <= vocab: the head's rows that take part */
    const void* ids;      /* [rows][ld_ids] int32, or int64 (ids64) */
    int64_t ld_ids;
    int32_t ids64;
    int32_t k;            /* entries a row, 1 .. DR_LOSS_MAX_K */
    const float* vals;    /* [rows][ld_vals] the teacher's logits, or NULL: tokens (k 1) */
    int64_t ld_vals;
    float temperature;    /* T from 2^-20 on, finite (tokens: 1) */
    float* loss;          /* [rows] */
    float* lse;           /* [rows] */
    float* logits;        /* [rows][k]: z at the entries (0 where none is held) */
    const float* g;       /* [rows], or NULL: ones */
    void* dx;             /* [rows][ld_dx] bf16, 16-byte aligned, ld_dx a multiple of 8, or NULL */
    int64_t ld_dx;
    void* dhead;          /* [vocab][ld_dhead] bf16, 16-byte aligned, ld_dhead a multiple of 8, or NULL */
    int64_t ld_dhead;
    void* workspace;      /* dr_head_loss_workspace_bytes, 256-byte aligned; its contents mean nothing between calls */
    int64_t workspace_bytes;
    void* stream;
} dr_head_loss;

/* Bytes of workspace the call needs (what: DR_LOSS_FORWARD, DR_LOSS_BACKWARD or both; dx and dhead NULL or not as in the call:
 * asked for neither, a backward needs and does nothing), -1 if it is invalid. */
int64_t dr_head_loss_workspace_bytes(const dr_head_loss* a, int what);

/* What the call launches, without launching it. A tile: rows and columns of the product, and the groups of wavefronts that
 * split its sum; 0 where the call makes no such product. */
typedef struct dr_head_loss_info {
    int32_t z[3];         /* the logits' tile (tokens by rows) for the loss */
    int32_t dz[3];        /* where they are computed again for their gradient */
    int32_t dhead[3];     /* (dim by tokens) */
    int32_t dhead_stages; /* of its K loop */
    int32_t dx[3];        /* (dim by rows) */
    int32_t dx_splits;    /* of its sum, where every row counts */
    int32_t piece, pieces; /* tokens whose dz is in memory at once, and how often */
    int32_t kept;         /* 1: the logits are kept from the loss to dz */
    int32_t few;          /* 1: few rows' launch between the products, 2: with what dz's rounding leaves */
} dr_head_loss_info;
int dr_head_loss_plan(const dr_head_loss* a, int what, dr_head_loss_info* info);

/* Enqueues the call on the stream: nothing is allocated, kept or waited for, so it can be captured. */
int dr_head_loss_run(const dr_head_loss* a, int what);

#ifdef __cplusplus
}
#endif

#endif
