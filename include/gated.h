/* gated.h: the C ABI of the gated feed-forward block in training on MI355X (gfx950), in libdense_reader.so beside
 * dense_reader.h.
 *
 * Weights gate, up [width][dim] bf16 (one row an output, as a linear layer holds them) against rows x [rows][dim] bf16:
 *   g = x . gate^T, u = x . up^T (float32 sums), h = a(g) u, with a(g) = g / (1 + exp(-g)) or gelu's tanh form;
 * and of dh [rows][width] bf16, the gradient of h:
 *   dg = dh u a'(g), du = dh a(g); dx = dg . gate + du . up, dgate = dg^T . x, dup = du^T . x.
 *
 * dg and du are rounded to bf16, which the matrix instructions take; sums are float32, h, dx, dgate and dup rounded once. What a
 * forward call keeps for its gradients is g and u in 24 bits each (float32 without the last 8 of the mantissa, cut off), which a
 * backward call of the same act makes a(g) and a'(g) of; one that is given none computes g and u again (two products more).
 *
 * No counterpart in the reference, which has no training: the block is its fused GLU stage (dense_reader/linear.py:568-744,
 * glu and glu_act) with weights as a training program holds them.
 */
#ifndef GATED_H
#define GATED_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define DR_GATED_MAX_LD (1 << 21) /* ldx, ld_gate, ld_up at most */

/* what a call computes */
#define DR_GATED_FORWARD 1  /* h, and kept unless it is NULL */
#define DR_GATED_BACKWARD 2 /* dx, dgate, dup (those that are not NULL) from dh and kept, or with kept NULL from x again */

typedef struct dr_gated {
    const void* x;    /* [rows][ldx] bf16; this and all below 16-byte aligned, with lds multiples of 8 */
    int64_t ldx;
    const void* gate; /* [width][ld_gate] bf16 */
    int64_t ld_gate;
    const void* up;   /* [width][ld_up] bf16 */
    int64_t ld_up;
    int32_t rows, dim, width; /* rows to 2^20, dim to 2^17, width to 2^20, multiples of 8 but the rows; rows * width below 2^38 */
    int32_t act;      /* 0 silu, 1 gelu_tanh (dense_reader.h's); of a backward call that of the call that kept */
    void* h;          /* [rows][ld_h] bf16 */
    int64_t ld_h;
    void* kept;       /* dr_gated_kept_bytes, or NULL */
    const void* dh;   /* [rows][ld_dh] bf16 */
    int64_t ld_dh;
    void* dx;         /* [rows][ld_dx] bf16, or NULL */
    int64_t ld_dx;
    void* dgate;      /* [width][ld_dgate] bf16, or NULL */
    int64_t ld_dgate;
    void* dup;        /* [width][ld_dup] bf16, or NULL */
    int64_t ld_dup;
    void* workspace;  /* dr_gated_workspace_bytes, 256-byte aligned; its contents mean nothing between calls */
    int64_t workspace_bytes;
    void* stream;
} dr_gated;

/* Bytes that a forward call keeps for its gradients (rows and width alone decide), -1 if the call is invalid. */
int64_t dr_gated_kept_bytes(const dr_gated* a);

/* Bytes of workspace the call needs (0: none), -1 if it is invalid. */
int64_t dr_gated_workspace_bytes(const dr_gated* a, int what);

/* What the call launches, without launching it. A tile: rows and columns of the product, and the groups of wavefronts that
 * split its sum; 0 where the call makes no such product. */
typedef struct dr_gated_info {
    int32_t act[3];    /* (gate's and up's outputs by rows) g and u, for h or for dg and du */
    int32_t dweight[3]; /* (dim by outputs) */
    int32_t dweight_stages; /* of its K loop */
    int32_t dx[3];     /* (dim by rows) */
    int32_t dx_splits; /* of its sum */
    int32_t act_once;  /* 1: act reads each weight once, past the caches */
} dr_gated_info;
int dr_gated_plan(const dr_gated* a, int what, dr_gated_info* info);

/* Enqueues the call on the stream: nothing is allocated, kept or waited for, so it can be captured. */
int dr_gated_run(const dr_gated* a, int what);

#ifdef __cplusplus
}
#endif

#endif
