/* grads.h: the C ABI of a model's gradients as a whole on MI355X (gfx950): their global norm, and clipping by it, in
 * libdense_reader.so beside dense_reader.h.
 *
 *   norm = sqrt(sum over all values of all tensors of v^2); factor = min(1, max_norm / (norm + 1e-6)); out = v factor
 *
 * Squares and their sums are float64 (no float32 overflows or is lost), each out is rounded once from the float32 product. A NaN
 * among the values makes the norm and every out NaN; an infinity makes the norm infinite, the factor 0 and its own out NaN. An infinite
 * max_norm is no limit: the factor is 1 unless the norm is NaN.
 *
 * No counterpart in the reference, which has no training.
 */
#ifndef GRADS_H
#define GRADS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* a tensor's type */
#define DR_GRADS_F32 0
#define DR_GRADS_BF16 1
#define DR_GRADS_F16 2

typedef struct dr_grads {
    int32_t count;            /* tensors, to 2^20 */
    const void* const* in;    /* each one's values, at a multiple of their size (fastest at one of 16) */
    const int64_t* sizes;     /* values of each, 0 or more, to 2^40 in all */
    const int32_t* types;
    void* const* out;         /* clip: where each one's values go, its own in (of the same type) or memory apart from every other's and the norm's */
    const int32_t* out_types;
    double max_norm;          /* clip: 0 or more, an infinity too */
    float* norm;              /* written; a clip with `given` reads it */
    int32_t given;            /* clip: norm holds the norm (of more gradients than these, say) */
    void* workspace;          /* dr_grads_workspace_bytes, 8-byte aligned; its contents mean nothing between calls */
    int64_t workspace_bytes;
    void* stream;
} dr_grads;

/* Bytes of workspace that a call over these tensors needs, -1 if it is invalid: at most DR_GRADS_LIST_BYTES for every DR_GRADS_LIST
 * tensors begun. */
#define DR_GRADS_LIST 128
#define DR_GRADS_LIST_BYTES 16384
int64_t dr_grads_workspace_bytes(const dr_grads* a);

/* Enqueue the norm, or the norm (unless given) and the clip, on the stream: nothing is allocated on the device, kept or waited for,
 * so a call can be captured. The lists are read before they return. */
int dr_grads_norm(const dr_grads* a);
int dr_grads_clip(const dr_grads* a);

#ifdef __cplusplus
}
#endif

#endif
