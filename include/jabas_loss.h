/*
 * jabas_loss.h -- C ABI of the losses in libjabas_sync.so: what ends a worker's forward pass over a large
 * vocabulary (or a set of classes) and starts its backward pass, on one MI355X (gfx950).
 *
 *   z_nv = sum_h x_nh w_vh + b_v       (or logits in hand)
 *   cross entropy, smoothing e:    L_n = lse_n - (1-e) z_n,t(n) - (e/V) sum_v z_nv,   lse_n = log sum_v exp z_nv
 *   distillation, temperature T:   q = softmax(z/T) over the whole vocabulary, the teacher's probabilities p_j at
 *                                  the entries i_j:  L_n = T^2 ( sum_j p_j (log p_j - log q_{i_j}) + rest )
 *     without teacher_lse: p = softmax of the entries' logits / T, rest = 0
 *     with teacher_lse:    p_j = exp(t_j/T - teacher_lse_n); what the entries leave, r = max(0, 1 - sum p), is one
 *                          more event: rest = r (log r - log R), R = q of all tokens that are no entry
 *                          (rest = 0 where every token is an entry; where there are others and all of them are at
 *                          -inf, R = 0: an infinite loss where r > 0, and no gradient for them)
 *
 * The conventions of jabas_sync.h hold: plain C types, caller-owned device memory, nothing allocated, freed or
 * synchronised, all work on the stream passed in, a negative JabasStatus before anything is launched. Nothing is
 * kept between calls but what the caller keeps (row_state, entry_index, entry_p).
 *
 * Rows that do not count (target == ignore_index; no teacher entry) have loss 0 and gradient 0 whatever their
 * hidden state or logits hold, and a row whose upstream gradient is 0 has gradient 0. A label, or a teacher index,
 * outside the vocabulary (a negative teacher index is "no entry") makes its row's loss and gradients NaN; no memory
 * outside the tensors is read.
 *
 * Row gradients dL/dz of many rows (over 64; bf16 over a large weight: 32) are held in fp16 between kernels: 11 bits
 * (bf16 calls) or 22 (fp32) of them, and below 2^-29 or 2^-25 of the row's upstream gradient times T in steps of 2^-39 or
 * 2^-50 of it; few rows keep 16 and 24 bits at any size.
 *
 * Sizes: from hidden and weight rows <= 2^22, vocab <= 2^28, width <= 2^20 and less than 2^23 tiles of 256 rows and 256
 * tokens; over logits rows times the parts of 32768 tokens of a row (more of them where rows are few) less than 2^24,
 * vocab <= 2^30. Others are JABAS_ERR_SIZE.
 */
#ifndef JABAS_LOSS_H
#define JABAS_LOSS_H

#include "jabas_sync.h"

#ifdef __cplusplus
extern "C" {
#endif

#define JABAS_LOSS_MAX_ENTRIES 255   /* entries of a teacher per row */

enum { JABAS_LOSS_NONE = 0, JABAS_LOSS_MEAN = 1, JABAS_LOSS_SUM = 2 };   /* reduction over the rows */

/* One loss. Element strides; every row is contiguous. hidden and weight, or logits, are set; target, or
 * teacher_index and teacher_logits. */
typedef struct JabasLoss {
    const void*    hidden;          /* rows x width, dtype                                                 */
    const void*    weight;          /* vocab x width, dtype                                                */
    const void*    bias;            /* vocab, dtype, or NULL                                               */
    const void*    logits;          /* rows x vocab, dtype (teacher only), instead of hidden and weight    */
    int64_t        hidden_stride, weight_stride, logits_stride;
    int64_t        rows, vocab, width;
    int32_t        dtype;           /* JABAS_F32 or JABAS_BF16: of hidden, weight, bias, logits, teacher_logits
                                       and of the gradients                                                 */
    int32_t        reduction;       /* JABAS_LOSS_*                                                         */
    const int64_t* target;          /* rows labels                                                          */
    int64_t        ignore_index;
    double         label_smoothing; /* 0 <= e < 1                                                           */
    const int64_t* teacher_index;   /* rows x entries, contiguous; negative: no entry                       */
    const void*    teacher_logits;  /* rows x entries, contiguous, dtype; -inf: no entry                    */
    const float*   teacher_lse;     /* rows: log sum exp(t/T) over the teacher's whole vocabulary, or NULL  */
    int64_t        entries;         /* 1..JABAS_LOSS_MAX_ENTRIES with a teacher, else 0                     */
    double         temperature;     /* > 0; 1 without a teacher                                             */
    /* written by the forward pass, read by the backward pass */
    float*         row_state;       /* 4 * rows + 4 floats, 16-byte aligned                                 */
    int32_t*       entry_index;     /* rows x entries (teacher only)                                        */
    float*         entry_p;         /* rows x entries (teacher only)                                        */
} JabasLoss;

/* Bytes of device workspace (256-byte aligned) of the forward or the backward call; 0 where `loss` is malformed.
 * The backward call works through the vocabulary in pieces, so its workspace does not grow with rows x vocab. */
size_t jabas_loss_workspace_bytes(const JabasLoss* loss, int32_t backward);

/* loss_out: rows floats (JABAS_LOSS_NONE) or one. Rows that do not count add nothing, and the mean over no rows
 * is 0. Counterpart of the criterion a trainer calls on its model's output (jabas/train/trainer.py:82-86). */
int jabas_loss_forward(const JabasLoss* loss, float* loss_out, void* workspace, size_t workspace_bytes,
                       jabas_stream_t stream);

/* upstream: the gradient of loss_out, one float or (JABAS_LOSS_NONE) one per row, on the device. d_hidden (rows x
 * width), d_weight (vocab x width) and d_bias (vocab), any of them NULL where it is not wanted, or d_logits (rows x
 * vocab): contiguous, dtype, written whole. */
int jabas_loss_backward(const JabasLoss* loss, const float* upstream, void* d_hidden, void* d_weight, void* d_bias,
                        void* d_logits, void* workspace, size_t workspace_bytes, jabas_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* JABAS_LOSS_H */
