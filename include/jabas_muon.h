/*
 * jabas_muon.h -- C ABI of libjabas_sync.so: orthogonalised updates of weight matrices on one MI355X (gfx950).
 *
 * A matrix G is taken to the polynomial of it that a few Newton-Schulz products make: with X of the shorter side first
 * (m x n, m <= n),
 *
 *   X = G / max(|G|_F, eps);    steps times:  A = X X^T,  X = a X + (b A + c A A) X
 *
 * whose singular vectors are G's and whose singular values all lie near one. jabas_orthogonalize does that to a batch of
 * matrices of one shape; jabas_muon_step makes an optimizer's step of it over a list of matrices of any shapes:
 *
 *   buf = buf + (1 - momentum) (g - buf);   u = g + momentum (buf - g) with nesterov, else buf
 *   w = w (1 - lr weight_decay) - lr lr_factor orthogonalised(u);   replicas of w are written too
 *
 * as torch.optim.Muon defines it (state under the same name and of the same size). It stands beside the optimizers of
 * jabas_sync.h, which the reference's examples build over their models (examples/vit/main.py:425-437); the reference itself has no
 * update that looks at a whole matrix.
 *
 * Precision. precision JABAS_F32: every factor of a product is two fp16 planes, a product three of theirs: 22 bits of X's
 * entries down to 2^-14 of the largest singular value that it can have (1 at first, then what the polynomial makes of that), steps of 2^-36
 * of it below. JABAS_BF16: one plane and one product, 11 bits of each factor; X itself keeps 22, so that directions that are weak in G do not lose theirs to the rounding of strong ones. Sums are fp32, |G|_F fp64.
 * A matrix that holds an infinity or a NaN becomes NaN as a whole.
 *
 * Conventions are those of jabas_sync.h: caller-owned device memory, no allocation, no synchronisation, all work on the
 * stream passed in, negative status before anything is launched. Results are the same from run to run.
 */
#ifndef JABAS_MUON_H
#define JABAS_MUON_H

#include "jabas_sync.h"

#ifdef __cplusplus
extern "C" {
#endif

#define JABAS_MUON_MAX_STEPS 32
#define JABAS_MUON_MAX_SIDE (1ll << 16)     /* the shorter side of a matrix */
#define JABAS_MUON_MAX_LENGTH (1ll << 22)   /* the longer one               */

typedef struct JabasNewtonSchulz {
    double a, b, c;                 /* may not let singular values grow past 256 (JABAS_ERR_OPT) */
    double eps;                     /* positive                                                   */
    int32_t steps;                  /* 1..JABAS_MUON_MAX_STEPS                                    */
    int32_t precision;              /* JABAS_F32 or JABAS_BF16, see above                         */
} JabasNewtonSchulz;

/* A batch of matrices of one shape. `in` and `out` may not overlap (JABAS_ERR_ALIAS). */
typedef struct JabasOrthogonalize {
    const void* in;                 /* [batch][rows][cols], cols contiguous                       */
    void* out;                      /* [batch][rows][cols] contiguous, of the same type           */
    int64_t batch, rows, cols;      /* any of them may be 0                                       */
    int64_t in_batch_stride, in_row_stride;     /* elements                                       */
    int32_t dtype;                  /* JABAS_F32 or JABAS_BF16                                    */
    int32_t reserved;
    JabasNewtonSchulz ns;
} JabasOrthogonalize;

size_t jabas_orthogonalize_workspace_bytes(const JabasOrthogonalize* o);    /* 0: refused by the call */
/* workspace: 256-byte aligned. */
int jabas_orthogonalize(const JabasOrthogonalize* o, void* workspace, size_t workspace_bytes, jabas_stream_t stream);

/* One matrix of a step; all buffers contiguous. Every written buffer (momentum, param, fanout) must be disjoint from the other
 * buffers of its matrix (JABAS_ERR_ALIAS); overlap between matrices is the caller's responsibility. Any element alignment. */
typedef struct JabasMatrix {
    const float* grad;
    float* momentum;
    float* param;
    float* fanout[JABAS_MAX_K - 1]; /* replicas that receive the new weights                      */
    int64_t rows, cols;             /* at least 1                                                 */
    double lr_factor;               /* what the group's lr is multiplied by for this shape        */
    uint32_t group;                 /* below JABAS_MAX_GROUPS                                     */
    uint32_t n_fanout;
} JabasMatrix;

/* The launch-invariant description of a list of matrices, as jabas_plan_encode makes one of spans: validated and encoded
 * into host memory, copied to the device once by the caller (16-byte aligned), both passed to every step. Pure host code.
 * Matrices go through the workspace some at a time, in order of their sides, so that it does not grow past 512 MiB with the
 * list (one that needs more is alone in it). At most 2^20 matrices. */
size_t jabas_muon_plan_bytes(const JabasMatrix* matrices, uint32_t n, int32_t precision);       /* what is enough; 0: refused by encode */
int jabas_muon_plan_encode(const JabasMatrix* matrices, uint32_t n, int32_t precision, void* host_blob, size_t blob_bytes);
size_t jabas_muon_workspace_bytes(const void* host_blob);       /* 0 on a malformed blob */

typedef struct JabasMuonArgs {
    JabasNewtonSchulz ns;           /* precision: the plan's (JABAS_ERR_PLAN otherwise)           */
    double momentum;                /* in [0, 1)                                                  */
    int32_t nesterov;
    int32_t n_groups;
    double lr[JABAS_MAX_GROUPS], weight_decay[JABAS_MAX_GROUPS];
    const float* grad_scale;        /* device scalar c or NULL: gradients are multiplied by c when c < 1 (clipping) */
} JabasMuonArgs;

/* Two launches and three for every Newton-Schulz step, per part of the list; one in all where a workgroup's LDS holds any of the matrices. */
int jabas_muon_step(const void* plan_host, const void* plan_dev, const JabasMuonArgs* args,
                    void* workspace, size_t workspace_bytes, jabas_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* JABAS_MUON_H */
