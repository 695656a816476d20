// Shared between the entry points of the losses (loss_api.hip), the kernels over rows (loss_rows.hip) and the
// matrix products (loss_product.hip). Not part of the public interface.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <tuple>

#include "jabas_loss.h"

namespace jabas {
namespace loss {

// What the backward pass needs of a row. With c = log2(e) / T, a token v that is no entry has the gradient
//     slope * 2^((z_v - peak_rest) c)   (minus e/V under label smoothing)
// and the entry (or label) j has   mass * 2^((z_j - peak) c) - p_j   (for a label: slope and 1 - e + e/V), all of it in
// units of upstream * T. Maxima and sums are kept apart, not as one log-sum-exp: at |lse| = 20 the rounding of a
// 32-bit lse alone is 1e-6 of every probability of its row. A row that does not count has slope = mass = 0.
struct RowState {
    float peak_rest, slope, peak, mass;
};
static_assert(sizeof(RowState) == 16, "a row's state is one 16-byte load");

// The row gradients dz travel between kernels as fp16 in units of 2^-15: |dz| <= 1 in units of upstream * T, so the range
// is used to the top and the smallest steps are 2^-39. Three more bits than bf16 at the same matrix rate; fp32 calls carry a
// second plane with 2^11 times what the first leaves: 22 bits down to 2^-25, smallest steps of 2^-50.
constexpr float kDzScale = 32768.0f, kLowScale = 2048.0f;

constexpr int kTile = 256;      // the largest output tile of a product; pieces of the vocabulary are whole ones
constexpr int kDepth = 64;      // elements of a product's inner axis are padded to a multiple of this
constexpr int64_t kMaxStride = int64_t{1} << 22;    // of an operand: offsets inside a tile are 32 bits

// An operand of a product, 16-byte aligned rows `stride` elements apart (at most kMaxStride); `plane` elements further on
// the second plane, where there is one. Either a row holds the inner axis, zeros up to the depth the call names, and there
// are `rows` of them; or there is a row for each place of the inner axis, zeros up to the depth, and it holds `rows` elements,
// a multiple of 8.
struct Operand {
    const void* p;
    int64_t stride, plane;
    int32_t rows;
};

// Entries of a row: the labels (entry_index NULL) or the teacher's.
struct Entries {
    const int64_t* target;
    int64_t ignore_index;
    const int32_t* index;
    const float* p;
    int32_t k;
};

struct LogitsArgs {
    Operand w, x;               // M = tokens of the piece, N = rows
    int32_t depth;              // padded width
    const float* unscale_w;     // factors that undo the scaling of the operands' rows, or NULL
    const float* unscale_x;
    const void* bias;           // of the whole vocabulary
    int32_t bias_dtype;
    int32_t first;              // first token of the piece
    float c;                    // log2(e) / T
    Entries entries;
    // forward
    float2* partial;            // [tile of the vocabulary][row]: maximum of the raw logits, sum of 2^((z - max) c)
    float* total;               // [tile][row]: sum of the logits (label smoothing), or NULL
    float* entry_logit;         // [row][max(k, 1)]
    // backward
    const RowState* state;
    const float* row_grad;      // gradient of row n in units of dz (bias gradient)
    float uniform;              // e / V
    float hit;                  // what a label takes off: 1 - e
    void* dz;                   // [row][token of the piece], fp16 planes, or NULL
    int64_t dz_stride, dz_plane;
    float* db;                  // [tile of the rows][token of the piece], or NULL
    int32_t pad_rows, pad_tokens;   // dz is written (with zeros) up to these
};

struct OutArgs {
    Operand a, b;               // out[n][m] = scale * row_scale[n] * sum_k a[k][m] b[n][k] (b_rows_of_k: b[k][n])
    int32_t b_rows_of_k;
    int32_t m, n;
    int32_t depth;
    const float* unscale0;      // device scalars, or NULL
    const float* unscale1;
    const float* row_scale;     // per n, or NULL
    float scale;
    float* acc;                 // fp32 sums over the pieces, or NULL where there is one piece
    int64_t acc_stride;         // a multiple of 4
    int32_t first, last;        // of the pieces
    void* out;
    int64_t out_stride;
    int32_t out_dtype;
    int32_t out_aligned;        // four elements of a row can be written at once
};

// Whether a product of m x n takes the large tiles, and how many of an operand's rows a tile of logits has.
bool large_tiles(int64_t m, int64_t n, int planes);
int logits_tile_tokens(bool large);
int logits_tile_rows(bool large, int planes);
int launch_logits_forward(const LogitsArgs& a, int planes, bool large, hipStream_t stream);
int launch_logits_backward(const LogitsArgs& a, int planes, bool large, hipStream_t stream);
int launch_out(const OutArgs& a, int planes, hipStream_t stream);

// Layout of operands: padded copies, split into fp16 planes and scaled by powers of two where the product asks for it.
constexpr int kMaxParts = 1024;
struct LayArgs {
    const void* in;
    int64_t in_stride;
    int32_t in_dtype;
    int32_t rows, cols;         // of `in`
    const float* row_factor;    // per row of `in`, or NULL: rows with factor 0 are zeros whatever they hold, others are multiplied
    const void* row_mask;       // per row of `in`, in_dtype, or NULL: rows with -inf here (tokens that the bias rules out) are zeros
    void* out;                  // [pad_rows][pad]
    int64_t out_stride, out_plane;
    int32_t pad_rows, pad;      // multiples of 8 columns
    int32_t planes;             // 0: copied as they are; 1 or 2 planes of fp16
    float* unscale;             // written: a factor per row (launch_lay_rows, planes > 0) or one for all (launch_lay_whole)
    float* parts;               // launch_lay_whole: kMaxParts partial maxima
};
int launch_lay_rows(const LayArgs& a, hipStream_t stream);
int launch_lay_whole(const LayArgs& a, hipStream_t stream);

// Rows.
struct TeacherArgs {
    const int64_t* index;
    const void* logits;
    int32_t dtype;
    const float* lse;
    int64_t rows, vocab;
    int32_t k;
    float inv_t;
    int32_t* entry_index;
    float* entry_p;
    float4* row;                // mass, sum p log p, counts, -
};
int launch_teacher(const TeacherArgs& a, hipStream_t stream);

struct JoinArgs {
    const float2* partial;
    const float* total;
    const float* entry_logit;
    int64_t rows, vocab;
    int32_t tiles;
    float c, inv_t, t;
    float smoothing;
    Entries entries;
    const float4* teacher_row;
    int32_t has_rest;           // teacher_lse was given
    RowState* state;
    float* row_loss;
};
int launch_join(const JoinArgs& a, hipStream_t stream);

// loss_out and reduce[0] = 1 / rows that count (mean) or 1
int launch_reduce(const float* row_loss, const RowState* state, int64_t rows, int reduction, float* loss_out, float* reduce, hipStream_t stream);

// grad[n] = upstream * T * reduce[0] (0 for rows that do not count), ratio[n] = grad[n] / *peak, *peak the largest |grad|
int launch_row_grad(const float* upstream, int per_row, const float* reduce, float t, const RowState* state, int64_t rows,
                    float* grad, float* ratio, float* peak, hipStream_t stream);

int launch_bias_sum(const float* parts, int32_t tiles, int64_t stride, int64_t n, void* out, int32_t dtype, hipStream_t stream);
int launch_zero(void* p, size_t bytes, hipStream_t stream);

struct TopkArgs {
    const void* logits;
    int64_t stride;
    int32_t dtype;
    int64_t rows, vocab;
    int32_t splits;
    int64_t chunk;              // tokens of a split
    float c;
    Entries entries;
    float2* partial;            // [split][row]
    float* entry_logit;
    const RowState* state;
    const float* row_grad;
    void* out;                  // [row][vocab]
};
int launch_topk_forward(const TopkArgs& a, hipStream_t stream);
int launch_topk_backward(const TopkArgs& a, hipStream_t stream);

}  // namespace loss
}  // namespace jabas
