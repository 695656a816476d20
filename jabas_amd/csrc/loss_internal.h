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
// second plane with 2^11 times what the first leaves: 22 bits down to 2^-25, smallest steps of 2^-50. Where a row's probabilities sum
// to more than 1 (a teacher_lse below its entries', a token named often) |dz| is as much larger: then a power of two of the row's own, `down`,
// takes its dz into the range, and its row gradient carries the inverse. No row has a say in another's steps.
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

// The rows that count, in order: row c of the products is row map[c] of the call, c < *live; map holds the others behind them. Rows that do
// not count cost nothing but this.
struct Live {
    const int32_t* map;
    const int32_t* live;
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
    Operand w, x;               // M = tokens of the piece, N = rows that count (at most x.rows of them)
    Live rows;
    int32_t depth;              // padded width
    const float* unscale_w;     // factors that undo the scaling of the operands' rows, or NULL
    const float* unscale_x;
    const void* bias;           // of the whole vocabulary
    int32_t bias_dtype;
    int32_t first;              // first token of the piece
    float c;                    // log2(e) / T
    Entries entries;
    // forward
    float2* partial;            // [tile of the vocabulary][row that counts]: maximum of the raw logits, sum of 2^((z - max) c)
    float* total;               // [tile][row that counts]: sum of the logits (label smoothing), or NULL
    float* entry_logit;         // [row of the call][max(k, 1)]
    // backward
    const RowState* state;
    const float* row_grad;      // gradient of row n in units of dz (bias gradient)
    const float* down;          // [row of the call]: see kDzScale, with entries
    float uniform;              // e / V
    float hit;                  // what a label takes off: 1 - e
    void* dz;                   // [row that counts][token of the piece], fp16 planes, or NULL
    int64_t dz_stride, dz_plane;
    float* db;                  // [tile of the rows][token of the piece], or NULL
    int32_t pad_tokens;         // dz is written (with zeros) up to this, and to whole steps of rows
};

// out[n][m] = scale * row_scale[n] * sum_k a[m][k] b[n][k] (rows_of_k: b[k][n]), the inner axis in `splits` ranges of `each`
// elements (the last may be shorter), whose sums are joined afterwards where there are several.
struct Job {
    Operand a, b;
    int32_t m, n, depth, splits, each;
    Live rows;
    int32_t live_depth;         // the inner axis is the rows that count: `depth` is what they are at most
    int32_t live_n;             // n is
    const float* unscale0;      // device scalars, or NULL
    const float* unscale1;
    const float* unscale_m;     // per m, readable up to a multiple of four, or NULL
    const float* row_scale;     // per row of the call, or NULL
    float scale;
    float* part;                // fp32 sums [split][n][part_stride] over the pieces of the inner axis, or NULL: written to `out` at once
    int64_t part_stride, part_plane;        // a multiple of 4; splits apart
    int32_t first;              // of the pieces: what `part` holds does not count
    int32_t keep;               // the sums stay in `part`, to be joined or added to; else they go to `out` with what `part` holds
    void* out;
    int64_t out_stride;
    int32_t out_dtype;
    int32_t out_aligned;        // four elements of a row can be written at once
};
// The gradients' products of a piece in one launch: `w` sums over rows of k of dz, `h` over contiguous ones. Either may have m = 0.
struct GradArgs {
    Job w, h;
    int32_t h_first;            // workgroups of h come first: they take longer
};
// Whether the logits of a piece take the large tiles, and how many tokens and rows a tile of logits has.
bool large_tiles(int64_t tokens, int64_t rows, int planes, bool backward);
int logits_tile(bool large);
int launch_logits_forward(const LogitsArgs& a, int planes, bool large, hipStream_t stream);
int launch_logits_backward(const LogitsArgs& a, int planes, bool large, hipStream_t stream);
struct Splits { int w, h; };
// How often to split the inner axes of a piece's products: features x tokens over `rows`, features x rows over `tokens`.
Splits choose_splits(int64_t features, int64_t tokens, int64_t rows, bool w, bool h, bool many_pieces, int planes);
int launch_grads(GradArgs& a, int planes, hipStream_t stream);
int launch_join_splits(const Job& j, hipStream_t stream);

// Layout of operands: padded copies, split into fp16 planes and scaled by powers of two where the product asks for it.
constexpr int kMaxParts = 1024, kPeakParts = 64;
struct LayArgs {
    const void* in;
    int64_t in_stride;
    int32_t in_dtype;
    int32_t rows, cols;         // of `in`
    Live live;                  // the rows of `in` that are laid out, or all of them
    const float* row_factor;    // per row of `in`, or NULL: rows with factor 0 are zeros whatever they hold, others are multiplied
    const void* row_mask;       // per row of `in`, in_dtype, or NULL: rows with -inf here (tokens that the bias rules out) are zeros, but for those
    const uint32_t* named;      // whose bit of the vocabulary is set here: they are a label or an entry, with a dz of their own
    int32_t first;              // token of row 0
    void* out;                  // launch_lay_rows: [rows][pad]; launch_lay_columns: [cols][pad]
    int64_t out_stride, out_plane;
    int32_t pad;                // a multiple of 64
    int32_t planes;             // 0: copied as they are; 1 or 2 planes of fp16
    float low;                  // what the second plane is multiplied by: 1 or kLowScale
    void* zero;                 // launch_lay_rows: [row of the call][cols] of in_dtype whose rows that do not count are zeroed, or NULL
    uint32_t* name;             // launch_lay_rows: zeros, in which the bits of the rows' labels and entries are set, or NULL
    Entries entries;
    int64_t vocab;
    float* unscale;             // written: a factor per row (launch_lay_rows, planes > 0), or (launch_lay_columns) one for all, with peaks per column
    float* peaks;               // launch_lay_columns: [kPeakParts][peak_stride] partial maxima of the columns, or NULL
    int64_t peak_stride;
    float* parts;               // kMaxParts partial maxima; launch_lay_rows: NULL, or one scale for all rows, written to unscale_all too
    float* unscale_all;
    int32_t pad_rows;           // launch_lay_rows with parts: places from rows to here become zeros
};
int launch_lay_rows(const LayArgs& a, hipStream_t stream);
int launch_lay_columns(const LayArgs& a, hipStream_t stream);

// Rows.
struct TeacherArgs {
    const int64_t* index;
    const void* logits;
    int32_t dtype;
    const float* lse;
    int64_t rows, vocab;
    int32_t k;
    float inv_t, t;
    int32_t* entry_index;
    float* entry_p;
    float4* row;                // mass, sum p log p, counts, -
};
int launch_teacher(const TeacherArgs& a, hipStream_t stream);

struct JoinArgs {
    Live live;                  // of launch_join
    const float2* partial;
    const float* total;
    const float* entry_logit;
    int64_t rows, vocab;
    int32_t tiles;
    float c;
    float smoothing;
    Entries entries;
    const float4* teacher_row;
    TeacherArgs teacher;
    RowState* state;
    float* row_loss;
    // launch_join: the last workgroup to finish reduces over the rows
    uint32_t* ticket;
    int32_t reduction;
    float* loss_out;
    float* reduce;
};
int launch_join(const JoinArgs& a, hipStream_t stream);
int launch_narrow_join(const JoinArgs& a, hipStream_t stream);        // a workgroup per row; partial and total: [row][tile]

// loss_out and reduce[0] = 1 / rows that count (mean) or 1
int launch_reduce(const float* row_loss, const RowState* state, int64_t rows, int reduction, float* loss_out, float* reduce, hipStream_t stream);

// Which rows count: map and *live; the others' state and loss become zeros.
struct LiveArgs {
    const int64_t* target;
    int64_t ignore_index;
    const float4* teacher_row;  // instead of labels
    int64_t rows;
    int32_t *map, *live;
    uint32_t* ticket;           // set to 0
    RowState* state;
    float* row_loss;
};
int launch_live(const LiveArgs& a, hipStream_t stream);

// down[n] of rows x k entries: see kDzScale
int launch_down(const float* p, int64_t rows, int32_t k, float* down, hipStream_t stream);

// grad[n] = upstream * T * reduce[0] / down[n] (0 for rows that do not count), ratio[n] = grad[n] / *peak, *peak the largest |grad|, and which rows
// have a grad.
struct RowGradArgs {
    const float* upstream;
    int32_t per_row;
    const float* reduce;        // the share of a row
    const float* down;          // or NULL: 1
    float t;
    const RowState* state;
    int64_t rows;
    float *grad, *ratio, *peak;
    int32_t *map, *live;
    uint32_t* zero;             // `zeros` words set to 0, or NULL
    int64_t zeros;
};
int launch_row_grad(const RowGradArgs& a, hipStream_t stream);

// out[i] = sum of parts[t][i] over the tiles of `tile` rows that count
int launch_bias_sum(const float* parts, const int32_t* live, int32_t tile, int64_t stride, int64_t n, void* out, int32_t dtype, hipStream_t stream);
int launch_zero(void* p, size_t bytes, hipStream_t stream);

// Few rows, hidden states and weight as they lie (loss_narrow.hip). With bf16, whose tiles read the weight as it lies too, a second block
// of rows pays for small weights only. Forward and backward, this and the tiles: fp32 16 x 32317 x 1024 170 and 434 us, 64 x 32317 x 1024 320
// and 457, 64 x 131072 x 4096 3805 and 8716; bf16 1 x 32317 x 1024 107 and 171, 32 x 32317 x 1024 119 and 176, 32 x 131072 x 4096 1225 and
// 2070, 64 x 4000 x 768 72 and 89, 64 x 8000 x 768 76 and 101, 64 x 16000 x 768 103 and 117,
// 40 x 32317 x 1024 188 and 176, 64 x 32317 x 1024 209 and 177.
constexpr int kNarrowRows = 64;
constexpr int64_t kNarrowWeight = int64_t{12} << 20;       // elements of the weight
struct NarrowArgs {
    const void *x, *w, *bias;
    int64_t x_stride, w_stride, vocab;
    int32_t rows, width;
    float c;
    Entries entries;
    // forward
    float2* partial;            // [row][tile]
    float* total;               // [row][tile], or NULL
    float* entry_logit;
    uint32_t* ticket;           // set to 0
    // backward
    const RowState* state;
    const float* upstream;
    int32_t per_row;
    const float* reduce;
    float t;
    float uniform, hit;
    float* dz;                  // [32 or 64 rows][dz_stride tokens], in the units of the result, or NULL; bf16: two planes, and once more by tokens
    int64_t dz_stride;          // the tokens in whole tiles
    void* d_bias;
    void* d_weight;
    void* d_hidden;
    int64_t first, tokens;      // of the piece, from a whole tile on
    int64_t hidden_units;       // workgroups of dX
    int64_t each;               // tokens of a split
    float* part;                // [split][row][part_stride], or NULL: one split, one piece
    int64_t part_stride, part_plane;
    int32_t add;                // to what `part` holds
};
int64_t narrow_tiles(int64_t vocab);
struct NarrowSplits { int64_t each; int32_t n; };
NarrowSplits narrow_splits(int64_t tokens, int64_t width);
int launch_narrow_forward(const NarrowArgs& a, int dtype, hipStream_t stream);
int launch_narrow_backward(const NarrowArgs& a, int dtype, hipStream_t stream);
int launch_narrow_grads(const NarrowArgs& a, int dtype, hipStream_t stream);

// Logits in hand. One split: a workgroup per row; else a workgroup per `chunk` tokens of a row.
struct TopkArgs {
    const void* logits;
    int64_t stride;
    int32_t dtype;
    int64_t rows, vocab;
    int32_t splits;
    int64_t chunk;              // a multiple of 32
    float c, t;
    TeacherArgs teacher;
    float2* partial;            // [row][split]
    RowState* state;
    float* row_loss;            // where a row has parts: and, behind the rows' losses, whether they count
    uint32_t* ticket;
    int32_t reduction;
    float *loss_out, *reduce_out;
    Entries entries;            // backward
    const float* upstream;
    int32_t per_row;
    const float* reduce;
    void* out;                  // [row][vocab]
};
int launch_topk_forward(const TopkArgs& a, hipStream_t stream);
int launch_topk_backward(const TopkArgs& a, hipStream_t stream);

}  // namespace loss
}  // namespace jabas
