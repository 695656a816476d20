// Shared by the sources of the orthogonalised update.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "jabas_muon.h"

namespace jabas {
namespace muon {

constexpr int kPad = 64;            // sides of the copies that the products read are multiples of this
constexpr int kParts = 1024;        // partial sums of a matrix's length, at most
constexpr int kMinChunk = 4096;     // elements of one of them, at least
constexpr int kLay = 64;            // tile of the pass that lays a matrix out

// One matrix as the kernels see it. The products work on X, m x n with m <= n: the matrix, or (tall) its transpose.
struct Matrix {
    const void* src;                // the gradient
    float* momentum;                // NULL: none, X is made of src
    void* out;                      // the weights (with momentum), else where X goes
    int64_t src_stride;             // of a row
    int64_t x_at, a_at, part_at;    // places in the workspace: X (two buffers of two planes) and A, B in halves, partial sums in doubles
    int64_t x_plane, a_plane;       // halves of a plane of X, of A
    int32_t rows, cols;             // of src and out
    int32_t m, n, pad_m, pad_n;
    int32_t tall;
    int32_t src_quads, out_quads;   // four elements at a time: all rows of src (and momentum), of out (and replicas) allow it
    int32_t parts, chunk;           // partial sums, elements of each
    int32_t group;
    float lr_factor;
    uint32_t n_fanout, fanout_at;   // replicas: pointers in the list's table
};

// Where element (row, col) of a matrix with `pad` columns lies, in halves, and how far behind its first plane its second is. Products of two planes read them
// from one line, 32 of either by turns; a product of one plane reads nothing of the second.
template <int P>
__host__ __device__ inline int64_t stride_of(int pad) { return P == 2 ? 2 * static_cast<int64_t>(pad) : pad; }
template <int P>
__host__ __device__ inline int64_t half_at(int row, int col, int pad) { return row * stride_of<P>(pad) + (P == 2 ? (col >> 5) * 64 + (col & 31) : col); }
template <int P>
__host__ __device__ inline int64_t second_of(int64_t plane) { return P == 2 ? 32 : plane; }

// Which workgroup does what. A list: `table` and a slot {matrix, tile} for every workgroup. A batch: matrix 0 and what lies between it and
// the next one.
struct Slot {                       // with what the products need of the matrix, so that they start one read of memory earlier
    uint32_t matrix, tile;
    int32_t m, n;
    int64_t x_at, a_at;
    uint32_t unit;                  // of the matrix's first workgroup in this launch
    int32_t splits;                 // workgroups that share a tile's inner axis: workgroup s of a tile is `tile` = s tiles + tile
};
struct Work {
    const Matrix* table;
    const Slot* slots;
    const uint64_t* fanout;
    Matrix one;
    int64_t src_step, out_step;     // bytes
    int64_t x_step, a_step, part_step;
    int32_t per, splits;            // workgroups of a matrix, and of a tile
    uint32_t total;                 // workgroups that have something to do
    void* halves;                   // workspace
    double* sums;
};

// A pass over the gradients: momentum and partial sums (launch_momentum), or the copy (launch_lay).
struct PassArgs {
    Work w;
    int32_t dtype;                  // of src
    int32_t nesterov;
    float momentum, fresh;          // momentum and 1 - momentum
    const float* grad_scale;
    double eps;
    float scale;                    // of X's planes
    int32_t planes;                 // of the products
    uint32_t* tickets;              // launch_momentum: set to zero
    uint32_t n_tickets;
};
int launch_momentum(const PassArgs& a, hipStream_t stream);
int launch_lay(const PassArgs& a, hipStream_t stream);

// X X^T (second: b A + c A A), written whole though half of it is computed; scales: powers of two.
struct SymmetricArgs {
    Work w;
    int32_t from;                   // buffer of X
    float own, product;             // result = own A + product acc
    float* shares;                  // a tile's sums over a part of the inner axis, 4096 of every workgroup
    uint32_t* tickets;              // how many of a tile's workgroups are done; zero before and after
};
// The last step's result: into the weights (lr by group, keep = 1 - lr weight_decay), or as it is, of `dtype`.
struct Out {
    int32_t dtype;
    float lr[JABAS_MAX_GROUPS], keep[JABAS_MAX_GROUPS];
};
// X <- a X + B X
struct UpdateArgs {
    Work w;
    int32_t from;
    int32_t last;                   // goes to out, scaled by 1
    float own, product;
    Out out;
};
// The products' kernels: their tiles and what tells them apart.
enum Kind { kSmall, kSmallMany, kMiddle, kMiddleDeep, kLarge, kKernels };     // 64, four stages or two; 128, two stages or four; 256
constexpr int kTile[kKernels] = {64, 64, 128, 128, 256};
int launch_symmetric(const SymmetricArgs& a, bool second, int planes, Kind kind, hipStream_t stream);
int launch_update(const UpdateArgs& a, int planes, Kind kind, hipStream_t stream);

// Everything of small matrices in one launch, one workgroup each. `blocks` of 32 cover the shorter side of all of them.
constexpr int kTinyBytes = 160 * 1024 - 256;        // of LDS
struct TinyStep {
    float first, second_own, second, update_own, update;
};
struct TinyArgs {
    PassArgs pass;
    Out out;
    int32_t steps;
    TinyStep step[JABAS_MUON_MAX_STEPS];
};
bool tiny_fits(int blocks, int64_t n);
int launch_tiny(const TinyArgs& a, int blocks, hipStream_t stream);

inline int64_t symmetric_tiles(int64_t m, int tile) { const int64_t t = (m + tile - 1) / tile; return t * (t + 1) / 2; }
inline int64_t update_tiles(int64_t m, int64_t n, int tile) { return (m + tile - 1) / tile * ((n + tile - 1) / tile); }

}  // namespace muon
}  // namespace jabas
