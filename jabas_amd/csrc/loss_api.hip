// Entry points of the losses: argument validation, workspace layout, and the order of the launches.
#include <math.h>

#include "loss_internal.h"

#define JABAS_API extern "C" __attribute__((visibility("default")))

namespace jabas {
namespace loss {
namespace {

constexpr int64_t kMaxSize = int64_t{1} << 30;      // rows, tokens; the tiles' numbers and tokens are 32 bits in the kernels
constexpr int64_t kMaxLinearVocab = int64_t{1} << 28;
constexpr int64_t kMaxGroups = int64_t{1} << 23;    // a launch has less than 2^32 threads, up to 512 a workgroup
constexpr int64_t kMaxWidth = int64_t{1} << 20;
constexpr int64_t kMaxLinearRows = kMaxStride;      // a feature's hidden states are one row of an operand

inline int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
inline int64_t tiles(int64_t n, int64_t tile) { return (n + tile - 1) / tile; }
inline size_t element_bytes(int dtype) { return dtype == JABAS_F32 ? 4 : 2; }

// Tokens whose row gradients are kept at once: 64 MiB at most. 32 x 262144 x 1024 fp32 with 2^14, 2^16, 2^17 and 2^18: 1684, 1435, 1455 and
// 1426 us.
constexpr int64_t kNarrowPiece = int64_t{1} << 17;

struct Shape {
    bool linear, teacher, narrow;
    int planes;                 // of the operands: fp32 takes two
    int64_t depth;              // padded width
    bool copy_w;                // the products cannot read the weight as it is
};

bool misaligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

void cut_rows(const JabasLoss* l, bool forward, int64_t& splits, int64_t& chunk);

int validate(const JabasLoss* l, Shape& s) {
    if (!l) return JABAS_ERR_NULL;
    if (l->dtype != JABAS_F32 && l->dtype != JABAS_BF16) return JABAS_ERR_DTYPE;
    s.linear = l->hidden || l->weight;
    s.teacher = l->entries != 0 || l->teacher_index || l->teacher_logits;
    if (l->reduction < JABAS_LOSS_NONE || l->reduction > JABAS_LOSS_SUM) return JABAS_ERR_SIZE;
    if (l->rows < 0 || l->rows > kMaxSize || l->vocab < 1 || l->vocab > kMaxSize) return JABAS_ERR_SIZE;
    if (s.linear) {
        if (!l->weight || (!l->hidden && l->rows) || l->logits) return JABAS_ERR_NULL;
        if (l->rows > kMaxLinearRows || l->width < 1 || l->width > kMaxWidth || l->hidden_stride < 0 || l->weight_stride < 0) return JABAS_ERR_SIZE;
        if (l->vocab > kMaxLinearVocab || tiles(l->rows, kTile) * tiles(l->vocab, kTile) >= kMaxGroups) return JABAS_ERR_SIZE;
    } else {
        if ((!l->logits && l->rows) || l->bias || !s.teacher) return JABAS_ERR_NULL;
        int64_t splits, chunk;
        cut_rows(l, false, splits, chunk);
        if (l->logits_stride < 0 || splits * l->rows >= 2 * kMaxGroups) return JABAS_ERR_SIZE;
    }
    if (s.teacher) {
        if (l->target || ((!l->teacher_index || !l->teacher_logits || !l->entry_index || !l->entry_p) && l->rows)) return JABAS_ERR_NULL;
        if (l->entries < 1 || l->entries > JABAS_LOSS_MAX_ENTRIES) return JABAS_ERR_SIZE;
        if (!(l->temperature > 0.0) || !isfinite(l->temperature) || l->label_smoothing != 0.0) return JABAS_ERR_SIZE;
    } else {
        if (!l->target && l->rows) return JABAS_ERR_NULL;
        if (!(l->label_smoothing >= 0.0 && l->label_smoothing < 1.0) || l->temperature != 1.0 || l->teacher_lse) return JABAS_ERR_SIZE;
    }
    if (!l->row_state) return JABAS_ERR_NULL;
    const size_t bytes = element_bytes(l->dtype);
    if (misaligned(l->row_state, 16) || misaligned(l->hidden, bytes) || misaligned(l->weight, bytes) || misaligned(l->bias, bytes) ||
        misaligned(l->logits, bytes) || misaligned(l->teacher_logits, bytes) || misaligned(l->teacher_index, 8) || misaligned(l->target, 8) ||
        misaligned(l->teacher_lse, 4) || misaligned(l->entry_index, 4) || misaligned(l->entry_p, 4))
        return JABAS_ERR_ALIGN;
    s.planes = l->dtype == JABAS_F32 ? 2 : 1;
    s.narrow = s.linear && l->rows > 0 && l->rows <= kNarrowRows &&
               (l->dtype == JABAS_F32 || l->rows <= kNarrowRows / 2 || l->vocab * l->width <= kNarrowWeight);
    s.depth = round_up(s.linear ? l->width : 1, kDepth);
    s.copy_w = !(s.planes == 1 && l->width % kDepth == 0 && l->weight_stride % 8 == 0 && l->weight_stride <= kMaxStride && !misaligned(l->weight, 16));
    return JABAS_OK;
}

// Workspace: 256-byte aligned pieces one after the other. Without memory it only counts.
struct Carver {
    char* base;
    size_t used;
    template <class T>
    T* take(size_t n) {
        T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
        used += (n * sizeof(T) + 255) / 256 * 256;
        return p;
    }
    size_t all() const { return used ? used : 256; }
};

// Tokens of a piece: what the pieces' copies may take is bounded, and a piece has whole tiles.
// fp32's pieces are larger: their planes take twice the bytes, and a piece's start and end more time. Forward and backward with 128, 256 and
// 768 MiB: 4096 x 131072 x 4096 bf16 15.38, 15.19 and 15.17 ms; 1024 x 131072 x 1024 fp32 4.66, 4.64 and 4.04; 2048 x 65536 x 4096 fp32
// 14.90, 13.59 and 13.04.
constexpr int64_t kPieceBytes[2] = {int64_t{256} << 20, int64_t{768} << 20};
int64_t piece_tokens(const JabasLoss* l, const Shape& s, bool backward) {
    int64_t per_token = 0;
    if (s.copy_w) per_token += s.depth * 2 * s.planes;
    if (backward) per_token += (round_up(l->rows, kDepth) + (s.planes == 1 ? s.depth : 0)) * 2 * s.planes;     // dz, bf16's weight in fp16
    if (!per_token) return round_up(l->vocab, kTile);
    int64_t n = kPieceBytes[s.planes - 1] / per_token / kTile * kTile;
    if (n < 4 * kTile) n = 4 * kTile;
    const int64_t whole = round_up(l->vocab, kTile);
    if (n >= whole) return whole;
    const int64_t pieces = (whole + n - 1) / n;         // of about one size
    return round_up((whole + pieces - 1) / pieces, kTile);
}

struct Forward {
    float2* partial;
    float* total;
    float* entry_logit;
    float4* teacher_row;
    float* row_loss;
    uint16_t *x, *w;
    float *unscale_x, *unscale_w;
    uint32_t* ticket;
    int32_t *map, *live;
    int64_t piece, splits, chunk;
    int64_t tiles;
    bool large;
};

// Logits in hand, workgroups per row, as many as their masks of entries (a bit a token) ask for, LDS's 32 KiB each, and more for a few
// long rows. Forward, the parts of a row cost a launch that joins them, so that only rows of kLongRow on are cut where there are less
// than kFullRows: 16 x 131072 bf16 25.7 us whole, 19.3 in parts; 16 x 49152 18.4 and 18.1; 16 x 16000 fp32 18.2 and 20.1;
// 192 x 131072 30.3 and 28.3; 256 x 131072 fp32 34.8 and 36.6; 512 x 32317 21.6 and 24.1. Backward, 256 x 131072 bf16 takes 53 us with 256
// workgroups, 50.6 with 1024.
constexpr int64_t kMaskTokens = int64_t{1} << 18;
constexpr int64_t kFullRows = 192, kLongRow = 49152;
constexpr int64_t kChunk = 32768, kLeastChunk = 2048, kWantedGroups = 1024;

void cut_rows(const JabasLoss* l, bool forward, int64_t& splits, int64_t& chunk) {
    const int64_t rows = l->rows > 0 ? l->rows : 1, largest = forward ? kMaskTokens : kChunk;
    splits = tiles(l->vocab, largest);
    if (!forward || (rows < kFullRows && l->vocab >= kLongRow)) {
        const int64_t want = tiles(kWantedGroups, rows), most = tiles(l->vocab, kLeastChunk);
        const int64_t more = want < most ? want : most;
        if (splits < more) splits = more;
    }
    chunk = round_up(tiles(l->vocab, splits), 32);
    splits = tiles(l->vocab, chunk);
}

size_t carve_forward(const JabasLoss* l, const Shape& s, char* base, Forward& f) {
    Carver c{base, 0};
    const int64_t rows = l->rows;
    f = Forward{};
    if (s.narrow) {
        f.tiles = narrow_tiles(l->vocab);
        f.ticket = c.take<uint32_t>(1);
    } else if (s.linear) {
        f.piece = piece_tokens(l, s, false);
        f.large = large_tiles(f.piece < l->vocab ? f.piece : l->vocab, rows, s.planes, false);
        f.tiles = tiles(l->vocab, logits_tile(f.large));
    } else {
        cut_rows(l, true, f.splits, f.chunk);
        f.tiles = f.splits;
        f.ticket = c.take<uint32_t>(1);
    }
    f.partial = c.take<float2>(f.tiles * rows);
    if (l->label_smoothing != 0.0) f.total = c.take<float>(f.tiles * rows);
    if (s.linear) f.entry_logit = c.take<float>(rows * (s.teacher ? l->entries : 1));
    if (s.linear && s.teacher) f.teacher_row = c.take<float4>(rows);
    f.row_loss = c.take<float>(s.narrow || f.splits > 1 ? 2 * rows : rows);
    if (s.narrow) return c.all();
    if (s.linear) {
        f.map = c.take<int32_t>(rows);
        f.live = c.take<int32_t>(1);
        f.ticket = c.take<uint32_t>(1);
    }
    if (s.linear) f.x = c.take<uint16_t>(rows * s.depth * s.planes);
    if (s.linear && s.copy_w) f.w = c.take<uint16_t>(f.piece * s.depth * s.planes);
    if (s.linear && s.planes == 2) {
        f.unscale_x = c.take<float>(rows);
        f.unscale_w = c.take<float>(f.piece);
    }
    return c.all();
}

struct Backward {
    float *grad, *ratio, *peak, *down;
    uint16_t *x, *w;            // operands of the logits; w where it is a copy
    uint16_t *x16, *w16, *dz;   // of the gradients' products
    int32_t *map, *live;
    float *unscale_x, *unscale_w, *unscale_x16, *unscale_w16, *parts;
    float* peaks;               // of the columns of x16
    uint32_t* named;
    float *db, *part_w, *part_h;
    int64_t piece, pad_rows, part_stride, splits, chunk;
    Splits inner;
    bool large;
    float* narrow_dz;
    NarrowSplits narrow;
};

size_t carve_backward(const JabasLoss* l, const Shape& s, char* base, Backward& b) {
    Carver c{base, 0};
    const int64_t rows = l->rows;
    b = Backward{};
    if (!s.linear) {
        cut_rows(l, false, b.splits, b.chunk);
        return c.all();
    }
    if (s.narrow) {
        b.piece = l->vocab < kNarrowPiece ? l->vocab : kNarrowPiece;
        b.narrow = narrow_splits(b.piece, l->width);
        b.narrow_dz = c.take<float>((rows <= 32 ? 32 : 64) * narrow_tiles(b.piece) * 32 * (s.planes == 1 ? 2 : 1));
        b.part_stride = round_up(l->width, 4);
        if (b.narrow.n > 1 || b.piece < l->vocab) b.part_h = c.take<float>(b.narrow.n * rows * b.part_stride);
        return c.all();
    }
    b.grad = c.take<float>(rows);
    b.ratio = c.take<float>(rows);
    b.peak = c.take<float>(1);
    if (s.teacher) b.down = c.take<float>(rows);
    b.map = c.take<int32_t>(rows);
    b.live = c.take<int32_t>(1);
    b.piece = piece_tokens(l, s, true);
    b.pad_rows = round_up(rows, kDepth);
    b.x = c.take<uint16_t>(rows * s.depth * s.planes);
    if (s.copy_w) b.w = c.take<uint16_t>(b.piece * s.depth * s.planes);
    b.unscale_x = c.take<float>(rows);
    b.unscale_w = c.take<float>(b.piece);
    b.part_stride = round_up(l->width, 4);
    b.peaks = c.take<float>(kPeakParts * b.part_stride);
    if (l->bias) b.named = c.take<uint32_t>(tiles(l->vocab, 32));
    b.unscale_x16 = c.take<float>(b.part_stride);
    b.unscale_w16 = c.take<float>(1);
    b.parts = c.take<float>(kMaxParts);
    b.x16 = c.take<uint16_t>(l->width * b.pad_rows * s.planes);
    if (s.planes == 1) b.w16 = c.take<uint16_t>(l->width * b.piece);
    b.dz = c.take<uint16_t>(b.pad_rows * b.piece * s.planes);
    const int64_t tokens = b.piece < l->vocab ? b.piece : l->vocab;
    b.inner = choose_splits(l->width, tokens, rows, true, true, b.piece < l->vocab, s.planes);
    if (b.inner.w > 1) b.part_w = c.take<float>(b.inner.w * tokens * b.part_stride);
    if (b.inner.h > 1 || b.piece < l->vocab) b.part_h = c.take<float>(b.inner.h * rows * b.part_stride);
    b.large = large_tiles(tokens, rows, s.planes, true);
    if (l->bias) b.db = c.take<float>(tiles(rows, logits_tile(b.large)) * b.piece);
    return c.all();
}

Entries entries_of(const JabasLoss* l, const Shape& s) {
    Entries e{};
    e.target = l->target;
    e.ignore_index = l->ignore_index;
    if (s.teacher) {
        e.index = l->entry_index;
        e.p = l->entry_p;
        e.k = static_cast<int32_t>(l->entries);
    }
    return e;
}

constexpr double kLog2e = 1.4426950408889634;

NarrowArgs narrow_args(const JabasLoss* l, const Entries& entries, float c) {
    NarrowArgs a{};
    a.x = l->hidden;
    a.w = l->weight;
    a.bias = l->bias;
    a.x_stride = l->hidden_stride;
    a.w_stride = l->weight_stride;
    a.vocab = l->vocab;
    a.rows = static_cast<int32_t>(l->rows);
    a.width = static_cast<int32_t>(l->width);
    a.c = c;
    a.entries = entries;
    return a;
}

const char* at(const void* p, int64_t elements, int dtype) {
    return static_cast<const char*>(p) + elements * static_cast<int64_t>(element_bytes(dtype));
}

#define JABAS_TRY(call)                        \
    do {                                       \
        const int status_ = (call);            \
        if (status_ != JABAS_OK) return status_; \
    } while (0)

// The hidden states of the rows that count; the other rows of `zero` become zeros, and the tokens the rows name are marked in `name`.
int lay_x(const JabasLoss* l, const Shape& s, const Live& live, void* zero, uint32_t* name, uint16_t* x, float* unscale, Operand& out, hipStream_t stream) {
    out.rows = static_cast<int32_t>(l->rows);
    LayArgs a{};
    a.live = live;
    a.zero = zero;
    a.name = name;
    a.entries = entries_of(l, s);
    a.vocab = l->vocab;
    a.in = l->hidden;
    a.in_stride = l->hidden_stride;
    a.in_dtype = l->dtype;
    a.rows = static_cast<int32_t>(l->rows);
    a.cols = static_cast<int32_t>(l->width);
    a.out = x;
    a.out_stride = s.depth;
    a.out_plane = l->rows * s.depth;
    a.pad = static_cast<int32_t>(s.depth);
    a.planes = s.planes == 2 ? 2 : 0;
    a.low = 1.0f;
    a.unscale = unscale;
    out.p = x;
    out.stride = a.out_stride;
    out.plane = a.out_plane;
    return launch_lay_rows(a, stream);
}

// The weight's rows of a piece. `parts`: two planes with one scale for all, fit for a product that sums over the tokens too: those that the
// bias rules out are zeros (those that are `named` are not), and as many more as make whole steps.
int lay_w(const JabasLoss* l, const Shape& s, int64_t first, int64_t n, int64_t piece, uint16_t* w, float* unscale, float* parts, float* unscale_all,
          const uint32_t* named, Operand& out, hipStream_t stream) {
    out.rows = static_cast<int32_t>(n);
    if (!s.copy_w) {
        out.p = at(l->weight, first * l->weight_stride, l->dtype);
        out.stride = l->weight_stride;
        out.plane = 0;
        return JABAS_OK;
    }
    LayArgs a{};
    a.in = at(l->weight, first * l->weight_stride, l->dtype);
    a.in_stride = l->weight_stride;
    a.in_dtype = l->dtype;
    a.rows = static_cast<int32_t>(n);
    a.cols = static_cast<int32_t>(l->width);
    a.out = w;
    a.out_stride = s.depth;
    a.out_plane = piece * s.depth;
    a.pad = static_cast<int32_t>(s.depth);
    a.planes = s.planes == 2 ? 2 : 0;
    a.low = kLowScale;
    a.unscale = unscale;
    if (parts) {
        a.parts = parts;
        a.unscale_all = unscale_all;
        a.row_mask = named ? at(l->bias, first, l->dtype) : nullptr;
        a.named = named;
        a.first = static_cast<int32_t>(first);
        a.pad_rows = static_cast<int32_t>(round_up(n, kDepth));
    }
    out.p = w;
    out.stride = a.out_stride;
    out.plane = a.out_plane;
    return launch_lay_rows(a, stream);
}

}  // namespace
}  // namespace loss
}  // namespace jabas

using namespace jabas;
using namespace jabas::loss;

JABAS_API size_t jabas_loss_workspace_bytes(const JabasLoss* l, int32_t backward) {
    Shape s;
    if (validate(l, s) != JABAS_OK) return 0;
    Forward f;
    Backward b;
    return backward ? carve_backward(l, s, nullptr, b) : carve_forward(l, s, nullptr, f);
}

JABAS_API int jabas_loss_forward(const JabasLoss* l, float* loss_out, void* workspace, size_t workspace_bytes, jabas_stream_t stream_) {
    Shape s;
    JABAS_TRY(validate(l, s));
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    if (!loss_out && (l->rows || l->reduction != JABAS_LOSS_NONE)) return JABAS_ERR_NULL;
    Forward f;
    if (!workspace || misaligned(workspace, 256) || workspace_bytes < carve_forward(l, s, static_cast<char*>(workspace), f)) return JABAS_ERR_WORKSPACE;
    RowState* state = reinterpret_cast<RowState*>(l->row_state);
    float* reduce = l->row_state + 4 * l->rows;
    if (s.linear && !s.narrow && l->reduction == JABAS_LOSS_NONE) f.row_loss = loss_out;
    if (!l->rows) return launch_reduce(f.row_loss, state, 0, l->reduction, loss_out, reduce, stream);
    const float inv_t = static_cast<float>(1.0 / l->temperature), c = static_cast<float>(kLog2e / l->temperature);
    const Entries entries = entries_of(l, s);
    TeacherArgs t{};
    if (s.teacher) {
        t.index = l->teacher_index;
        t.logits = l->teacher_logits;
        t.dtype = l->dtype;
        t.lse = l->teacher_lse;
        t.rows = l->rows;
        t.vocab = l->vocab;
        t.k = static_cast<int32_t>(l->entries);
        t.inv_t = inv_t;
        t.t = static_cast<float>(l->temperature);
        t.entry_index = l->entry_index;
        t.entry_p = l->entry_p;
        t.row = f.teacher_row;
        if (s.linear) JABAS_TRY(launch_teacher(t, stream));
    }
    if (s.narrow) {
        NarrowArgs a = narrow_args(l, entries, c);
        a.partial = f.partial;
        a.total = f.total;
        a.entry_logit = f.entry_logit;
        a.ticket = f.ticket;
        JABAS_TRY(launch_narrow_forward(a, l->dtype, stream));
    } else if (s.linear) {
        LogitsArgs a{};
        LiveArgs live{};
        live.target = l->target;
        live.ignore_index = l->ignore_index;
        live.teacher_row = f.teacher_row;
        live.rows = l->rows;
        live.map = f.map;
        live.live = f.live;
        live.ticket = f.ticket;
        live.state = state;
        live.row_loss = f.row_loss;
        JABAS_TRY(launch_live(live, stream));
        a.rows = Live{f.map, f.live};
        JABAS_TRY(lay_x(l, s, a.rows, nullptr, nullptr, f.x, f.unscale_x, a.x, stream));
        a.depth = static_cast<int32_t>(s.depth);
        a.unscale_x = f.unscale_x;
        a.unscale_w = f.unscale_w;
        a.bias = l->bias;
        a.bias_dtype = l->dtype;
        a.c = c;
        a.entries = entries;
        a.partial = f.partial;
        a.total = f.total;
        a.entry_logit = f.entry_logit;
        for (int64_t first = 0; first < l->vocab; first += f.piece) {
            const int64_t n = l->vocab - first < f.piece ? l->vocab - first : f.piece;
            JABAS_TRY(lay_w(l, s, first, n, f.piece, f.w, f.unscale_w, nullptr, nullptr, nullptr, a.w, stream));
            a.first = static_cast<int32_t>(first);
            JABAS_TRY(launch_logits_forward(a, s.planes, f.large, stream));
        }
    } else {
        TopkArgs a{};
        a.logits = l->logits;
        a.stride = l->logits_stride;
        a.dtype = l->dtype;
        a.rows = l->rows;
        a.vocab = l->vocab;
        a.splits = static_cast<int32_t>(f.splits);
        a.chunk = f.chunk;
        a.c = c;
        a.teacher = t;
        a.partial = f.partial;
        a.state = state;
        a.row_loss = f.row_loss;
        a.ticket = f.ticket;
        a.reduction = l->reduction;
        a.loss_out = loss_out;
        a.reduce_out = reduce;
        return launch_topk_forward(a, stream);
    }
    JoinArgs j{};
    j.live = Live{f.map, f.live};
    j.partial = f.partial;
    j.total = f.total;
    j.entry_logit = f.entry_logit;
    j.rows = l->rows;
    j.vocab = l->vocab;
    j.tiles = static_cast<int32_t>(f.tiles);
    j.c = c;
    j.smoothing = static_cast<float>(l->label_smoothing);
    j.entries = entries;
    j.teacher_row = f.teacher_row;
    j.teacher = t;
    j.state = state;
    j.row_loss = f.row_loss;
    j.ticket = f.ticket;
    j.reduction = l->reduction;
    j.loss_out = loss_out;
    j.reduce = reduce;
    return s.narrow ? launch_narrow_join(j, stream) : launch_join(j, stream);
}

JABAS_API int jabas_loss_backward(const JabasLoss* l, const float* upstream, void* d_hidden, void* d_weight, void* d_bias, void* d_logits,
                                  void* workspace, size_t workspace_bytes, jabas_stream_t stream_) {
    Shape s;
    JABAS_TRY(validate(l, s));
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    if (!upstream && (l->rows || l->reduction != JABAS_LOSS_NONE)) return JABAS_ERR_NULL;
    if (s.linear ? d_logits != nullptr : d_hidden || d_weight || d_bias) return JABAS_ERR_NULL;
    if (d_bias && !l->bias) return JABAS_ERR_NULL;
    const size_t bytes = element_bytes(l->dtype);
    if (misaligned(d_hidden, bytes) || misaligned(d_weight, bytes) || misaligned(d_bias, bytes) || misaligned(d_logits, bytes) || misaligned(upstream, 4))
        return JABAS_ERR_ALIGN;
    Backward b;
    if (!workspace || misaligned(workspace, 256) || workspace_bytes < carve_backward(l, s, static_cast<char*>(workspace), b)) return JABAS_ERR_WORKSPACE;
    if (!l->rows) {
        if (d_weight) JABAS_TRY(launch_zero(d_weight, static_cast<size_t>(l->vocab) * l->width * bytes, stream));
        if (d_bias) JABAS_TRY(launch_zero(d_bias, static_cast<size_t>(l->vocab) * bytes, stream));
        return JABAS_OK;
    }
    const RowState* state = reinterpret_cast<const RowState*>(l->row_state);
    const float* reduce = l->row_state + 4 * l->rows;
    const float c = static_cast<float>(kLog2e / l->temperature);
    const int per_row = l->reduction == JABAS_LOSS_NONE;
    if (!s.linear) {
        if (!d_logits) return JABAS_OK;
        TopkArgs a{};
        a.logits = l->logits;
        a.stride = l->logits_stride;
        a.dtype = l->dtype;
        a.rows = l->rows;
        a.vocab = l->vocab;
        a.splits = static_cast<int32_t>(b.splits);
        a.chunk = b.chunk;
        a.c = c;
        a.entries = entries_of(l, s);
        a.t = static_cast<float>(l->temperature);
        a.state = const_cast<RowState*>(state);
        a.upstream = upstream;
        a.per_row = per_row;
        a.reduce = reduce;
        a.out = d_logits;
        return launch_topk_backward(a, stream);
    }
    if (!d_hidden && !d_weight && !d_bias) return JABAS_OK;
    const float uniform = static_cast<float>(l->label_smoothing / static_cast<double>(l->vocab)), hit = static_cast<float>(1.0 - l->label_smoothing);
    if (s.narrow) {
        NarrowArgs a = narrow_args(l, entries_of(l, s), c);
        a.state = state;
        a.upstream = upstream;
        a.per_row = per_row;
        a.reduce = reduce;
        a.t = static_cast<float>(l->temperature);
        a.uniform = uniform;
        a.hit = hit;
        a.dz = d_hidden || d_weight ? b.narrow_dz : nullptr;
        a.dz_stride = narrow_tiles(b.piece) * 32;
        a.d_bias = d_bias;
        a.d_weight = d_weight;
        a.d_hidden = d_hidden;
        a.each = b.narrow.each;
        a.part = b.part_h;
        a.part_stride = b.part_stride;
        a.part_plane = l->rows * b.part_stride;
        for (a.first = 0; a.first < l->vocab; a.first += b.piece) {
            a.tokens = l->vocab - a.first < b.piece ? l->vocab - a.first : b.piece;
            a.hidden_units = d_hidden ? tiles(l->width, 128) * tiles(a.tokens, a.each) : 0;
            a.add = a.first > 0;        // a shorter last piece adds to the first of the splits
            JABAS_TRY(launch_narrow_backward(a, l->dtype, stream));
            if (a.dz) JABAS_TRY(launch_narrow_grads(a, l->dtype, stream));
        }
        if (!d_hidden || !a.part) return JABAS_OK;
        Job j{};
        j.m = a.width;
        j.n = a.rows;
        j.splits = b.narrow.n;
        j.part = a.part;
        j.part_stride = a.part_stride;
        j.part_plane = a.part_plane;
        j.out = d_hidden;
        j.out_stride = l->width;
        j.out_dtype = l->dtype;
        j.out_aligned = l->width % 4 == 0 && !misaligned(d_hidden, 4 * bytes);
        return launch_join_splits(j, stream);
    }
    RowGradArgs r{};
    r.upstream = upstream;
    r.per_row = per_row;
    r.reduce = reduce;
    r.down = b.down;
    r.t = static_cast<float>(l->temperature);
    r.state = state;
    r.rows = l->rows;
    r.grad = b.grad;
    r.ratio = b.ratio;
    r.peak = b.peak;
    r.map = b.map;
    r.live = b.live;
    // Tokens that the bias rules out may hold any weight: dz is 0 there, but at a label or an entry, and everywhere under label smoothing.
    uint32_t* named = l->bias && d_hidden && l->label_smoothing == 0.0 ? b.named : nullptr;
    r.zero = named;
    r.zeros = tiles(l->vocab, 32);
    if (s.teacher) JABAS_TRY(launch_down(l->entry_p, l->rows, static_cast<int32_t>(l->entries), b.down, stream));
    JABAS_TRY(launch_row_grad(r, stream));
    const Live live = {b.map, b.live};
    LogitsArgs a{};
    a.rows = live;
    JABAS_TRY(lay_x(l, s, live, d_hidden, named, b.x, b.unscale_x, a.x, stream));
    a.depth = static_cast<int32_t>(s.depth);
    a.unscale_x = b.unscale_x;
    a.unscale_w = b.unscale_w;
    a.bias = l->bias;
    a.bias_dtype = l->dtype;
    a.c = c;
    a.entries = entries_of(l, s);
    a.state = state;
    a.row_grad = b.grad;
    a.down = b.down;
    a.uniform = uniform;
    a.hit = hit;
    a.dz = d_hidden || d_weight ? b.dz : nullptr;
    a.dz_stride = b.piece;
    a.dz_plane = b.pad_rows * b.piece;
    a.db = d_bias ? b.db : nullptr;
    LayArgs lay{};
    lay.in_dtype = l->dtype;
    lay.cols = static_cast<int32_t>(l->width);
    lay.planes = s.planes;
    lay.low = 1.0f;
    lay.parts = b.parts;
    if (d_weight) {
        lay.peaks = b.peaks;        // a feature of large values, or a row of a large gradient, takes no bits from the other features
        lay.peak_stride = b.part_stride;
        lay.in = l->hidden;
        lay.in_stride = l->hidden_stride;
        lay.rows = static_cast<int32_t>(l->rows);
        lay.live = live;
        lay.row_factor = b.ratio;
        lay.out = b.x16;
        lay.out_stride = b.pad_rows;
        lay.out_plane = l->width * b.pad_rows;
        lay.pad = static_cast<int32_t>(b.pad_rows);
        lay.unscale = b.unscale_x16;
        JABAS_TRY(launch_lay_columns(lay, stream));
    }
    lay.peaks = nullptr;
    lay.live = Live{};
    lay.row_factor = nullptr;
    lay.in_stride = l->weight_stride;
    lay.out = b.w16;
    lay.out_stride = b.piece;
    lay.out_plane = l->width * b.piece;
    lay.unscale = b.unscale_w16;
    const int32_t width = static_cast<int32_t>(l->width), rows = static_cast<int32_t>(l->rows);
    const auto each = [](int64_t depth, int splits) { return static_cast<int32_t>(round_up((depth + splits - 1) / splits, kDepth)); };
    const auto splits = [](int64_t depth, int64_t each) { return static_cast<int32_t>((depth + each - 1) / each); };
    GradArgs g{};
    const int64_t whole = round_up(l->vocab < b.piece ? l->vocab : b.piece, kDepth);        // the first piece, the largest
    g.h.each = each(whole, b.inner.h);
    const int32_t splits_h = splits(whole, g.h.each);
    g.w.scale = g.h.scale = 1.0f / kDzScale;
    g.w.out_stride = g.h.out_stride = l->width;
    g.w.out_dtype = g.h.out_dtype = l->dtype;
    g.w.part_stride = g.h.part_stride = b.part_stride;
    g.w.splits = g.h.splits = 1;
    g.w.rows = g.h.rows = live;
    g.w.live_depth = g.h.live_n = 1;
    for (int64_t first = 0; first < l->vocab; first += b.piece) {
        const int64_t n = l->vocab - first < b.piece ? l->vocab - first : b.piece;
        const int32_t pad = static_cast<int32_t>(round_up(n, kDepth));
        JABAS_TRY(lay_w(l, s, first, n, b.piece, b.w, b.unscale_w, s.planes == 2 && d_hidden ? b.parts : nullptr, b.unscale_w16, named, a.w, stream));
        a.first = static_cast<int32_t>(first);
        a.pad_tokens = pad;
        JABAS_TRY(launch_logits_backward(a, s.planes, b.large, stream));
        if (d_bias) JABAS_TRY(launch_bias_sum(b.db, b.live, logits_tile(b.large), n, n, static_cast<char*>(d_bias) + first * bytes, l->dtype, stream));
        if (!d_weight && !d_hidden) continue;
        if (d_weight) {     // sum over the rows of dz[row][token] x[row][feature]
            g.w.a = Operand{b.x16, b.pad_rows, l->width * b.pad_rows, width};
            g.w.b = Operand{b.dz, a.dz_stride, a.dz_plane, pad};
            g.w.m = width;
            g.w.n = static_cast<int32_t>(n);
            g.w.depth = static_cast<int32_t>(b.pad_rows);
            g.w.each = each(b.pad_rows, b.inner.w);
            g.w.splits = splits(b.pad_rows, g.w.each);
            g.w.unscale_m = b.unscale_x16;
            g.w.unscale1 = b.peak;
            g.w.part = g.w.splits > 1 ? b.part_w : nullptr;
            g.w.part_plane = n * b.part_stride;
            g.w.first = g.w.keep = 1;
            g.w.out = static_cast<char*>(d_weight) + first * l->width * static_cast<int64_t>(bytes);
            g.w.out_aligned = width % 4 == 0 && !misaligned(g.w.out, 4 * bytes);
        }
        if (d_hidden) {     // sum over the tokens of dz[row][token] w[token][feature]
            if (s.planes == 1) {
                lay.in = at(l->weight, first * l->weight_stride, l->dtype);
                lay.rows = static_cast<int32_t>(n);
                lay.row_mask = named ? at(l->bias, first, l->dtype) : nullptr;
                lay.named = named;
                lay.first = static_cast<int32_t>(first);
                lay.pad = pad;
                JABAS_TRY(launch_lay_columns(lay, stream));
                g.h.a = Operand{b.w16, b.piece, 0, width};
            } else {            // as it lies for the logits
                g.h.a = Operand{a.w.p, a.w.stride, a.w.plane, static_cast<int32_t>(s.depth)};
            }
            g.h.b = Operand{b.dz, a.dz_stride, a.dz_plane, rows};
            g.h.m = width;
            g.h.n = rows;
            g.h.depth = pad;
            g.h.splits = splits(pad, g.h.each);     // a shorter last piece adds to the first of them
            g.h.unscale0 = b.unscale_w16;
            g.h.row_scale = b.grad;
            g.h.part = b.part_h;
            g.h.part_plane = l->rows * b.part_stride;
            g.h.first = first == 0;
            g.h.keep = splits_h > 1 || first + b.piece < l->vocab;
            g.h.out = d_hidden;
            g.h.out_aligned = width % 4 == 0 && !misaligned(d_hidden, 4 * bytes);
        }
        JABAS_TRY(launch_grads(g, s.planes, stream));
        if (g.w.splits > 1) JABAS_TRY(launch_join_splits(g.w, stream));
    }
    if (!d_hidden || splits_h == 1) return JABAS_OK;
    g.h.splits = splits_h;
    return launch_join_splits(g.h, stream);
}
