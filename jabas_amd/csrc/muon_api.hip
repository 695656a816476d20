// Entry points of the orthogonalised update: argument validation, plans, workspace layout, and the order of the launches.
#include <math.h>
#include <string.h>

#include <algorithm>
#include <map>
#include <new>
#include <numeric>
#include <vector>

#include "muon_internal.h"

#define JABAS_API extern "C" __attribute__((visibility("default")))

namespace jabas {
namespace muon {
namespace {

inline int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
inline bool misaligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }
constexpr int64_t kMaxSlots = int64_t{1} << 23;     // a launch has less than 2^32 threads, up to 512 a workgroup

// What the products' factors are multiplied by, powers of two: no entry of a matrix is larger than its largest singular value, and how far
// the polynomial lets those grow is known. The bound goes to between 2^13 and 2^14, and fp16's finest step, 2^-24, is 2^-37 of it or finer.
struct Scales {
    double x[JABAS_MUON_MAX_STEPS + 1], a[JABAS_MUON_MAX_STEPS], b[JABAS_MUON_MAX_STEPS];
};
double scale_for(double most) {
    if (!(most > 0.0)) return 16384.0;
    return ldexp(1.0, std::min(40, 14 - static_cast<int>(ceil(log2(most)))));
}
int scales_of(const JabasNewtonSchulz& ns, Scales& s) {
    if (ns.precision != JABAS_F32 && ns.precision != JABAS_BF16) return JABAS_ERR_DTYPE;
    if (ns.steps < 1 || ns.steps > JABAS_MUON_MAX_STEPS || !isfinite(ns.a) || !isfinite(ns.b) || !isfinite(ns.c)) return JABAS_ERR_OPT;
    if (!(ns.eps >= 1e-30) || !isfinite(ns.eps)) return JABAS_ERR_OPT;
    double most = 1.0;          // the largest singular value is at most the length, one
    for (int k = 0; k < ns.steps; ++k) {
        const double end = most * most;
        const auto second = [&](double t) { return fabs(ns.b * t + ns.c * t * t); };
        const auto value = [&](double t) { return sqrt(t) * fabs(ns.a + ns.b * t + ns.c * t * t); };
        double b = second(end), next = value(end);
        if (ns.c != 0.0) {
            const double t = -ns.b / (2.0 * ns.c), root = 9.0 * ns.b * ns.b - 20.0 * ns.a * ns.c;
            if (t > 0.0 && t < end) b = std::max(b, second(t));
            if (root >= 0.0)
                for (double sign : {-1.0, 1.0}) {
                    const double at = (-3.0 * ns.b + sign * sqrt(root)) / (10.0 * ns.c);
                    if (at > 0.0 && at < end) next = std::max(next, value(at));
                }
        } else if (ns.b != 0.0) {
            const double at = -ns.a / (3.0 * ns.b);
            if (at > 0.0 && at < end) next = std::max(next, value(at));
        }
        if (!(next <= 256.0) || !(b <= 65536.0)) return JABAS_ERR_OPT;
        s.x[k] = scale_for(most);
        s.a[k] = scale_for(end);
        s.b[k] = scale_for(b);
        most = std::max(next, 1e-6);
    }
    s.x[ns.steps] = 1.0;
    return JABAS_OK;
}

bool shape_fits(int64_t rows, int64_t cols) {
    return std::min(rows, cols) <= JABAS_MUON_MAX_SIDE && std::max(rows, cols) <= JABAS_MUON_MAX_LENGTH;
}

// Sides, padding and partial sums; places come from whoever lays the workspace out.
void describe(Matrix& x, int64_t rows, int64_t cols) {
    x.rows = static_cast<int32_t>(rows);
    x.cols = static_cast<int32_t>(cols);
    x.tall = rows > cols;
    x.m = x.tall ? x.cols : x.rows;
    x.n = x.tall ? x.rows : x.cols;
    x.pad_m = static_cast<int32_t>(round_up(x.m, kPad));
    x.pad_n = static_cast<int32_t>(round_up(x.n, kPad));
    x.x_plane = static_cast<int64_t>(x.pad_m) * x.pad_n;
    x.a_plane = static_cast<int64_t>(x.pad_m) * x.pad_m;
    const int64_t count = rows * cols, chunk = std::max<int64_t>(kMinChunk, round_up((count + kParts - 1) / kParts, 1024));
    x.chunk = static_cast<int32_t>(chunk);
    x.parts = static_cast<int32_t>((count + chunk - 1) / chunk);
}
// Behind them, of any call: tiles' sums of launches that share tiles between workgroups, and the tiles' tickets.
constexpr int64_t kSplitUnits = 512;        // workgroups of a launch that shares tiles, at most
constexpr int64_t kShareBytes = kSplitUnits * (4096 + 1) * 4;
// halves of the workspace: X twice in two planes, A and B in as many as the products take
int64_t halves_of(const Matrix& x, int planes) { return 4 * x.x_plane + 2 * planes * x.a_plane; }
int64_t lay_tiles(const Matrix& x) { return static_cast<int64_t>(x.pad_m / kLay) * (x.pad_n / kLay); }

// Which kernel a product of some matrices takes: the one that ends first by what was measured. `each` workgroups of a kernel share a CU; a tile takes `start`
// us and, for 64 of the inner axis, `first` us in X X^T and A A or `update` us in a X + B X with the chip full, `alone` with most CUs idle. Measured, us,
// X X^T and then a X + B X, for kSmall, kSmallMany, kMiddle, kMiddleDeep, kLarge (fp32; bf16 next):
//   12 x  768 x  768   31 32 32 25 54    53 53 44 44 61     18 18 20 18 29    32 28 25 30 31
//    6 x 1024 x 4096  105 109 110 84 233  203 180 151 168 170   52 52 49 39 84   114 96 75 94 80
//        1024 x 4096   32 58 92 60 217    37 36 35 30 71     18 33 43 29 79    23 20 20 18 32
//    3 x 2048 x 2048  112 98 89 87 132   206 183 147 148 151   54 49 37 44 52    91 87 68 73 61
//        4096 x 4096  329 298 246 240 250  508 471 360 365 327  163 133 108 109 93   249 222 145 159 127
//   64 x  129 x  257    9 10 13 11 23     14 13 16 19 25      7 7 9 8 12      13 10 12 16 17
//    4 x  384 x  384    8 10 14 13 31      8 9 15 13 32       6 7 11 11 19     7 7 11 10 19
struct Cost {
    int each;
    double start, alone, symmetric, update;
};
constexpr Cost kCosts[2][kKernels] = {
    {{2, 2.5, 0.20, 0.38, 0.46}, {4, 4.0, 0.50, 0.75, 0.75}, {2, 7.0, 0.62, 0.90, 1.00}, {1, 5.0, 0.38, 0.53, 0.60}, {1, 13.0, 1.25, 1.75, 1.75}},
    {{2, 3.5, 0.45, 0.76, 0.95}, {4, 4.5, 0.90, 1.60, 1.60}, {2, 8.0, 1.35, 2.60, 2.65}, {1, 6.0, 0.95, 1.15, 1.35}, {1, 18.0, 3.40, 4.75, 4.75}}};
constexpr int64_t kCus = 256, kFew = 160;
// Tiles of 64 of a symmetric product, which read every row most often, wait for memory where a matrix has more than kNear bytes: 4096 x 4096 above takes 1.25
// (fp32) and 1.18 times (bf16) what the steps of 6 of 1024 x 4096 make it, two of 2048 x 4096 with two of 1024 x 4096 200 us for 160.
constexpr double kNear = 16 << 20, kFar = 1.25;
constexpr double kLaunch = 4.0, kJoin = 4.0;    // us of a launch, beside its tiles, and of tiles' parts that meet

enum Product { kFirst, kSecond, kUpdate, kProducts };
struct Shape {
    int32_t m, n, pad_m, pad_n;
    int64_t count;
    Shape(const Matrix& x, int64_t count) : m(x.m), n(x.n), pad_m(x.pad_m), pad_n(x.pad_n), count(count) {}
    int64_t tiles(Product p, Kind k) const { return p == kUpdate ? update_tiles(m, n, kTile[k]) : symmetric_tiles(m, kTile[k]); }
    double steps(Product p) const { return (p == kFirst ? pad_n : pad_m) / 64.0; }
};

// When `slots` workgroups are done with tiles of given lengths, longest first, each taken by whoever is free first.
struct Tiles {
    double length;
    int64_t count;
};
double makespan(std::vector<Tiles> work, int64_t slots) {
    std::sort(work.begin(), work.end(), [](const Tiles& a, const Tiles& b) { return a.length > b.length; });
    std::map<double, int64_t> free_at{{0.0, slots}};
    double end = 0.0;
    for (Tiles& w : work)
        while (w.count > 0) {
            const auto next = free_at.begin();
            if (free_at.size() == 1 && w.count >= 4 * slots) {         // whole rounds
                const int64_t rounds = w.count / slots - 1;
                const double until = next->first + rounds * w.length;
                w.count -= rounds * slots;
                free_at = {{until, slots}};
                end = std::max(end, until);
                continue;
            }
            const int64_t take = std::min(w.count, next->second);
            const double until = next->first + w.length;
            w.count -= take;
            end = std::max(end, until);
            if ((next->second -= take) == 0) free_at.erase(next);
            free_at[until] += take;
        }
    return end;
}

// Workgroups that share a tile's inner axis, where a launch (of `total` tiles) leaves CUs room for more and the axis is long: the parts meet through memory, which
// takes 4 us with few of them and 6 with many. Without and with it, us of a call: 256 x 4096 fp32 241 and 149, four of 64 x 4096 222 and 121, a step of 21
// convolutions' matrices (43 tiles) 159 and 148, of one of 4096 x 1024 (136 tiles, three workgroups each) 388 and 353, 1024 x 4096 bf16 230 and 222; but
// with two workgroups a tile 768 x 768 fp32 168 and 175, 1000 x 2048 bf16 180 and 189.
constexpr int64_t kMostSplits = 8;
int splits_of(const Shape& s, Product p, Kind k, int64_t total, int planes) {
    if (p != kFirst || k != kSmall) return 1;       // A A has no long axis where there are few tiles
    const int64_t splits = std::min({kSplitUnits / std::max<int64_t>(total, 1), static_cast<int64_t>(s.steps(p)) / (planes == 2 ? 6 : 12), kMostSplits});
    return splits >= 3 ? static_cast<int>(splits) : 1;
}

double time_of(const Shape* shapes, size_t n, Product p, Kind k, int planes) {
    const Cost& c = kCosts[planes - 1][k];
    int64_t tiles = 0, units = 0;
    for (size_t i = 0; i < n; ++i) tiles += shapes[i].count * shapes[i].tiles(p, k);
    for (size_t i = 0; i < n; ++i) units += shapes[i].count * shapes[i].tiles(p, k) * splits_of(shapes[i], p, k, tiles, planes);
    const double step = units <= kFew ? c.alone : p == kUpdate ? c.update : c.symmetric;
    const auto work_of = [&](const Shape& s) {
        const int splits = splits_of(s, p, k, tiles, planes);
        const double far = k == kSmall && p != kUpdate && 2 * planes * 64 * s.steps(p) * s.pad_m > kNear ? kFar : 1.0;
        return Tiles{c.start + s.steps(p) / splits * step * far + (splits > 1 ? kJoin : 0.0), s.count * s.tiles(p, k) * splits};
    };
    if (n == 1) return kLaunch + (units + kCus * c.each - 1) / (kCus * c.each) * work_of(shapes[0]).length;
    std::vector<Tiles> work;
    for (size_t i = 0; i < n; ++i) work.push_back(work_of(shapes[i]));
    return kLaunch + makespan(work, kCus * c.each);
}
Kind kernel_of(const Shape* shapes, size_t n, Product p, int planes, double* time = nullptr) {
    int at = 0;
    double least = 0.0;
    for (int k = 0; k < kKernels; ++k) {
        const double here = time_of(shapes, n, p, static_cast<Kind>(k), planes);
        if (k == 0 || here < least) {
            least = here;
            at = k;
        }
    }
    if (time) *time += least;
    return static_cast<Kind>(at);
}
double step_of(const Shape* shapes, size_t n, int planes) {
    double time = 0.0;
    for (int p = 0; p < kProducts; ++p) kernel_of(shapes, n, static_cast<Product>(p), planes, &time);
    return time;
}

enum { kMomentum = kProducts, kLayOut, kKinds };        // launches of their own beside the products

// The launches of some matrices that share a workspace.
struct Run {
    Work work[kKinds];
    Kind kernel[kProducts];
    int tiny;                       // blocks of tiny_fits, or 0
    int planes, dtype, nesterov;
    float momentum, fresh;
    const float* grad_scale;
    float* shares;
};
int run(const Run& r, const JabasNewtonSchulz& ns, const Scales& s, UpdateArgs& last, hipStream_t stream) {
    PassArgs pass{r.work[kMomentum], r.dtype, r.nesterov, r.momentum, r.fresh, r.grad_scale, ns.eps, static_cast<float>(s.x[0]), r.planes,
                  r.shares ? reinterpret_cast<uint32_t*>(r.shares + kSplitUnits * 4096) : nullptr, r.shares ? static_cast<uint32_t>(kSplitUnits) : 0};
    TinyStep steps[JABAS_MUON_MAX_STEPS];
    for (int k = 0; k < ns.steps; ++k)
        steps[k] = {static_cast<float>(s.a[k] / s.x[k] / s.x[k]), static_cast<float>(ns.b * s.b[k] / s.a[k]), static_cast<float>(ns.c * s.b[k] / s.a[k] / s.a[k]),
                    static_cast<float>(ns.a * s.x[k + 1] / s.x[k]), static_cast<float>(s.x[k + 1] / s.b[k] / s.x[k])};
    if (r.tiny) {
        TinyArgs all{pass, last.out, ns.steps, {}};
        std::copy(steps, steps + ns.steps, all.step);
        return launch_tiny(all, r.tiny, stream);
    }
    int status = launch_momentum(pass, stream);
    if (status != JABAS_OK) return status;
    pass.w = r.work[kLayOut];
    if ((status = launch_lay(pass, stream)) != JABAS_OK) return status;
    for (int k = 0; k < ns.steps; ++k) {
        if ((status = launch_symmetric({r.work[kFirst], k & 1, 0.0f, steps[k].first, r.shares, pass.tickets}, false, r.planes, r.kernel[kFirst], stream)) != JABAS_OK) return status;
        if ((status = launch_symmetric({r.work[kSecond], k & 1, steps[k].second_own, steps[k].second, nullptr, nullptr}, true, r.planes, r.kernel[kSecond], stream)) != JABAS_OK) return status;
        last.w = r.work[kUpdate];
        last.from = k & 1;
        last.last = k + 1 == ns.steps;
        last.own = steps[k].update_own;
        last.product = steps[k].update;
        if ((status = launch_update(last, r.planes, r.kernel[kUpdate], stream)) != JABAS_OK) return status;
    }
    return JABAS_OK;
}

// ---- a batch of one shape

// Matrices that go through the workspace together take at most this, or are one. How many do is what ends first by the costs above: the last tiles of a launch
// leave CUs idle, and a launch has its own time.
constexpr int64_t kTogether = int64_t{500} << 20;
constexpr int64_t kTurns = 16;          // ways of cutting that are tried

// Whatever fits one workgroup's LDS goes through tiny_kernel. Measured, us a call in fp32 (bf16 within 10 %), there and with the launches of the larger ones'
// kernels, batches of 1, 256 and 2048: 16 x 16 14, 14, 87 and 66, 76, 192; 64 x 64 24, 26, 183 and 70, 87, 267; 32 x 1216 72, 91, 752 and 100, 256, 2191;
// 64 x 544 65, 86, 677 and 92, 187, 1265; 96 x 288 67, 81, 635 and 91, 272, 1840; 128 x 160 71, 88, 667 and 91, 226, 1496. A list pays for its largest
// matrix's blocks in every workgroup: one of 128 x 160 with 256 of 16 x 16 86 and 98, but with 512 of them 128 and 113, with 2048 371 and 205.
inline int blocks_of(const Matrix& x) { return (x.m + 31) / 32; }

struct Batch {
    Matrix x;
    int planes, tiny;
    int64_t at_once, sums_bytes, bytes;
};
int describe_batch(const JabasOrthogonalize* o, Batch& b, Scales& s) {
    if (!o) return JABAS_ERR_NULL;
    if (o->dtype != JABAS_F32 && o->dtype != JABAS_BF16) return JABAS_ERR_DTYPE;
    const int status = scales_of(o->ns, s);
    if (status != JABAS_OK) return status;
    if (o->batch < 0 || o->rows < 0 || o->cols < 0 || !shape_fits(o->rows, o->cols) || o->batch > (int64_t{1} << 31)) return JABAS_ERR_SIZE;
    b.planes = o->ns.precision == JABAS_F32 ? 2 : 1;
    b.bytes = 256;
    b.at_once = 0;
    if (!o->batch || !o->rows || !o->cols) return JABAS_OK;
    memset(&b.x, 0, sizeof b.x);
    describe(b.x, o->rows, o->cols);
    const int64_t size = o->dtype == JABAS_F32 ? 4 : 2;
    if (!o->in || !o->out) return JABAS_ERR_NULL;
    if (misaligned(o->in, size) || misaligned(o->out, size)) return JABAS_ERR_ALIGN;
    constexpr int64_t kMaxStride = int64_t{1} << 40;
    if (o->in_row_stride < o->cols || o->in_row_stride > kMaxStride || o->in_batch_stride < 0 || o->in_batch_stride > kMaxStride) return JABAS_ERR_SIZE;
    const char *in = static_cast<const char*>(o->in), *out = static_cast<const char*>(o->out);
    const int64_t in_bytes = size * ((o->batch - 1) * o->in_batch_stride + (o->rows - 1) * o->in_row_stride + o->cols), out_bytes = size * o->batch * o->rows * o->cols;
    if (in < out + out_bytes && out < in + in_bytes) return JABAS_ERR_ALIAS;
    b.x.src_stride = o->in_row_stride;
    const size_t quad = 4 * size;
    b.x.src_quads = !misaligned(o->in, quad) && o->in_row_stride % 4 == 0 && (o->batch == 1 || o->in_batch_stride % 4 == 0);
    b.x.out_quads = !misaligned(o->out, quad) && o->cols % 4 == 0;
    b.tiny = tiny_fits(blocks_of(b.x), b.x.n) ? blocks_of(b.x) : 0;
    if (b.tiny) {
        b.at_once = std::min(o->batch, kMaxSlots / 4);          // of 1024 threads
        return JABAS_OK;
    }
    const int64_t each = halves_of(b.x, b.planes);
    // launches count their workgroups in 32 bits
    const int64_t most = kMaxSlots / std::max({lay_tiles(b.x), static_cast<int64_t>(b.x.parts), update_tiles(b.x.m, b.x.n, 64), symmetric_tiles(b.x.m, 64)});
    if (most < 1) return JABAS_ERR_SIZE;
    b.at_once = std::min({o->batch, std::max<int64_t>(1, kTogether / (2 * each)), most});
    b.sums_bytes = round_up(8 * b.at_once * b.x.parts, 256);
    b.bytes = b.sums_bytes + round_up(2 * b.at_once * each, 256) + kShareBytes;
    const int64_t least = (o->batch + b.at_once - 1) / b.at_once;
    double best = 0.0;
    for (int64_t turns = least; o->batch > 1 && turns < least + kTurns && turns <= o->batch; ++turns) {
        const int64_t here = (o->batch + turns - 1) / turns;        // turns of one size: a short last one would leave CUs idle
        const int64_t whole = o->batch / here, rest = o->batch - whole * here;
        const Shape both[2] = {Shape(b.x, here), Shape(b.x, rest)};
        double time = whole * step_of(both, 1, b.planes);
        if (rest) time += step_of(both + 1, 1, b.planes);
        if (turns == least || time < best) {
            best = time;
            b.at_once = here;
        }
        if (here == 1) break;
    }
    return JABAS_OK;
}

// ---- lists

constexpr uint32_t kMagic = 0x4d4e5331, kMaxMatrices = 1u << 20;
struct Part {
    uint64_t slots_at[kKinds];
    uint32_t total[kKinds];
    int32_t kernel[kProducts];
    int32_t reserved;
};
struct Header {
    uint32_t magic, n, n_parts, n_groups;
    int32_t precision, tiny;
    uint64_t bytes, matrices_at, fanout_at, parts_at, sums_bytes, workspace;
};

struct Span {
    const char* p;
    int64_t bytes;
    bool written;
};

int check_matrix(const JabasMatrix& j) {
    if (!j.grad || !j.momentum || !j.param) return JABAS_ERR_NULL;
    if (j.rows < 1 || j.cols < 1 || !shape_fits(j.rows, j.cols)) return JABAS_ERR_SIZE;
    if (j.group >= JABAS_MAX_GROUPS) return JABAS_ERR_GROUP;
    if (j.n_fanout > JABAS_MAX_K - 1) return JABAS_ERR_K;
    if (!isfinite(j.lr_factor)) return JABAS_ERR_OPT;
    Span all[JABAS_MAX_K + 2];
    int n = 0;
    const int64_t bytes = 4 * j.rows * j.cols;
    all[n++] = {reinterpret_cast<const char*>(j.grad), bytes, false};
    all[n++] = {reinterpret_cast<const char*>(j.momentum), bytes, true};
    all[n++] = {reinterpret_cast<const char*>(j.param), bytes, true};
    for (uint32_t f = 0; f < j.n_fanout; ++f) {
        if (!j.fanout[f]) return JABAS_ERR_NULL;
        all[n++] = {reinterpret_cast<const char*>(j.fanout[f]), bytes, true};
    }
    for (int a = 0; a < n; ++a) {
        if (misaligned(all[a].p, 4)) return JABAS_ERR_ALIGN;
        for (int b = 0; b < a; ++b)
            if ((all[a].written || all[b].written) && all[a].p < all[b].p + bytes && all[b].p < all[a].p + bytes) return JABAS_ERR_ALIAS;
    }
    return JABAS_OK;
}

// Slots of one launch: every matrix's tiles are dealt out to the eight dies in runs, dies in turn where a matrix has fewer than eight, and die d has slots
// d, d + 8, ... . `work`: matrices and their tiles, the longest first.
struct Dealt {
    uint32_t matrix;
    int64_t tiles;                  // workgroups
    int32_t splits;
};
void deal(std::vector<Slot>& out, const std::vector<Dealt>& work, const std::vector<Matrix>& all) {
    std::vector<Slot> die[8];
    int turn = 0;
    int64_t total = 0;
    for (const Dealt& w : work) {
        const int64_t each = w.tiles / 8, left = w.tiles % 8;
        Slot s{w.matrix, 0, all[w.matrix].m, all[w.matrix].n, all[w.matrix].x_at, all[w.matrix].a_at, static_cast<uint32_t>(total), w.splits};
        for (int d = 0; d < 8; ++d) {
            const int64_t here = each + (d < left);
            for (int64_t t = 0; t < here; ++t, ++s.tile) die[(turn + d) & 7].push_back(s);
        }
        turn = (turn + static_cast<int>(left)) & 7;
        total += w.tiles;
    }
    // `turn` keeps the dies within one slot of each other, those from 0 on the longer ones
    for (int64_t s = 0; s < total; ++s) out.push_back(die[s & 7][s >> 3]);
}

std::vector<Shape> shapes_of(const std::vector<Matrix>& all, uint32_t first, uint32_t last) {
    std::vector<Shape> shapes;
    for (uint32_t i = first; i < last; ++i) {
        if (!shapes.empty() && shapes.back().m == all[i].m && shapes.back().n == all[i].n) ++shapes.back().count;
        else shapes.emplace_back(all[i], 1);
    }
    return shapes;
}

// Ends of the parts of a list that go through the workspace one after another, of about one size.
int cut(const std::vector<Matrix>& all, int planes, std::vector<uint32_t>& ends) {
    const uint32_t n = static_cast<uint32_t>(all.size());
    int64_t whole = 0;
    for (const Matrix& x : all) whole += 2 * halves_of(x, planes);
    double best = 0.0;
    // matrices that need more than kTogether are alone in their parts: there are never more parts than matrices
    const int64_t least = std::min<int64_t>((whole + kTogether - 1) / kTogether, n);
    for (int64_t parts = least; parts < least + kTurns && parts <= n; ++parts) {
        std::vector<uint32_t> here;
        double time = 0.0;
        int64_t left = whole;
        for (uint32_t first = 0; first < n;) {
            const int64_t share = left / std::max<int64_t>(1, parts - static_cast<int64_t>(here.size()));
            int64_t bytes = 0, slots[kKinds] = {};
            uint32_t last = first;
            for (; last < n; ++last) {
                const Matrix& x = all[last];
                const int64_t need = 2 * halves_of(x, planes), tiles = update_tiles(x.m, x.n, 64);
                const int64_t more[kKinds] = {symmetric_tiles(x.m, 64), symmetric_tiles(x.m, 64), tiles, x.parts, lay_tiles(x)};
                bool full = last > first && (bytes + need > kTogether || bytes + need / 2 > share);
                for (int k = 0; k < kKinds; ++k) {
                    if (more[k] > kMaxSlots) return JABAS_ERR_SIZE;
                    full = full || (last > first && slots[k] + more[k] > kMaxSlots);
                }
                if (full) break;
                bytes += need;
                for (int k = 0; k < kKinds; ++k) slots[k] += more[k];
            }
            const std::vector<Shape> shapes = shapes_of(all, first, last);
            time += step_of(shapes.data(), shapes.size(), planes);
            left -= bytes;
            here.push_back(last);
            first = last;
        }
        if (ends.empty() || time < best) {
            best = time;
            ends = here;
        }
    }
    return ends.empty() ? JABAS_ERR_SIZE : JABAS_OK;
}

struct Built {
    std::vector<Matrix> matrices;
    std::vector<uint64_t> fanout;
    std::vector<Part> parts;
    std::vector<Slot> slots;        // a part's kinds one after another
    Header head;
};

int build(const JabasMatrix* list, uint32_t n, int32_t precision, Built& b) {
    if (!list) return JABAS_ERR_NULL;
    if (n < 1 || n > kMaxMatrices) return JABAS_ERR_SIZE;
    if (precision != JABAS_F32 && precision != JABAS_BF16) return JABAS_ERR_DTYPE;
    const int planes = precision == JABAS_F32 ? 2 : 1;
    b.head = Header{};
    std::vector<uint32_t> order(n);
    std::iota(order.begin(), order.end(), 0u);
    for (uint32_t i = 0; i < n; ++i) {
        const int status = check_matrix(list[i]);
        if (status != JABAS_OK) return status;
        b.head.n_groups = std::max(b.head.n_groups, list[i].group + 1);
    }
    const auto sides = [&](uint32_t i) { return std::minmax(list[i].rows, list[i].cols); };
    std::stable_sort(order.begin(), order.end(), [&](uint32_t i, uint32_t j) {
        const auto x = sides(i), y = sides(j);
        return x.first != y.first ? x.first > y.first : x.second > y.second;
    });
    for (uint32_t i : order) {
        const JabasMatrix& j = list[i];
        Matrix x{};
        describe(x, j.rows, j.cols);
        x.src = j.grad;
        x.momentum = j.momentum;
        x.out = j.param;
        x.src_stride = j.cols;
        x.src_quads = !misaligned(j.grad, 16) && !misaligned(j.momentum, 16) && j.cols % 4 == 0;
        x.out_quads = !misaligned(j.param, 16) && j.cols % 4 == 0;
        for (uint32_t f = 0; f < j.n_fanout; ++f) x.out_quads = x.out_quads && !misaligned(j.fanout[f], 16);
        x.group = static_cast<int32_t>(j.group);
        x.lr_factor = static_cast<float>(j.lr_factor);
        x.n_fanout = j.n_fanout;
        x.fanout_at = static_cast<uint32_t>(b.fanout.size());
        for (uint32_t f = 0; f < j.n_fanout; ++f) b.fanout.push_back(reinterpret_cast<uint64_t>(j.fanout[f]));
        b.matrices.push_back(x);
    }
    // the matrices come with the longest shorter side first
    const int blocks = blocks_of(b.matrices[0]);
    bool tiny = true;
    for (const Matrix& x : b.matrices) tiny = tiny && tiny_fits(blocks, x.n);
    b.head.tiny = tiny ? blocks : 0;
    uint64_t halves_most = 0, sums_most = 0;
    if (tiny) {
        std::vector<Dealt> work;
        for (uint32_t i = 0; i < n; ++i) work.push_back({i, 1, 1});
        Part p{};
        deal(b.slots, work, b.matrices);
        p.total[kMomentum] = n;
        b.parts.push_back(p);
    } else {
        std::vector<uint32_t> ends;
        const int status = cut(b.matrices, planes, ends);
        if (status != JABAS_OK) return status;
        uint32_t first = 0;
        for (uint32_t last : ends) {
            int64_t halves = 0, sums = 0;
            for (uint32_t i = first; i < last; ++i) {
                Matrix& x = b.matrices[i];
                x.x_at = halves;
                x.a_at = halves + 4 * x.x_plane;
                x.part_at = sums;
                halves += halves_of(x, planes);
                sums += x.parts;
            }
            halves_most = std::max<uint64_t>(halves_most, halves);
            sums_most = std::max<uint64_t>(sums_most, sums);
            const std::vector<Shape> shapes = shapes_of(b.matrices, first, last);
            Part p{};
            for (int k = 0; k < kProducts; ++k) p.kernel[k] = kernel_of(shapes.data(), shapes.size(), static_cast<Product>(k), planes);
            for (int k = 0; k < kKinds; ++k) {
                std::vector<Dealt> work;
                int64_t total = 0;
                for (const Shape& s : shapes) total += k < kProducts ? s.count * s.tiles(static_cast<Product>(k), static_cast<Kind>(p.kernel[k])) : 0;
                for (uint32_t i = first; i < last; ++i) {
                    const Matrix& x = b.matrices[i];
                    if (k >= kProducts) {
                        work.push_back({i, k == kMomentum ? x.parts : lay_tiles(x), 1});
                        continue;
                    }
                    const Shape one(x, 1);
                    const Product product = static_cast<Product>(k);
                    const int splits = splits_of(one, product, static_cast<Kind>(p.kernel[k]), total, planes);
                    work.push_back({i, one.tiles(product, static_cast<Kind>(p.kernel[k])) * splits, splits});
                }
                if (k == kFirst)
                    std::stable_sort(work.begin(), work.end(), [&](const Dealt& v, const Dealt& w) { return b.matrices[v.matrix].n > b.matrices[w.matrix].n; });
                p.slots_at[k] = b.slots.size();
                deal(b.slots, work, b.matrices);
                p.total[k] = static_cast<uint32_t>(b.slots.size() - p.slots_at[k]);
            }
            b.parts.push_back(p);
            first = last;
        }
    }
    Header& h = b.head;
    h.magic = kMagic;
    h.n = n;
    h.n_parts = static_cast<uint32_t>(b.parts.size());
    h.precision = precision;
    h.matrices_at = round_up(sizeof(Header), 16);
    h.fanout_at = h.matrices_at + round_up(sizeof(Matrix) * n, 16);
    h.parts_at = h.fanout_at + round_up(8 * b.fanout.size(), 16);
    const uint64_t slots_at = h.parts_at + round_up(sizeof(Part) * b.parts.size(), 16);
    for (Part& p : b.parts)
        for (uint64_t& at : p.slots_at) at = slots_at + at * sizeof(Slot);
    h.bytes = round_up(slots_at + b.slots.size() * sizeof(Slot), 16);
    h.sums_bytes = round_up(8 * sums_most, 256);
    h.workspace = tiny ? 256 : h.sums_bytes + round_up(2 * halves_most, 256) + kShareBytes;
    return JABAS_OK;
}

// Nothing that C++ throws leaves the library; there is too little host memory where it does.
template <class F>
int guarded(const F& f) {
    try {
        return f();
    } catch (...) {
        return JABAS_ERR_SIZE;
    }
}

const Header* header_of(const void* blob) {
    const Header* h = static_cast<const Header*>(blob);
    return h && !misaligned(blob, 8) && h->magic == kMagic && h->n_parts ? h : nullptr;
}

}  // namespace
}  // namespace muon
}  // namespace jabas

using namespace jabas::muon;

JABAS_API size_t jabas_orthogonalize_workspace_bytes(const JabasOrthogonalize* o) {
    Batch b;
    Scales s;
    return guarded([&] { return describe_batch(o, b, s); }) == JABAS_OK ? static_cast<size_t>(b.bytes) : 0;
}

static int orthogonalize(const JabasOrthogonalize* o, void* workspace, size_t workspace_bytes, jabas_stream_t stream) {
    Batch b;
    Scales s;
    const int status = describe_batch(o, b, s);
    if (status != JABAS_OK) return status;
    if (!b.at_once) return JABAS_OK;
    if (!workspace || misaligned(workspace, 256) || workspace_bytes < static_cast<size_t>(b.bytes)) return JABAS_ERR_WORKSPACE;
    const Matrix& x = b.x;
    const int64_t size = o->dtype == JABAS_F32 ? 4 : 2, each = halves_of(x, b.planes);
    for (int64_t done = 0; done < o->batch; done += b.at_once) {
        const int64_t here = std::min(b.at_once, o->batch - done);
        Run r{};
        const Shape shape(x, here);
        if (!b.tiny)
            for (int k = 0; k < kProducts; ++k) r.kernel[k] = kernel_of(&shape, 1, static_cast<Product>(k), b.planes);
        r.planes = b.planes;
        r.dtype = o->dtype;
        r.tiny = b.tiny;
        Work w{};
        w.one = x;
        w.one.src = static_cast<const char*>(o->in) + size * done * o->in_batch_stride;
        w.one.out = static_cast<char*>(o->out) + size * done * o->rows * o->cols;
        w.one.a_at = here * 4 * x.x_plane;
        w.src_step = size * o->in_batch_stride;
        w.out_step = size * o->rows * o->cols;
        w.x_step = 4 * x.x_plane;
        w.a_step = each - w.x_step;
        w.part_step = x.parts;
        w.sums = static_cast<double*>(workspace);
        w.halves = static_cast<char*>(workspace) + (b.tiny ? 0 : b.sums_bytes);
        int64_t per[kKinds];
        for (int k = 0; k < kProducts; ++k) per[k] = b.tiny ? 0 : shape.tiles(static_cast<Product>(k), r.kernel[k]);
        per[kMomentum] = b.tiny ? 1 : x.parts;
        per[kLayOut] = lay_tiles(x);
        if (!b.tiny) r.shares = reinterpret_cast<float*>(static_cast<char*>(workspace) + (b.bytes - kShareBytes));
        for (int k = 0; k < kKinds; ++k) {
            r.work[k] = w;
            r.work[k].splits = 1;
            if (k < kProducts && !b.tiny) {
                r.work[k].splits = splits_of(shape, static_cast<Product>(k), r.kernel[k], per[k] * here, b.planes);
                per[k] *= r.work[k].splits;
            }
            r.work[k].per = static_cast<int32_t>(per[k]);
            r.work[k].total = static_cast<uint32_t>(per[k] * here);
        }
        UpdateArgs last{};
        last.out.dtype = o->dtype;
        const int launched = run(r, o->ns, s, last, static_cast<hipStream_t>(stream));
        if (launched != JABAS_OK) return launched;
    }
    return JABAS_OK;
}

JABAS_API int jabas_orthogonalize(const JabasOrthogonalize* o, void* workspace, size_t workspace_bytes, jabas_stream_t stream) {
    return guarded([&] { return orthogonalize(o, workspace, workspace_bytes, stream); });
}

JABAS_API size_t jabas_muon_plan_bytes(const JabasMatrix* matrices, uint32_t n, int32_t precision) {
    if (!matrices || n < 1 || n > kMaxMatrices || (precision != JABAS_F32 && precision != JABAS_BF16)) return 0;
    // every launch with the smallest tiles, every matrix a part
    uint64_t slots = 0, fanout = 0;
    for (uint32_t i = 0; i < n; ++i) {
        if (check_matrix(matrices[i]) != JABAS_OK) return 0;
        Matrix x{};
        describe(x, matrices[i].rows, matrices[i].cols);
        const int64_t symmetric = symmetric_tiles(x.m, 64);
        slots += x.parts + lay_tiles(x) + symmetric + std::min(kMostSplits * symmetric, symmetric + kSplitUnits) + update_tiles(x.m, x.n, 64);
        fanout += matrices[i].n_fanout;
    }
    return static_cast<size_t>(round_up(sizeof(Header), 16) + round_up(sizeof(Matrix) * n, 16) + round_up(8 * fanout, 16) + round_up(sizeof(Part) * n, 16) +
                               round_up(sizeof(Slot) * slots, 16));
}

JABAS_API int jabas_muon_plan_encode(const JabasMatrix* matrices, uint32_t n, int32_t precision, void* host_blob, size_t blob_bytes) {
    return guarded([&]() -> int {
        Built b;
        const int status = build(matrices, n, precision, b);
        if (status != JABAS_OK) return status;
        if (!host_blob) return JABAS_ERR_NULL;
        if (misaligned(host_blob, 8) || blob_bytes < b.head.bytes) return JABAS_ERR_PLAN;
        char* at = static_cast<char*>(host_blob);
        memset(at, 0, b.head.bytes);
        memcpy(at, &b.head, sizeof(Header));
        memcpy(at + b.head.matrices_at, b.matrices.data(), sizeof(Matrix) * n);
        if (!b.fanout.empty()) memcpy(at + b.head.fanout_at, b.fanout.data(), 8 * b.fanout.size());
        memcpy(at + b.head.parts_at, b.parts.data(), sizeof(Part) * b.parts.size());
        memcpy(at + b.parts[0].slots_at[0], b.slots.data(), sizeof(Slot) * b.slots.size());
        return JABAS_OK;
    });
}

JABAS_API size_t jabas_muon_workspace_bytes(const void* host_blob) {
    const Header* h = header_of(host_blob);
    return h ? h->workspace : 0;
}

JABAS_API int jabas_muon_step(const void* plan_host, const void* plan_dev, const JabasMuonArgs* args, void* workspace, size_t workspace_bytes,
                              jabas_stream_t stream) {
    if (!plan_host || !plan_dev || !args) return JABAS_ERR_NULL;
    const Header* h = header_of(plan_host);
    if (!h || misaligned(plan_dev, 16)) return JABAS_ERR_PLAN;
    Scales s;
    const int status = scales_of(args->ns, s);
    if (status != JABAS_OK) return status;
    if (args->ns.precision != h->precision) return JABAS_ERR_PLAN;
    if (!(args->momentum >= 0.0 && args->momentum < 1.0)) return JABAS_ERR_OPT;
    if (args->n_groups < static_cast<int32_t>(h->n_groups) || args->n_groups > JABAS_MAX_GROUPS) return JABAS_ERR_GROUP;
    if (!workspace || misaligned(workspace, 256) || workspace_bytes < h->workspace) return JABAS_ERR_WORKSPACE;
    const char *host = static_cast<const char*>(plan_host), *dev = static_cast<const char*>(plan_dev);
    const Part* parts = reinterpret_cast<const Part*>(host + h->parts_at);
    Work w{};
    w.table = reinterpret_cast<const Matrix*>(dev + h->matrices_at);
    w.fanout = reinterpret_cast<const uint64_t*>(dev + h->fanout_at);
    w.sums = static_cast<double*>(workspace);
    w.halves = static_cast<char*>(workspace) + h->sums_bytes;
    UpdateArgs last{};
    for (int g = 0; g < args->n_groups; ++g) {
        last.out.lr[g] = static_cast<float>(args->lr[g]);
        last.out.keep[g] = static_cast<float>(1.0 - args->lr[g] * args->weight_decay[g]);
    }
    for (uint32_t p = 0; p < h->n_parts; ++p) {
        Run r{};
        for (int k = 0; k < kProducts; ++k) r.kernel[k] = static_cast<Kind>(parts[p].kernel[k]);
        r.tiny = h->tiny;
        if (!r.tiny) r.shares = reinterpret_cast<float*>(static_cast<char*>(workspace) + (h->workspace - kShareBytes));
        r.planes = h->precision == JABAS_F32 ? 2 : 1;
        r.dtype = JABAS_F32;
        r.nesterov = args->nesterov != 0;
        r.momentum = static_cast<float>(args->momentum);
        r.fresh = static_cast<float>(1.0 - args->momentum);
        r.grad_scale = args->grad_scale;
        for (int k = 0; k < kKinds; ++k) {
            r.work[k] = w;
            r.work[k].slots = reinterpret_cast<const Slot*>(dev + parts[p].slots_at[k]);
            r.work[k].total = parts[p].total[k];
        }
        const int launched = run(r, args->ns, s, last, static_cast<hipStream_t>(stream));
        if (launched != JABAS_OK) return launched;
    }
    return JABAS_OK;
}
