// Kernels over the rows of a loss: the teacher's probabilities, the join of the vocabulary's tiles to a row's loss and
// state, the reduction over rows, and the distillation loss of logits in hand.
#include "loss_internal.h"

namespace jabas {
namespace loss {
namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

__device__ inline float bf16_as_float(uint32_t bits) { return __uint_as_float(bits << 16); }

__device__ inline float load_as_float(const void* p, int64_t i, int dtype) {
    if (dtype == JABAS_F32) return static_cast<const float*>(p)[i];
    return bf16_as_float(static_cast<const uint16_t*>(p)[i]);
}

__device__ inline uint16_t to_bf16(float x) {
    const uint32_t u = __float_as_uint(x);
    if ((u & 0x7fffffffu) > 0x7f800000u) return static_cast<uint16_t>((u >> 16) | 0x40);
    return static_cast<uint16_t>((u + 0x7fffu + ((u >> 16) & 1)) >> 16);
}

__device__ inline float wave_max(float x) {
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) x = fmaxf(x, __shfl_xor(x, i));
    return x;
}
__device__ inline float wave_sum(float x) {
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) x += __shfl_xor(x, i);
    return x;
}
__device__ inline double wave_sum(double x) {
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) x += __shfl_xor(x, i);
    return x;
}

// s 2^((from - to) c), 0 where there is nothing (from may then be -inf)
__device__ inline float rescale(float s, float from, float to, float c) {
    return s == 0.0f ? 0.0f : s * __builtin_amdgcn_exp2f((from - to) * c);
}

constexpr int kEntriesPerLane = 4;
static_assert(kNarrowRows <= 64, "a lane per row");
static_assert(64 * kEntriesPerLane > JABAS_LOSS_MAX_ENTRIES, "a row's entries fit a wave");

// A row's entries, entry lane + 64 i in place i of the lanes that hold it.
struct WaveEntries {
    int32_t index[kEntriesPerLane];     // -1: none (also where a name outside the vocabulary makes the row's loss NaN)
    float p[kEntriesPerLane];
    float mass, entropy;                // sums of p and p log p; the latter NaN with a name outside the vocabulary
    bool counts;
};

// The teacher's probabilities of a row, by one wave. Entries that name a token twice are one event with both probabilities: the first keeps
// the sum. `names` and `probs`: 256 places of LDS of the wave's own.
__device__ inline WaveEntries wave_entries(const TeacherArgs& a, int64_t row, int32_t* names, float* probs) {
    const int lane = threadIdx.x & 63;
    WaveEntries w;
    float t[kEntriesPerLane], logp[kEntriesPerLane], peak = -INFINITY, sum = 0.0f;
    bool is[kEntriesPerLane], outside = false;
#pragma unroll
    for (int i = 0; i < kEntriesPerLane; ++i) {
        const int j = lane + 64 * i;
        const int64_t name = j < a.k ? a.index[row * a.k + j] : -1;
        t[i] = j < a.k ? load_as_float(a.logits, row * a.k + j, a.dtype) : -INFINITY;
        is[i] = name >= 0 && !(t[i] == -INFINITY);
        outside |= is[i] && name >= a.vocab;
        w.index[i] = is[i] ? static_cast<int32_t>(name < a.vocab ? name : a.vocab) : -1;
        if (is[i]) peak = fmaxf(peak, t[i]);
    }
    peak = wave_max(peak);
    outside = __any(outside);
    float norm;
    if (a.lse) {
        norm = a.lse[row];
    } else {
#pragma unroll
        for (int i = 0; i < kEntriesPerLane; ++i)
            if (is[i]) sum += expf((t[i] - peak) * a.inv_t);
        norm = logf(wave_sum(sum));
    }
    bool any = false;
#pragma unroll
    for (int i = 0; i < kEntriesPerLane; ++i) {
        logp[i] = a.lse ? t[i] * a.inv_t - norm : (t[i] - peak) * a.inv_t - norm;
        w.p[i] = is[i] ? expf(logp[i]) : 0.0f;
        any |= is[i];
        names[lane + 64 * i] = w.index[i];
        probs[lane + 64 * i] = w.p[i];
    }
    w.counts = __any(any);
    asm volatile("" ::: "memory");        // the wave's own writes, in order: read back as they were written
    int again[kEntriesPerLane] = {};        // how many of the names are this one
    for (int o = 0; o < a.k; o += 4) {
        const int4 four = *reinterpret_cast<const int4*>(names + o);
#pragma unroll
        for (int i = 0; i < kEntriesPerLane; ++i) again[i] += (four.x == w.index[i]) + (four.y == w.index[i]) + (four.z == w.index[i]) + (four.w == w.index[i]);
    }
    w.mass = w.entropy = 0.0f;
#pragma unroll
    for (int i = 0; i < kEntriesPerLane; ++i) {
        if (is[i] && again[i] > 1) {        // seldom
            const int j = lane + 64 * i;
            float all = 0.0f;
            bool first = true;
            for (int o = 0; o < a.k; ++o)
                if (names[o] == w.index[i]) {
                    first &= o >= j;
                    all += probs[o];
                }
            is[i] = first;
            w.p[i] = first ? all : 0.0f;
            logp[i] = logf(all);
        }
        if (is[i]) {
            w.mass += w.p[i];
            if (w.p[i] != 0.0f) w.entropy += w.p[i] * logp[i];
        }
        if (!is[i] || outside) w.index[i] = -1;
    }
    w.mass = wave_sum(w.mass);
    w.entropy = outside ? NAN : wave_sum(w.entropy);
    return w;
}

__device__ inline void keep_entries(const TeacherArgs& a, int64_t row, const WaveEntries& w) {
#pragma unroll
    for (int i = 0; i < kEntriesPerLane; ++i) {
        const int j = (threadIdx.x & 63) + 64 * i;
        if (j < a.k) {
            a.entry_index[row * a.k + j] = w.index[i];
            a.entry_p[row * a.k + j] = w.p[i];
        }
    }
}

// What a row's entries, their logits and the rest of its tokens (peak and sum) make of it, by one wave.
struct RowResult {
    RowState state;
    float loss;
};
__device__ inline RowResult row_result(const TeacherArgs& a, const WaveEntries& w, const float (&z)[kEntriesPerLane], float rest_peak, float rest_sum) {
    const float c = a.inv_t * kLog2e;
    float top = rest_peak;
#pragma unroll
    for (int i = 0; i < kEntriesPerLane; ++i)
        if (w.index[i] >= 0) top = fmaxf(top, z[i]);
    top = wave_max(top);
    float held = 0.0f, cross = 0.0f;
#pragma unroll
    for (int i = 0; i < kEntriesPerLane; ++i)
        if (w.index[i] >= 0 && z[i] != -INFINITY) held += __builtin_amdgcn_exp2f((z[i] - top) * c);
    held = wave_sum(held);
    const float all = held + rescale(rest_sum, rest_peak, top, c), log_all = logf(all);
#pragma unroll
    for (int i = 0; i < kEntriesPerLane; ++i)
        if (w.index[i] >= 0 && w.p[i] != 0.0f) cross += w.p[i] * ((z[i] - top) * a.inv_t - log_all);
    cross = wave_sum(cross);
    RowResult r = {{0.0f, 0.0f, 0.0f, 0.0f}, 0.0f};
    int named = 0;
#pragma unroll
    for (int i = 0; i < kEntriesPerLane; ++i) named += __popcll(__ballot(w.index[i] >= 0));
    if (!w.counts) return r;
    // Tokens that are no entry may all be at -inf (their sum is 0): the student cannot meet what is left then, R = 0 and the loss is
    // infinite. M holds it all the same; r q / R, which has no value at those tokens, is taken as 0.
    const bool others = named < a.vocab, met = rest_sum != 0.0f;
    const float left = a.lse && others ? fmaxf(1.0f - w.mass, 0.0f) : 0.0f, mass = w.mass + left;
    float rest = -INFINITY, share = 0.0f;       // of the student: log R and R
    if (met) {
        rest = (rest_peak - top) * a.inv_t + logf(rest_sum) - log_all;
        share = expf(rest);
    }
    r.loss = w.entropy - cross;
    if (left != 0.0f) r.loss += left * (logf(left) - rest);
    r.loss *= a.t * a.t;
    r.state.peak_rest = met ? rest_peak : 0.0f;
    r.state.slope = met ? (mass * share - left) / rest_sum : 0.0f;
    r.state.peak = top;
    r.state.mass = mass / all;
    if (r.state.slope == 0.0f && r.state.mass == 0.0f) r.state.mass = 0x1p-149f;       // every token an entry, every p next to nothing: it counts all the same
    if (w.entropy != w.entropy) r.state.slope = r.state.mass = NAN;
    return r;
}

// A wave per row; bound by its chain of loads and sums: 7 us for 800 rows of 32 entries, 10 for 4096 of 64.
__global__ __launch_bounds__(kThreads) void teacher_kernel(TeacherArgs a) {
    __shared__ __align__(16) int32_t names[kThreads / 64][64 * kEntriesPerLane];
    __shared__ float probs[kThreads / 64][64 * kEntriesPerLane];
    const int wave = threadIdx.x >> 6;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / 64) + wave;
    if (row >= a.rows) return;
    const WaveEntries w = wave_entries(a, row, names[wave], probs[wave]);
    keep_entries(a, row, w);
    if ((threadIdx.x & 63) == 0) a.row[row] = make_float4(w.mass, w.entropy, w.counts ? 1.0f : 0.0f, 0.0f);
}

// A row against its entries, as the teacher's kernel and the logits' kernels left them, by one wave.
__device__ inline RowResult entries_result(const JoinArgs& a, int64_t row, float peak, float sum) {
    const float4 teacher = a.teacher_row[row];
    WaveEntries w;
    w.mass = teacher.x;
    w.entropy = teacher.y;
    w.counts = teacher.z != 0.0f;
    float z[kEntriesPerLane];
#pragma unroll
    for (int i = 0; i < kEntriesPerLane; ++i) {
        const int j = (threadIdx.x & 63) + 64 * i;
        w.index[i] = j < a.entries.k ? a.entries.index[row * a.entries.k + j] : -1;
        w.p[i] = j < a.entries.k ? a.entries.p[row * a.entries.k + j] : 0.0f;
        z[i] = w.index[i] >= 0 ? a.entry_logit[row * a.entries.k + j] : 0.0f;
    }
    return row_result(a.teacher, w, z, peak, sum);
}

// A row against its label.
__device__ inline RowResult label_result(const JoinArgs& a, int64_t row, float peak, float sum, float total) {
    RowResult r = {{0.0f, 0.0f, 0.0f, 0.0f}, 0.0f};
    const int64_t label = a.entries.target[row];
    if (label == a.entries.ignore_index) return r;
    r.state.peak_rest = r.state.peak = peak;
    r.state.slope = r.state.mass = 1.0f / sum;
    const float e = a.smoothing;
    if (label < 0 || label >= a.vocab) {
        r.loss = r.state.slope = r.state.mass = NAN;
    } else {
        r.loss = logf(sum) + (1.0f - e) * (peak - a.entry_logit[row]);
        if (e != 0.0f) r.loss += e * (peak - total / static_cast<float>(a.vocab));
    }
    return r;
}

constexpr int kJoinThreads = 1024, kJoinRows = 16, kJoinWaves = kJoinThreads / 64;

__device__ inline bool counts(const RowState& st) { return !(st.slope == 0.0f && st.mass == 0.0f); }

// The sum over a workgroup of WAVES waves, in thread 0.
template <int WAVES>
__device__ inline double group_sum(double x) {
    __shared__ double sums[WAVES];
    x = wave_sum(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = x;
    __syncthreads();
    x = sums[0];
    for (int i = 1; i < WAVES; ++i) x += sums[i];
    return x;
}

// The loss and the share of a row from the sums, by one thread.
__device__ inline void finish(double sum, double number, int reduction, float* loss_out, float* reduce) {
    const double share = reduction == JABAS_LOSS_MEAN && number > 0.0 ? 1.0 / number : 1.0;
    *reduce = static_cast<float>(share);
    if (reduction != JABAS_LOSS_NONE) *loss_out = static_cast<float>(sum * share);
}

__global__ __launch_bounds__(kJoinThreads) void reduce_kernel(const float* row_loss, const RowState* state, int64_t rows, int reduction,
                                                              float* loss_out, float* reduce) {
    double sum = 0.0, number = 0.0;
    for (int64_t i = threadIdx.x; i < rows; i += kJoinThreads) {
        const float loss = row_loss[i];
        sum += loss;
        number += counts(state[i]) ? 1.0 : 0.0;
        if (reduction == JABAS_LOSS_NONE) loss_out[i] = loss;
    }
    sum = group_sum<kJoinWaves>(sum);
    number = group_sum<kJoinWaves>(number);
    if (threadIdx.x == 0) finish(sum, number, reduction, loss_out, reduce);
}

// A row's loss, and whether it counts, stored past the dies' own caches for the workgroup that sums over the rows.
__device__ inline void hand_over(float* row_loss, int64_t rows, int64_t row, float loss, bool counts) {
    __hip_atomic_store(row_loss + row, loss, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(row_loss + rows + row, counts ? 1.0f : 0.0f, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline float handed_over(const float* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// A row of a part of the vocabulary joined with another's: (peak, sum) of both.
__device__ inline void merge(float& peak, float& sum, float other_peak, float other_sum, float c) {
    const float p = fmaxf(peak, other_peak);
    sum = rescale(sum, peak, p, c) + rescale(other_sum, other_peak, p, c);
    peak = p;
}

// The wave's stores are in memory, not only on their way.
__device__ inline void stores_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// 4096 rows of 512 tiles take 15 us (17 MB; 24 with 64 rows a workgroup, whose chain of loads is four times as long), 800 of 253 with 32
// entries each 11. kJoinRows rows per workgroup: 16 lanes of a wave take a row each, a sixty-fourth of the vocabulary's tiles; then the parts are joined,
// and each wave takes the entries of its row.
__global__ __launch_bounds__(kJoinThreads) void join_kernel(JoinArgs a) {
    constexpr int kParts = kJoinThreads / kJoinRows;
    static_assert(kJoinRows == kJoinWaves, "a row's entries per wave");
    __shared__ float peaks[kJoinWaves][kJoinRows], sums[kJoinWaves][kJoinRows], totals[kJoinWaves][kJoinRows];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, at = lane % kJoinRows;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kJoinRows, mine = first + at, rows = *a.live.live;
    if (first >= rows && first) return;
    float peak = -INFINITY, sum = 0.0f, total = 0.0f;
    if (mine < rows)
        for (int i = threadIdx.x / kJoinRows; i < a.tiles; i += kParts) {
            const float2 part = a.partial[static_cast<int64_t>(i) * a.rows + mine];
            merge(peak, sum, part.x, part.y, a.c);
            if (a.total) total += a.total[static_cast<int64_t>(i) * a.rows + mine];
        }
#pragma unroll
    for (int x = kJoinRows; x < 64; x *= 2) {
        merge(peak, sum, __shfl_xor(peak, x), __shfl_xor(sum, x), a.c);
        total += __shfl_xor(total, x);
    }
    if (lane < kJoinRows) {
        peaks[wave][at] = peak;
        sums[wave][at] = sum;
        totals[wave][at] = total;
    }
    __syncthreads();
    if (wave == 0) {
        for (int i = 1; i < kJoinWaves; ++i) {
            merge(peak, sum, peaks[i][at], sums[i][at], a.c);
            total += totals[i][at];
        }
        if (lane < kJoinRows) {
            peaks[0][at] = peak;
            sums[0][at] = sum;
        }
    }
    __syncthreads();
    if (!a.entries.index && threadIdx.x < kJoinRows && mine < rows) {
        const int32_t row = a.live.map[mine];
        const RowResult r = label_result(a, row, peak, sum, total);
        a.state[row] = r.state;
        __hip_atomic_store(a.row_loss + row, r.loss, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (a.entries.index && first + wave < rows) {
        const int64_t row = a.live.map[first + wave];
        const RowResult result = entries_result(a, row, peaks[0][wave], sums[0][wave]);
        if (lane == 0) {
            a.state[row] = result.state;
            __hip_atomic_store(a.row_loss + row, result.loss, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    if (a.reduction == JABAS_LOSS_NONE) {       // row_loss is the result
        if (first == 0 && threadIdx.x == 0) *a.reduce = 1.0f;
        return;
    }
    // The last workgroup to finish sums the rows' losses, in order. They were stored past the dies' own caches, where every wave waits for
    // them to be, so one thread's release is enough, and they are loaded past them.
    __shared__ uint32_t done;
    stores_done();
    __syncthreads();
    if (threadIdx.x == 0) done = __hip_atomic_fetch_add(a.ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (done + 1 != (rows > kJoinRows ? static_cast<uint32_t>((rows + kJoinRows - 1) / kJoinRows) : 1)) return;
    double loss = 0.0;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < a.rows; i += kJoinThreads) loss += handed_over(a.row_loss + i);
    loss = group_sum<kJoinWaves>(loss);
    if (threadIdx.x == 0) finish(loss, static_cast<double>(rows), a.reduction, a.loss_out, a.reduce);
}

// Few rows: a workgroup joins a row's tiles; the last one to finish sums the rows' losses, in order.
__global__ __launch_bounds__(kThreads) void narrow_join_kernel(JoinArgs a) {
    __shared__ float peaks[kThreads / 64], sums[kThreads / 64], totals[kThreads / 64];
    const int t = threadIdx.x, wave = t >> 6;
    const int64_t row = blockIdx.x;
    float peak = -INFINITY, sum = 0.0f, total = 0.0f;
    for (int i = t; i < a.tiles; i += kThreads) {
        const float2 part = a.partial[row * a.tiles + i];
        const float p = fmaxf(peak, part.x);
        sum = rescale(sum, peak, p, a.c) + rescale(part.y, part.x, p, a.c);
        peak = p;
        if (a.total) total += a.total[row * a.tiles + i];
    }
    const float top = wave_max(peak);
    sum = wave_sum(rescale(sum, peak, top, a.c));
    total = wave_sum(total);
    if ((t & 63) == 0) {
        peaks[wave] = top;
        sums[wave] = sum;
        totals[wave] = total;
    }
    __syncthreads();
    if (wave) return;
    peak = peaks[0];
    sum = sums[0];
    total = totals[0];
    for (int i = 1; i < kThreads / 64; ++i) {
        const float p = fmaxf(peak, peaks[i]);
        sum = rescale(sum, peak, p, a.c) + rescale(sums[i], peaks[i], p, a.c);
        peak = p;
        total += totals[i];
    }
    const RowResult r = a.entries.index ? entries_result(a, row, peak, sum) : label_result(a, row, peak, sum, total);
    uint32_t done = 0;
    if (t == 0) {
        a.state[row] = r.state;
        hand_over(a.row_loss, a.rows, row, r.loss, counts(r.state));
        if (a.reduction == JABAS_LOSS_NONE) a.loss_out[row] = r.loss;
        done = __hip_atomic_fetch_add(a.ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    }
    done = __builtin_amdgcn_readfirstlane(done);
    if (done + 1 != a.rows) return;
    const int lane = t & 63;
    double loss = 0.0, number = 0.0;
    if (lane < a.rows) {
        loss = handed_over(a.row_loss + lane);
        number = handed_over(a.row_loss + a.rows + lane);
    }
    loss = wave_sum(loss);
    number = wave_sum(number);
    if (lane == 0) finish(loss, number, a.reduction, a.loss_out, a.reduce);
}

// The gradient of a row's loss in units of dz; 0 where it does not count.
__device__ inline float row_gradient(const float* upstream, int per_row, const float* reduce, float t, const RowState& st, int64_t row) {
    return counts(st) ? upstream[per_row ? row : 0] * (*reduce * t) : 0.0f;
}

// Lists the rows for which is(n, load(n)), in order, and from the end of the list on those for which not, by one workgroup: kRun rows a
// thread at a time, whose loads are all under way before the first is looked at.
constexpr int kRun = 8;
template <class L, class F>
__device__ inline void list_live(int64_t rows, int32_t* map, int32_t* live, const L& load, const F& is) {
    __shared__ int32_t counts_of[kRun][kJoinWaves];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    int32_t before = 0;
    for (int64_t first = 0; first < rows; first += kJoinThreads * kRun) {
        decltype(load(0)) held[kRun];
        uint64_t bits[kRun];        // of the wave's 64 rows in run i
#pragma unroll
        for (int i = 0; i < kRun; ++i) held[i] = load(min(first + i * kJoinThreads + t, rows - 1));
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
            const int64_t n = first + i * kJoinThreads + t;
            bits[i] = __ballot(n < rows && is(n, held[i]));
            if (lane == 0) counts_of[i][wave] = __popcll(bits[i]);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
            int32_t at = before;
#pragma unroll
            for (int w = 0; w < kJoinWaves; ++w) {
                if (w < wave) at += counts_of[i][w];
                before += counts_of[i][w];
            }
            at += __popcll(bits[i] & ((uint64_t{1} << lane) - 1));
            const int64_t n = first + i * kJoinThreads + t;
            if (n < rows) map[(bits[i] >> lane) & 1 ? at : rows - 1 - (n - at)] = static_cast<int32_t>(n);     // n - at: rows before n not on the list
        }
        __syncthreads();
    }
    if (t == 0) *live = before;
}

// One workgroup, because the list is in order; bound by latency: 6400 rows 9 us, 1600 8 us.
__global__ __launch_bounds__(kJoinThreads) void live_kernel(LiveArgs a) {
    if (threadIdx.x == 0) *a.ticket = 0;
    const auto drop = [&](int64_t n, bool is) {
        if (!is) {
            a.state[n] = RowState{0.0f, 0.0f, 0.0f, 0.0f};
            a.row_loss[n] = 0.0f;
        }
        return is;
    };
    if (a.teacher_row)
        list_live(a.rows, a.map, a.live, [&](int64_t n) { return a.teacher_row[n].z; }, [&](int64_t n, float counts) { return drop(n, counts != 0.0f); });
    else
        list_live(a.rows, a.map, a.live, [&](int64_t n) { return a.target[n]; }, [&](int64_t n, int64_t label) { return drop(n, label != a.ignore_index); });
}

// A wave per row; bound by latency: 800 rows of 32 entries 4.9 us, 4096 of 64 4.6. fp16 holds up to 2 in units of dz; a row whose sum is not
// finite has no gradient that is.
__global__ __launch_bounds__(kThreads) void down_kernel(const float* p, int64_t rows, int32_t k, float* down) {
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / 64) + (threadIdx.x >> 6);
    if (row >= rows) return;
    const int lane = threadIdx.x & 63;
    float mass = 0.0f;
#pragma unroll
    for (int i = 0; i < kEntriesPerLane; ++i)
        if (lane + 64 * i < k) mass += p[row * k + lane + 64 * i];
    mass = wave_sum(mass);
    if (lane) return;
    int e;
    frexpf(mass, &e);
    down[row] = mass > 1.9f && mass < INFINITY ? ldexpf(1.0f, -e) : 1.0f;
}

// As above: 6400 rows 12 us, 1600 9 us.
__global__ __launch_bounds__(kJoinThreads) void row_grad_kernel(RowGradArgs a) {
    __shared__ float peaks[kJoinWaves];
    float top = 0.0f;
    bool bad = false;
    const float share = a.reduce[0] * a.t;
    if (a.zero)
        for (int64_t i = threadIdx.x; i < a.zeros; i += kJoinThreads) a.zero[i] = 0;
    struct Row {
        RowState state;
        float upstream, down;
    };
    list_live(a.rows, a.map, a.live, [&](int64_t n) { return Row{a.state[n], a.upstream[a.per_row ? n : 0], a.down ? a.down[n] : 1.0f}; }, [&](int64_t n, const Row& r) {
        const float g = counts(r.state) ? r.upstream * share / r.down : 0.0f;
        a.grad[n] = g;
        bad |= !(fabsf(g) < INFINITY);
        top = fmaxf(top, fabsf(g));
        return g != 0.0f;       // rows without an upstream gradient have no part in the products either, whatever they hold
    });
    top = wave_max(top);
    if (__any(bad)) top = INFINITY;
    if ((threadIdx.x & 63) == 0) peaks[threadIdx.x >> 6] = top;
    __syncthreads();
    for (int i = 0; i < kJoinWaves; ++i) top = fmaxf(top, peaks[i]);
    // rows of a gradient that is not finite make everything that sums over rows NaN: the ratio says 1 for all that count
    const bool whole = top < INFINITY;
    if (threadIdx.x == 0) *a.peak = whole ? top : NAN;
    for (int64_t first = threadIdx.x; first < a.rows; first += kJoinThreads * kRun) {
        float g[kRun];
#pragma unroll
        for (int i = 0; i < kRun; ++i) g[i] = a.grad[min(first + i * kJoinThreads, a.rows - 1)];
#pragma unroll
        for (int i = 0; i < kRun; ++i)
            if (first + i * kJoinThreads < a.rows)
                a.ratio[first + i * kJoinThreads] = g[i] == 0.0f ? 0.0f : whole ? g[i] / top : 1.0f;
    }
}

// 16384 tokens of 20 tiles 9 us.
__global__ __launch_bounds__(kThreads) void bias_sum_kernel(const float* parts, const int32_t* live, int32_t tile, int64_t stride, int64_t n, void* out, int32_t dtype) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= n) return;
    const int32_t tiles = (*live + tile - 1) / tile;
    float sum = 0.0f;
    for (int t = 0; t < tiles; ++t) sum += parts[t * stride + i];
    if (dtype == JABAS_F32) static_cast<float*>(out)[i] = sum;
    else static_cast<uint16_t*>(out)[i] = to_bf16(sum);
}

__global__ __launch_bounds__(kThreads) void zero_kernel(uint16_t* p, size_t n) {
    for (size_t i = static_cast<size_t>(blockIdx.x) * kThreads + threadIdx.x; i < n; i += static_cast<size_t>(gridDim.x) * kThreads) p[i] = 0;
}

// ------------------------------------------------------------------ logits in hand

template <class T>
struct Vec;
template <>
struct Vec<float> {
    static constexpr int n = 4;
    static constexpr int dtype = JABAS_F32;
    static __device__ float get(float x) { return x; }
    static __device__ float put(float x) { return x; }
};
template <>
struct Vec<uint16_t> {
    static constexpr int n = 8;
    static constexpr int dtype = JABAS_BF16;
    static __device__ float get(uint16_t x) { return bf16_as_float(x); }
    static __device__ uint16_t put(float x) { return to_bf16(x); }
};

// 16 bytes at any element: rows of an odd vocabulary start anywhere
template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
    T v[Vec<T>::n];
};
typedef uint32_t LoosePack __attribute__((ext_vector_type(4), aligned(2)));

// STREAM: past the caches, see kCacheBytes
template <bool STREAM, class T>
__device__ inline Pack<T> load_pack(const T* p) {
    if constexpr (!STREAM) return *reinterpret_cast<const Pack<T>*>(p);
    const LoosePack v = __builtin_nontemporal_load(reinterpret_cast<const LoosePack*>(p));
    Pack<T> out;
    __builtin_memcpy(&out, &v, 16);
    return out;
}
template <bool STREAM, class T>
__device__ inline void store_pack(T* p, const Pack<T>& x) {
    if constexpr (!STREAM) {
        *reinterpret_cast<Pack<T>*>(p) = x;
    } else {
        LoosePack v;
        __builtin_memcpy(&v, &x, 16);
        __builtin_nontemporal_store(v, reinterpret_cast<LoosePack*>(p));
    }
}

// Bits of the tokens [begin, end) that are entries of a row, by thread j for entry j; `mask` holds zeros.
static_assert(JABAS_LOSS_MAX_ENTRIES <= kThreads, "a thread per entry");
__device__ inline void mark(uint32_t* mask, int64_t name, int64_t begin, int64_t end) {
    if (name >= begin && name < end) atomicOr(&mask[(name - begin) >> 5], 1u << ((name - begin) & 31));
}

// Running maximum and sum of 2^((z - max) c) over the tokens [begin, end) of a row that the mask leaves, for the workgroup: each thread
// takes kUnroll vectors at a time, so that 64 bytes of each are on their way; its maximum moves once for all of them.
constexpr int kUnroll = 4;
template <bool STREAM, class T>
__device__ inline void stream_row(const T* z, int64_t begin, int64_t end, const uint32_t* mask, float c, float& peak, float& sum) {
    constexpr int n = Vec<T>::n;
    peak = -INFINITY;
    sum = 0.0f;
    const auto take = [&](float (&x)[kUnroll * n]) {
        float top = peak;
#pragma unroll
        for (int i = 0; i < kUnroll * n; ++i) top = fmaxf(top, x[i]);
        const float base = top == -INFINITY ? 0.0f : top;
        float more = 0.0f;
#pragma unroll
        for (int i = 0; i < kUnroll * n; ++i) more += __builtin_amdgcn_exp2f((x[i] - base) * c);
        sum = rescale(sum, peak, base, c) + more;
        peak = top;
    };
    const auto drop = [&](float* x, int64_t at) {       // n divides 32: one word holds a vector's bits
        const int off = static_cast<int>(at - begin);
        const uint32_t hits = mask[off >> 5] >> (off & 31) & ((1u << n) - 1);
        if (hits)
#pragma unroll
            for (int i = 0; i < n; ++i)
                if ((hits >> i) & 1) x[i] = -INFINITY;
    };
    int64_t first = begin;
    constexpr int64_t kRound = static_cast<int64_t>(kThreads) * n * kUnroll;
    for (; first + kRound <= end; first += kRound) {
        Pack<T> p[kUnroll];
        float x[kUnroll * n];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) p[u] = load_pack<STREAM>(z + first + (u * kThreads + threadIdx.x) * n);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
            for (int i = 0; i < n; ++i) x[u * n + i] = Vec<T>::get(p[u].v[i]);
            drop(x + u * n, first + (u * kThreads + threadIdx.x) * n);
        }
        take(x);
    }
    if (first + static_cast<int>(threadIdx.x) * n < end) {
        float x[kUnroll * n];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int64_t at = first + (u * kThreads + threadIdx.x) * n;
            if (at + n <= end) {
                const Pack<T> p = *reinterpret_cast<const Pack<T>*>(z + at);
#pragma unroll
                for (int i = 0; i < n; ++i) x[u * n + i] = Vec<T>::get(p.v[i]);
            } else {
#pragma unroll
                for (int i = 0; i < n; ++i) x[u * n + i] = at + i < end ? Vec<T>::get(z[at + i]) : -INFINITY;
            }
            if (at < end) drop(x + u * n, at);
        }
        take(x);
    }
    __shared__ float peaks[kThreads / 64], sums[kThreads / 64];
    const float top = wave_max(peak);
    sum = wave_sum(rescale(sum, peak, top, c));
    if ((threadIdx.x & 63) == 0) {
        peaks[threadIdx.x >> 6] = top;
        sums[threadIdx.x >> 6] = sum;
    }
    __syncthreads();
    peak = peaks[0];
    sum = sums[0];
#pragma unroll
    for (int i = 1; i < kThreads / 64; ++i) {
        const float p = fmaxf(peak, peaks[i]);
        sum = rescale(sum, peak, p, c) + rescale(sums[i], peaks[i], p, c);
        peak = p;
    }
}

// A row per workgroup: entries, stream, loss and state in one launch. Wave 0 sees to the entries. Long rows are bound by memory: 4096 x 131072
// bf16 178 us (6.0 TB/s); of 64 KB a row, the latency of the entries in front and behind weighs: 2560 x 32317 bf16 48 us (3.4 TB/s).
template <class T, bool STREAM>
__global__ __launch_bounds__(kThreads) void topk_row_kernel(TopkArgs a) {
    extern __shared__ __align__(16) uint32_t mask[];
    __shared__ __align__(16) int32_t names[64 * kEntriesPerLane];
    __shared__ float probs[64 * kEntriesPerLane];
    const int64_t row = blockIdx.x;
    const int t = threadIdx.x;
    const T* z = static_cast<const T*>(a.logits) + row * a.stride;
    const int64_t name = t < a.teacher.k ? a.teacher.index[row * a.teacher.k + t] : -1;
    const bool is = name >= 0 && !(load_as_float(a.teacher.logits, row * a.teacher.k + t, a.dtype) == -INFINITY);
    const int words = static_cast<int>((a.vocab + 31) / 32);
    for (int i = t; i < words; i += kThreads) mask[i] = 0;
    const bool counts = __syncthreads_or(is);
    if (is) mark(mask, name, 0, a.vocab);
    __syncthreads();
    float peak = -INFINITY, sum = 0.0f;
    if (counts) stream_row<STREAM>(z, 0, a.vocab, mask, a.c, peak, sum);
    if (t >= 64) return;
    const WaveEntries w = wave_entries(a.teacher, row, names, probs);
    keep_entries(a.teacher, row, w);
    float logits[kEntriesPerLane];
#pragma unroll
    for (int i = 0; i < kEntriesPerLane; ++i) logits[i] = w.index[i] >= 0 ? Vec<T>::get(z[w.index[i]]) : 0.0f;
    const RowResult r = row_result(a.teacher, w, logits, peak, sum);
    if (t == 0) {
        a.state[row] = r.state;
        a.row_loss[row] = r.loss;
    }
}

// A chunk of a row per workgroup, joined by topk_join_kernel.
template <class T, bool STREAM>
__global__ __launch_bounds__(kThreads) void topk_split_kernel(TopkArgs a) {
    extern __shared__ __align__(16) uint32_t mask[];
    const int64_t row = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
    const int64_t begin = split * a.chunk, end = min(a.vocab, begin + a.chunk);
    const int t = threadIdx.x;
    const T* z = static_cast<const T*>(a.logits) + row * a.stride;
    const int64_t name = t < a.teacher.k ? a.teacher.index[row * a.teacher.k + t] : -1;
    const bool is = name >= 0 && !(load_as_float(a.teacher.logits, row * a.teacher.k + t, a.dtype) == -INFINITY);
    const int words = static_cast<int>((end - begin + 31) / 32);
    for (int i = t; i < words; i += kThreads) mask[i] = 0;
    const bool counts = __syncthreads_or(is);
    if (is) mark(mask, name, begin, end);
    __syncthreads();
    float peak = -INFINITY, sum = 0.0f;
    if (counts) stream_row<STREAM>(z, begin, end, mask, a.c, peak, sum);
    if (t == 0) {
        a.partial[row * a.splits + split] = make_float2(peak, sum);
        if (blockIdx.x == 0) *a.ticket = 0;
    }
}

// A wave per row; the last workgroup to finish sums the rows' losses, in order.
template <class T>
__global__ __launch_bounds__(kThreads) void topk_join_kernel(TopkArgs a) {
    constexpr int kWaves = kThreads / 64;
    __shared__ __align__(16) int32_t names[kWaves][64 * kEntriesPerLane];
    __shared__ float probs[kWaves][64 * kEntriesPerLane];
    __shared__ uint32_t done;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kWaves + wave;
    if (row < a.rows) {
        float peak = -INFINITY, sum = 0.0f;
        for (int i = lane; i < a.splits; i += 64) {
            const float2 part = a.partial[row * a.splits + i];
            merge(peak, sum, part.x, part.y, a.c);
        }
        const float top = wave_max(peak);
        sum = wave_sum(rescale(sum, peak, top, a.c));
        const WaveEntries w = wave_entries(a.teacher, row, names[wave], probs[wave]);
        keep_entries(a.teacher, row, w);
        const T* z = static_cast<const T*>(a.logits) + row * a.stride;
        float logits[kEntriesPerLane];
#pragma unroll
        for (int i = 0; i < kEntriesPerLane; ++i) logits[i] = w.index[i] >= 0 ? Vec<T>::get(z[w.index[i]]) : 0.0f;
        const RowResult r = row_result(a.teacher, w, logits, top, sum);
        if (lane == 0) {
            a.state[row] = r.state;
            hand_over(a.row_loss, a.rows, row, r.loss, counts(r.state));
            if (a.reduction == JABAS_LOSS_NONE) a.loss_out[row] = r.loss;
        }
    }
    stores_done();
    __syncthreads();
    if (threadIdx.x == 0) done = __hip_atomic_fetch_add(a.ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (done + 1 != gridDim.x) return;
    double loss = 0.0, number = 0.0;
    for (int64_t i = threadIdx.x; i < a.rows; i += kThreads) {
        loss += handed_over(a.row_loss + i);
        number += handed_over(a.row_loss + a.rows + i);
    }
    loss = group_sum<kWaves>(loss);
    number = group_sum<kWaves>(number);
    if (threadIdx.x == 0) finish(loss, number, a.reduction, a.loss_out, a.reduce_out);
}

// One read and one write; the entries' places are written again, by a thread each, so that the stream has no test for them. Bound by
// memory: 4096 x 131072 bf16 394 us (5.5 TB/s).
template <class T, bool STREAM>
__global__ __launch_bounds__(kThreads) void topk_backward_kernel(TopkArgs a) {
    constexpr int n = Vec<T>::n;
    const int64_t row = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
    const int64_t begin = split * a.chunk, end = min(a.vocab, begin + a.chunk);
    const T* z = static_cast<const T*>(a.logits) + row * a.stride;
    T* out = static_cast<T*>(a.out) + row * a.vocab;
    const RowState st = a.state[row];
    const float g = row_gradient(a.upstream, a.per_row, a.reduce, a.t, st, row);
    if (g == 0.0f) {            // nothing to read
        for (int64_t at = begin + threadIdx.x * n; at < end; at += kThreads * n) {
            if (at + n <= end) store_pack<STREAM>(out + at, Pack<T>{});
            else
                for (int64_t i = at; i < end; ++i) out[i] = T(0);
        }
        return;
    }
    const float slope = st.slope * g;
    const auto grad = [&](T x) { return Vec<T>::put(slope * __builtin_amdgcn_exp2f((Vec<T>::get(x) - st.peak_rest) * a.c)); };
    int64_t first = begin;
    constexpr int64_t kRound = static_cast<int64_t>(kThreads) * n * kUnroll;
    for (; first + kRound <= end; first += kRound) {
        Pack<T> p[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) p[u] = load_pack<STREAM>(z + first + (u * kThreads + threadIdx.x) * n);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
            for (int i = 0; i < n; ++i) p[u].v[i] = grad(p[u].v[i]);
            store_pack<STREAM>(out + first + (u * kThreads + threadIdx.x) * n, p[u]);
        }
    }
    for (int64_t at = first + threadIdx.x * n; at < end; at += kThreads * n) {
        if (at + n <= end) {
            Pack<T> p = *reinterpret_cast<const Pack<T>*>(z + at);
#pragma unroll
            for (int i = 0; i < n; ++i) p.v[i] = grad(p.v[i]);
            *reinterpret_cast<Pack<T>*>(out + at) = p;
        } else {
            for (int64_t i = at; i < end; ++i) out[i] = grad(z[i]);
        }
    }
    stores_done();
    __syncthreads();            // the entries' places are written again
    const int j = threadIdx.x;
    if (j >= a.entries.k) return;
    const int64_t v = a.entries.index[row * a.entries.k + j];
    if (v >= begin && v < end)
        out[v] = Vec<T>::put(g * (st.mass * __builtin_amdgcn_exp2f((Vec<T>::get(z[v]) - st.peak) * a.c) - a.entries.p[row * a.entries.k + j]));
}

template <class... P, class... A>
int launch_with(size_t lds, void (*kernel)(P...), unsigned grid, unsigned block, hipStream_t stream, A... args) {
    std::tuple<P...> held(args...);
    void* params[sizeof...(P)];
    size_t i = 0;
    std::apply([&](auto&... x) { ((params[i++] = &x), ...); }, held);
    return hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3(grid), dim3(block), params, lds, stream) == hipSuccess ? JABAS_OK : JABAS_ERR_LAUNCH;
}
template <class... P, class... A>
int launch(void (*kernel)(P...), unsigned grid, unsigned block, hipStream_t stream, A... args) {
    return launch_with(0, kernel, grid, block, stream, args...);
}

}  // namespace

int launch_teacher(const TeacherArgs& a, hipStream_t stream) {
    return launch(teacher_kernel, static_cast<unsigned>((a.rows + 3) / 4), kThreads, stream, a);
}
int launch_join(const JoinArgs& a, hipStream_t stream) {
    return launch(join_kernel, static_cast<unsigned>((a.rows + kJoinRows - 1) / kJoinRows), kJoinThreads, stream, a);
}
int launch_narrow_join(const JoinArgs& a, hipStream_t stream) {
    return launch(narrow_join_kernel, static_cast<unsigned>(a.rows), kThreads, stream, a);
}
int launch_reduce(const float* row_loss, const RowState* state, int64_t rows, int reduction, float* loss_out, float* reduce, hipStream_t stream) {
    return launch(reduce_kernel, 1, kJoinThreads, stream, row_loss, state, rows, reduction, loss_out, reduce);
}
int launch_live(const LiveArgs& a, hipStream_t stream) { return launch(live_kernel, 1, kJoinThreads, stream, a); }
int launch_down(const float* p, int64_t rows, int32_t k, float* down, hipStream_t stream) {
    return launch(down_kernel, static_cast<unsigned>((rows + 3) / 4), kThreads, stream, p, rows, k, down);
}
int launch_row_grad(const RowGradArgs& a, hipStream_t stream) { return launch(row_grad_kernel, 1, kJoinThreads, stream, a); }
int launch_bias_sum(const float* parts, const int32_t* live, int32_t tile, int64_t stride, int64_t n, void* out, int32_t dtype, hipStream_t stream) {
    return launch(bias_sum_kernel, static_cast<unsigned>((n + kThreads - 1) / kThreads), kThreads, stream, parts, live, tile, stride, n, out, dtype);
}
int launch_zero(void* p, size_t bytes, hipStream_t stream) {
    const size_t n = bytes / 2;
    const size_t blocks = (n + kThreads - 1) / kThreads;
    return launch(zero_kernel, static_cast<unsigned>(blocks < 4096 ? blocks : 4096), kThreads, stream, static_cast<uint16_t*>(p), n);
}
template <class T, bool STREAM>
static int topk_forward(const TopkArgs& a, hipStream_t stream) {
    const size_t lds = static_cast<size_t>((a.chunk + 31) / 32) * 4;
    if (a.splits == 1) {
        const int status = launch_with(lds, topk_row_kernel<T, STREAM>, static_cast<unsigned>(a.rows), kThreads, stream, a);
        return status != JABAS_OK ? status : launch_reduce(a.row_loss, a.state, a.rows, a.reduction, a.loss_out, a.reduce_out, stream);
    }
    const int status = launch_with(lds, topk_split_kernel<T, STREAM>, static_cast<unsigned>(a.rows * a.splits), kThreads, stream, a);
    return status != JABAS_OK ? status : launch(topk_join_kernel<T>, static_cast<unsigned>((a.rows + kThreads / 64 - 1) / (kThreads / 64)), kThreads, stream, a);
}
// Calls that touch more bytes than the last cache holds go past the caches. 6400 x 32317 bf16 (414 MB): forward 117 us through them,
// 111 past them, backward 210 and 183; 2560 x 32317 (165 MB): 51.0 and 57.6, 83.7 and 79.1; 2048 x 32317: 44.5 and 49.5, 50.8 and 65.3.
constexpr int64_t kCacheBytes = int64_t{256} << 20;
static bool streams(const TopkArgs& a, int64_t times) { return times * a.rows * a.vocab > kCacheBytes / (a.dtype == JABAS_F32 ? 4 : 2); }
int launch_topk_forward(const TopkArgs& a, hipStream_t stream) {
    if (a.dtype == JABAS_F32) return streams(a, 1) ? topk_forward<float, true>(a, stream) : topk_forward<float, false>(a, stream);
    return streams(a, 1) ? topk_forward<uint16_t, true>(a, stream) : topk_forward<uint16_t, false>(a, stream);
}
template <class T>
static int topk_backward(const TopkArgs& a, hipStream_t stream) {
    const unsigned grid = static_cast<unsigned>(a.rows * a.splits);
    return streams(a, 2) ? launch(topk_backward_kernel<T, true>, grid, kThreads, stream, a) : launch(topk_backward_kernel<T, false>, grid, kThreads, stream, a);
}
int launch_topk_backward(const TopkArgs& a, hipStream_t stream) {
    return a.dtype == JABAS_F32 ? topk_backward<float>(a, stream) : topk_backward<uint16_t>(a, stream);
}

}  // namespace loss
}  // namespace jabas
