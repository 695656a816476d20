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
static_assert(64 * kEntriesPerLane > JABAS_LOSS_MAX_ENTRIES, "a row's entries fit a wave");

// One wave per row. Entries that name a token twice are one event with both probabilities: the first keeps the sum.
__global__ __launch_bounds__(kThreads) void teacher_kernel(TeacherArgs a) {
    __shared__ int64_t names[kThreads / 64][64 * kEntriesPerLane];
    __shared__ float probs[kThreads / 64][64 * kEntriesPerLane];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / 64) + wave;
    const bool here = row < a.rows;
    int64_t idx[kEntriesPerLane];
    float t[kEntriesPerLane], p[kEntriesPerLane];
    bool is[kEntriesPerLane];
    float peak = -INFINITY, sum = 0.0f;
    bool outside = false;
    for (int i = 0; i < kEntriesPerLane; ++i) {
        const int j = lane + 64 * i;
        const bool valid = here && j < a.k;
        idx[i] = valid ? a.index[row * a.k + j] : -1;
        t[i] = valid ? load_as_float(a.logits, row * a.k + j, a.dtype) : -INFINITY;
        is[i] = idx[i] >= 0 && !(t[i] == -INFINITY);
        outside |= is[i] && idx[i] >= a.vocab;
        if (is[i]) peak = fmaxf(peak, t[i]);
    }
    peak = wave_max(peak);
    outside = __any(outside);
    float norm = 0.0f;
    if (a.lse) {
        norm = here ? a.lse[row] : 0.0f;
    } else {
        for (int i = 0; i < kEntriesPerLane; ++i)
            if (is[i]) sum += expf((t[i] - peak) * a.inv_t);
        norm = logf(wave_sum(sum));
    }
    float logp[kEntriesPerLane];
    for (int i = 0; i < kEntriesPerLane; ++i) {
        logp[i] = a.lse ? t[i] * a.inv_t - norm : (t[i] - peak) * a.inv_t - norm;
        p[i] = is[i] ? expf(logp[i]) : 0.0f;
        names[wave][lane + 64 * i] = is[i] ? idx[i] : -1;
        probs[wave][lane + 64 * i] = p[i];
    }
    __syncthreads();
    float mass = 0.0f, entropy = 0.0f, count = 0.0f;
    for (int i = 0; i < kEntriesPerLane; ++i) {
        const int j = lane + 64 * i;
        if (is[i]) {
            bool first = true, twice = false;
            float all = p[i];
            for (int o = 0; o < a.k; ++o)
                if (o != j && names[wave][o] == idx[i]) {
                    if (o < j) first = false;
                    all += probs[wave][o];
                    twice = true;
                }
            count += 1.0f;
            if (!first) is[i] = false;
            else if (twice) {
                p[i] = all;
                logp[i] = logf(all);
            }
        }
        if (is[i]) {
            mass += p[i];
            if (p[i] != 0.0f) entropy += p[i] * logp[i];
        }
        if (here && j < a.k) {
            a.entry_index[row * a.k + j] = is[i] && !outside ? static_cast<int32_t>(idx[i]) : -1;
            a.entry_p[row * a.k + j] = is[i] ? p[i] : 0.0f;
        }
    }
    mass = wave_sum(mass);
    entropy = wave_sum(entropy);
    count = wave_sum(count);
    if (here && lane == 0) a.row[row] = make_float4(mass, outside ? NAN : entropy, count, 0.0f);
}

constexpr int kJoinThreads = 1024, kJoinRows = 64, kJoinWaves = kJoinThreads / 64;

// 64 rows per workgroup: each wave joins a sixteenth of the vocabulary's tiles with a row per lane, then the waves' results
// are joined, and each wave takes the entries of its rows in turn.
__global__ __launch_bounds__(kJoinThreads) void join_kernel(JoinArgs a) {
    __shared__ float peaks[kJoinWaves][kJoinRows], sums[kJoinWaves][kJoinRows], totals[kJoinWaves][kJoinRows];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kJoinRows, mine = first + lane;
    float peak = -INFINITY, sum = 0.0f, total = 0.0f;
    if (mine < a.rows)
        for (int i = wave; i < a.tiles; i += kJoinWaves) {
            const float2 part = a.partial[static_cast<int64_t>(i) * a.rows + mine];
            const float p = fmaxf(peak, part.x);
            sum = rescale(sum, peak, p, a.c) + rescale(part.y, part.x, p, a.c);
            peak = p;
            if (a.total) total += a.total[static_cast<int64_t>(i) * a.rows + mine];
        }
    peaks[wave][lane] = peak;
    sums[wave][lane] = sum;
    totals[wave][lane] = total;
    __syncthreads();
    if (wave == 0) {
        for (int i = 1; i < kJoinWaves; ++i) {
            const float p = fmaxf(peak, peaks[i][lane]);
            sum = rescale(sum, peak, p, a.c) + rescale(sums[i][lane], peaks[i][lane], p, a.c);
            peak = p;
            total += totals[i][lane];
        }
        peaks[0][lane] = peak;
        sums[0][lane] = sum;
        totals[0][lane] = total;
    }
    __syncthreads();
    if (!a.entries.index) {
        if (wave != 0 || mine >= a.rows) return;
        const int64_t label = a.entries.target[mine];
        RowState st = {0.0f, 0.0f, 0.0f, 0.0f};
        float loss = 0.0f;
        if (label != a.entries.ignore_index) {
            st.peak_rest = st.peak = peak;
            st.slope = st.mass = 1.0f / sum;
            const float e = a.smoothing;
            if (label < 0 || label >= a.vocab) {
                loss = st.slope = st.mass = NAN;
            } else {
                loss = logf(sum) + (1.0f - e) * (peak - a.entry_logit[mine]);
                if (e != 0.0f) loss += e * (peak - total / static_cast<float>(a.vocab));
            }
        }
        a.state[mine] = st;
        a.row_loss[mine] = loss;
        return;
    }
    for (int r = wave; r < kJoinRows && first + r < a.rows; r += kJoinWaves) {
        const int64_t row = first + r;
        const float rest_peak = peaks[0][r], rest_sum = sums[0][r];
        const float4 teacher = a.teacher_row[row];
        float top = rest_peak;
        for (int j = lane; j < a.entries.k; j += 64)
            if (a.entries.index[row * a.entries.k + j] >= 0) top = fmaxf(top, a.entry_logit[row * a.entries.k + j]);
        top = wave_max(top);
        float held = 0.0f;
        for (int j = lane; j < a.entries.k; j += 64)
            if (a.entries.index[row * a.entries.k + j] >= 0) {
                const float z = a.entry_logit[row * a.entries.k + j];
                if (z != -INFINITY) held += __builtin_amdgcn_exp2f((z - top) * a.c);
            }
        held = wave_sum(held);
        const float all = held + rescale(rest_sum, rest_peak, top, a.c), log_all = logf(all);
        float cross = 0.0f;
        for (int j = lane; j < a.entries.k; j += 64)
            if (a.entries.index[row * a.entries.k + j] >= 0) {
                const float p = a.entries.p[row * a.entries.k + j];
                if (p != 0.0f) cross += p * ((a.entry_logit[row * a.entries.k + j] - top) * a.inv_t - log_all);
            }
        cross = wave_sum(cross);
        if (lane) continue;
        RowState st = {0.0f, 0.0f, 0.0f, 0.0f};
        float loss = 0.0f;
        if (teacher.z != 0.0f) {
            const bool others = rest_sum != 0.0f;
            float left = a.has_rest && others ? 1.0f - teacher.x : 0.0f;
            if (left < 0.0f) left = 0.0f;
            const float mass = teacher.x + left;
            float rest = 0.0f, share = 0.0f;    // of the student: log R and R
            if (others) {
                rest = (rest_peak - top) * a.inv_t + logf(rest_sum) - log_all;
                share = expf(rest);
            }
            loss = teacher.y - cross;
            if (left != 0.0f) loss += left * (logf(left) - rest);
            loss *= a.t * a.t;
            st.peak_rest = others ? rest_peak : 0.0f;
            st.slope = others ? (mass * share - left) / rest_sum : 0.0f;
            st.peak = top;
            st.mass = mass / all;
            if (teacher.y != teacher.y) st.slope = st.mass = NAN;       // a name outside the vocabulary
        }
        a.state[row] = st;
        a.row_loss[row] = loss;
    }
}

__device__ inline bool counts(const RowState& st) { return !(st.slope == 0.0f && st.mass == 0.0f); }

__global__ __launch_bounds__(kJoinThreads) void reduce_kernel(const float* row_loss, const RowState* state, int64_t rows, int reduction,
                                                              float* loss_out, float* reduce) {
    __shared__ double sums[kJoinWaves], numbers[kJoinWaves];
    double sum = 0.0, number = 0.0;
    for (int64_t i = threadIdx.x; i < rows; i += kJoinThreads) {
        const float loss = row_loss[i];
        sum += loss;
        number += counts(state[i]) ? 1.0 : 0.0;
        if (reduction == JABAS_LOSS_NONE) loss_out[i] = loss;
    }
    sum = wave_sum(sum);
    number = wave_sum(number);
    if ((threadIdx.x & 63) == 0) {
        sums[threadIdx.x >> 6] = sum;
        numbers[threadIdx.x >> 6] = number;
    }
    __syncthreads();
    if (threadIdx.x) return;
    for (int i = 1; i < kJoinWaves; ++i) {
        sum += sums[i];
        number += numbers[i];
    }
    const double share = reduction == JABAS_LOSS_MEAN && number > 0.0 ? 1.0 / number : 1.0;
    *reduce = static_cast<float>(share);
    if (reduction != JABAS_LOSS_NONE) *loss_out = static_cast<float>(sum * share);
}

__global__ __launch_bounds__(kJoinThreads) void row_grad_kernel(const float* upstream, int per_row, const float* reduce, float t, const RowState* state,
                                                                int64_t rows, float* grad, float* ratio, float* peak) {
    __shared__ float peaks[kJoinWaves];
    const float share = *reduce * t;
    float top = 0.0f;
    bool bad = false;
    for (int64_t i = threadIdx.x; i < rows; i += kJoinThreads) {
        const float g = counts(state[i]) ? upstream[per_row ? i : 0] * share : 0.0f;
        grad[i] = g;
        bad |= !(fabsf(g) < INFINITY);
        top = fmaxf(top, fabsf(g));
    }
    top = wave_max(top);
    if (__any(bad)) top = INFINITY;
    if ((threadIdx.x & 63) == 0) peaks[threadIdx.x >> 6] = top;
    __syncthreads();
    for (int i = 0; i < kJoinWaves; ++i) top = fmaxf(top, peaks[i]);
    // rows of a gradient that is not finite make everything that sums over rows NaN: the ratio says 1 for all that count
    const bool whole = top < INFINITY;
    if (threadIdx.x == 0) *peak = whole ? top : NAN;
    for (int64_t i = threadIdx.x; i < rows; i += kJoinThreads) {
        const float g = counts(state[i]) ? upstream[per_row ? i : 0] * share : 0.0f;
        ratio[i] = g == 0.0f ? 0.0f : whole ? g / top : 1.0f;
    }
}

__global__ __launch_bounds__(kThreads) void bias_sum_kernel(const float* parts, int32_t tiles, int64_t stride, int64_t n, void* out, int32_t dtype) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= n) return;
    float sum = 0.0f;
    for (int t = 0; t < tiles; ++t) sum += parts[t * stride + i];
    if (dtype == JABAS_F32) static_cast<float*>(out)[i] = sum;
    else static_cast<uint16_t*>(out)[i] = to_bf16(sum);
}

__global__ __launch_bounds__(kThreads) void zero_kernel(uint16_t* p, size_t n) {
    for (size_t i = static_cast<size_t>(blockIdx.x) * kThreads + threadIdx.x; i < n; i += static_cast<size_t>(gridDim.x) * kThreads) p[i] = 0;
}

// ------------------------------------------------------------------ logits in hand

constexpr int kMaskTokens = 32768;      // tokens of a split at most: a bit for each in LDS

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

// Bits of the split's tokens that are entries of the row.
__device__ inline void build_mask(const Entries& en, int64_t row, int64_t begin, int64_t end, uint32_t* mask) {
    const int words = static_cast<int>((end - begin + 31) / 32);
    for (int i = threadIdx.x; i < words; i += kThreads) mask[i] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < en.k; j += kThreads) {
        const int64_t v = static_cast<int64_t>(en.index[row * en.k + j]) - begin;
        if (v >= 0 && v < end - begin) atomicOr(&mask[v >> 5], 1u << (v & 31));
    }
    __syncthreads();
}

template <class T>
__global__ __launch_bounds__(kThreads) void topk_forward_kernel(TopkArgs a) {
    __shared__ uint32_t mask[kMaskTokens / 32];
    __shared__ float peaks[kThreads / 64], sums[kThreads / 64];
    constexpr int n = Vec<T>::n;
    const int64_t row = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
    const int64_t begin = split * a.chunk, end = min(a.vocab, begin + a.chunk);
    const T* z = static_cast<const T*>(a.logits) + row * a.stride;
    build_mask(a.entries, row, begin, end, mask);
    for (int j = threadIdx.x; j < a.entries.k; j += kThreads) {
        const int64_t v = a.entries.index[row * a.entries.k + j];
        if (v >= begin && v < end) a.entry_logit[row * a.entries.k + j] = Vec<T>::get(z[v]);
    }
    float peak = -INFINITY, sum = 0.0f;
    for (int64_t at = begin + threadIdx.x * n; at < end; at += kThreads * n) {
        float x[n];
        if (at + n <= end) {
            const Pack<T> p = *reinterpret_cast<const Pack<T>*>(z + at);
#pragma unroll
            for (int i = 0; i < n; ++i) x[i] = Vec<T>::get(p.v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < n; ++i) x[i] = at + i < end ? Vec<T>::get(z[at + i]) : -INFINITY;
        }
        const int off = static_cast<int>(at - begin);
        const uint32_t hits = mask[off >> 5] >> (off & 31);     // n divides 32: one word holds them all
        float top = peak;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            if ((hits >> i) & 1) x[i] = -INFINITY;
            top = fmaxf(top, x[i]);
        }
        const float base = top == -INFINITY ? 0.0f : top;
        sum = rescale(sum, peak, base, a.c);
#pragma unroll
        for (int i = 0; i < n; ++i) sum += __builtin_amdgcn_exp2f((x[i] - base) * a.c);
        peak = top;
    }
    const float top = wave_max(peak);
    sum = wave_sum(rescale(sum, peak, top, a.c));
    if ((threadIdx.x & 63) == 0) {
        peaks[threadIdx.x >> 6] = top;
        sums[threadIdx.x >> 6] = sum;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        float p = peaks[0], s = sums[0];
        for (int i = 1; i < kThreads / 64; ++i) {
            const float q = fmaxf(p, peaks[i]);
            s = rescale(s, p, q, a.c) + rescale(sums[i], peaks[i], q, a.c);
            p = q;
        }
        a.partial[split * a.rows + row] = make_float2(p, s);
    }
}

template <class T>
__global__ __launch_bounds__(kThreads) void topk_backward_kernel(TopkArgs a) {
    constexpr int n = Vec<T>::n;
    const int64_t row = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
    const int64_t begin = split * a.chunk, end = min(a.vocab, begin + a.chunk);
    const T* z = static_cast<const T*>(a.logits) + row * a.stride;
    T* out = static_cast<T*>(a.out) + row * a.vocab;
    const RowState st = a.state[row];
    const float g = a.row_grad[row];
    const bool live = counts(st) && g != 0.0f;
    const float slope = st.slope * g;
    for (int64_t at = begin + threadIdx.x * n; at < end; at += kThreads * n) {
        if (at + n <= end) {
            Pack<T> p = *reinterpret_cast<const Pack<T>*>(z + at);
#pragma unroll
            for (int i = 0; i < n; ++i)
                p.v[i] = Vec<T>::put(live ? slope * __builtin_amdgcn_exp2f((Vec<T>::get(p.v[i]) - st.peak_rest) * a.c) : 0.0f);
            *reinterpret_cast<Pack<T>*>(out + at) = p;
        } else {
            for (int64_t i = at; i < end; ++i)
                out[i] = Vec<T>::put(live ? slope * __builtin_amdgcn_exp2f((Vec<T>::get(z[i]) - st.peak_rest) * a.c) : 0.0f);
        }
    }
    if (!live) return;
    __syncthreads();            // the entries' places are written again: behind the stores above, which the barrier waits for
    for (int j = threadIdx.x; j < a.entries.k; j += kThreads) {
        const int64_t v = a.entries.index[row * a.entries.k + j];
        if (v >= begin && v < end)
            out[v] = Vec<T>::put(g * (st.mass * __builtin_amdgcn_exp2f((Vec<T>::get(z[v]) - st.peak) * a.c) - a.entries.p[row * a.entries.k + j]));
    }
}

inline int launched() { return hipGetLastError() == hipSuccess ? JABAS_OK : JABAS_ERR_LAUNCH; }

template <class... P, class... A>
int launch(void (*kernel)(P...), unsigned grid, unsigned block, hipStream_t stream, A... args) {
    std::tuple<P...> held(args...);
    void* params[sizeof...(P)];
    size_t i = 0;
    std::apply([&](auto&... x) { ((params[i++] = &x), ...); }, held);
    return hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3(grid), dim3(block), params, 0, stream) == hipSuccess ? JABAS_OK : JABAS_ERR_LAUNCH;
}

}  // namespace

int launch_teacher(const TeacherArgs& a, hipStream_t stream) {
    return launch(teacher_kernel, static_cast<unsigned>((a.rows + 3) / 4), kThreads, stream, a);
}
int launch_join(const JoinArgs& a, hipStream_t stream) {
    return launch(join_kernel, static_cast<unsigned>((a.rows + kJoinRows - 1) / kJoinRows), kJoinThreads, stream, a);
}
int launch_reduce(const float* row_loss, const RowState* state, int64_t rows, int reduction, float* loss_out, float* reduce, hipStream_t stream) {
    return launch(reduce_kernel, 1, kJoinThreads, stream, row_loss, state, rows, reduction, loss_out, reduce);
}
int launch_row_grad(const float* upstream, int per_row, const float* reduce, float t, const RowState* state, int64_t rows,
                    float* grad, float* ratio, float* peak, hipStream_t stream) {
    return launch(row_grad_kernel, 1, kJoinThreads, stream, upstream, per_row, reduce, t, state, rows, grad, ratio, peak);
}
int launch_bias_sum(const float* parts, int32_t tiles, int64_t stride, int64_t n, void* out, int32_t dtype, hipStream_t stream) {
    return launch(bias_sum_kernel, static_cast<unsigned>((n + kThreads - 1) / kThreads), kThreads, stream, parts, tiles, stride, n, out, dtype);
}
int launch_zero(void* p, size_t bytes, hipStream_t stream) {
    const size_t n = bytes / 2;
    const size_t blocks = (n + kThreads - 1) / kThreads;
    return launch(zero_kernel, static_cast<unsigned>(blocks < 4096 ? blocks : 4096), kThreads, stream, static_cast<uint16_t*>(p), n);
}
int launch_topk_forward(const TopkArgs& a, hipStream_t stream) {
    const unsigned grid = static_cast<unsigned>(a.rows * a.splits);
    return a.dtype == JABAS_F32 ? launch(topk_forward_kernel<float>, grid, kThreads, stream, a) : launch(topk_forward_kernel<uint16_t>, grid, kThreads, stream, a);
}
int launch_topk_backward(const TopkArgs& a, hipStream_t stream) {
    const unsigned grid = static_cast<unsigned>(a.rows * a.splits);
    return a.dtype == JABAS_F32 ? launch(topk_backward_kernel<float>, grid, kThreads, stream, a) : launch(topk_backward_kernel<uint16_t>, grid, kThreads, stream, a);
}

}  // namespace loss
}  // namespace jabas
