// Losses of few rows (kNarrowRows at most) from hidden states and weight: what counts is to read the weight once for the logits, once for the
// hidden states' gradient, and to write its gradient once. Nothing is copied or laid out first: fragments come from memory as they lie, at
// any alignment, and there is no LDS in the inner loops, so nothing waits for a barrier.
//
// Logits: 32 tokens a workgroup, the four waves take the width's blocks of 64 in turn. Lane (r, half) holds 32 consecutive elements of
// token r: which elements of the inner axis meet in one matrix instruction is free as long as both operands agree, so each lane reads
// whole 64 or 128 bytes. bf16 through 32x32x16, fp32 through 32x32x2: its rate (16 bytes of weight per clock and CU at 32 rows) is above
// what memory gives.
// It takes 21 us for 66 MB of weight and one row (3.2 TB/s), 280 us for 1.07 GB and eight (3.8 TB/s): a load of a wave touches 32 rows, and
// what it would take to load whole lines through LDS gives a tenth at most.
// Gradients: dz in the units of the result, fp32, or for bf16 two bf16 planes (16 bits, where the results have 8), so that the row
// gradients keep their bits whatever their size. fp32's products take 32x32x2, whose lane holds one element of the inner axis, so that
// operands whose rows are that axis need no transposing; bf16's take 32x32x16 with four features of eight rows turned about in a lane's
// registers. 8 rows, 131072 x 4096: dX 230 us with bf16 (4.7 TB/s), 525 with fp32 (4.1 TB/s), dW 300 and 457 us; with 32x32x2 and checked
// loads for bf16 too both took 1081 us, 546 now. What bounds them is how much a CU has on its way, so two
// workgroups have to fit one, with 33 to 64 rows too, though registers run out there (120 bytes a lane with fp32, 260 with bf16 go to scratch
// memory): 64 x 32317 x 1024 fp32 374 us with one, 320 with two, 64 x 131072 x 4096 4360 and 3805.
// The logits' kernels do so with bf16 (64 x 16000 x 768 116 and 104 us); fp32's would have to spill (64 x 32317 x 1024 forward 93 and 120 us), so that
// one wave a SIMD is left with 33 to 64 rows.
#include "loss_internal.h"

namespace jabas {
namespace loss {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;

__device__ inline uint16_t to_bf16(float x) {
    const uint32_t u = __float_as_uint(x);
    if ((u & 0x7fffffffu) > 0x7f800000u) return static_cast<uint16_t>((u >> 16) | 0x40);
    return static_cast<uint16_t>((u + 0x7fffu + ((u >> 16) & 1)) >> 16);
}
template <class T> __device__ inline float widen(T x);
template <> __device__ inline float widen<float>(float x) { return x; }
template <> __device__ inline float widen<uint16_t>(uint16_t x) { return __uint_as_float(static_cast<uint32_t>(x) << 16); }
template <class T> __device__ inline T narrow(float x);
template <> __device__ inline float narrow<float>(float x) { return x; }
template <> __device__ inline uint16_t narrow<uint16_t>(float x) { return to_bf16(x); }

// N elements at any element
template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Some {
    T v[N];
};

// 32 consecutive elements of a row from column c on, zeros past the end.
template <class T>
struct Run {
    T v[32];
    __device__ void load(const T* row, int c, int cols) {
        constexpr int n = 16 / sizeof(T);
        if (c + 32 <= cols) {
#pragma unroll
            for (int i = 0; i < 32; i += n) {
                const Some<T, n> x = *reinterpret_cast<const Some<T, n>*>(row + c + i);
#pragma unroll
                for (int j = 0; j < n; ++j) v[i + j] = x.v[j];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = c + i < cols ? row[c + i] : T(0);
        }
    }
};

__device__ inline f32x16 multiply(const Run<float>& a, const Run<float>& b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 32; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[i], b.v[i], c, 0, 0, 0);
    return c;
}
__device__ inline f32x16 multiply(const Run<uint16_t>& a, const Run<uint16_t>& b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
        bf16x8 x, y;
        __builtin_memcpy(&x, a.v + i, 16);
        __builtin_memcpy(&y, b.v + i, 16);
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
    }
    return c;
}

__device__ inline int block_m(int e) { return 8 * (e >> 2) + 4 * ((threadIdx.x & 63) >> 5) + (e & 3); }

constexpr int kTokens = 32, kPitch = kTokens + 1;

// The logits of the workgroup's tokens into zs[row][token]; part: [3][RB * 32][kPitch] of the other waves' shares.
template <class T, int RB>
__device__ inline void narrow_logits(const NarrowArgs& a, int64_t first, float (*zs)[kPitch], float (*part)[RB * 32][kPitch]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, half = lane >> 5;
    const T* w = static_cast<const T*>(a.w) + min(first + r, a.vocab - 1) * a.w_stride;
    const T* x[RB];
    f32x16 acc[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        x[b] = static_cast<const T*>(a.x) + static_cast<int64_t>(min(b * 32 + r, a.rows - 1)) * a.x_stride;
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[b][e] = 0.0f;
    }
    Run<T> fw[2], fx[2][RB];
    const auto load = [&](int at, Run<T>& f, Run<T> (&g)[RB]) {
        f.load(w, at + half * 32, a.width);
#pragma unroll
        for (int b = 0; b < RB; ++b) g[b].load(x[b], at + half * 32, a.width);
    };
    int at = wave * 64;
    if (at < a.width) load(at, fw[0], fx[0]);
    for (; at < a.width; at += 512) {
        if (at + 256 < a.width) load(at + 256, fw[1], fx[1]);
#pragma unroll
        for (int b = 0; b < RB; ++b) acc[b] = multiply(fw[0], fx[0][b], acc[b]);
        if (at + 256 >= a.width) break;
        if (at + 512 < a.width) load(at + 512, fw[0], fx[0]);
#pragma unroll
        for (int b = 0; b < RB; ++b) acc[b] = multiply(fw[1], fx[1][b], acc[b]);
    }
    if (wave)
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) part[wave - 1][b * 32 + r][block_m(e)] = acc[b][e];
    __syncthreads();
    if (wave == 0)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int m = block_m(e);
            const float bias = a.bias && first + m < a.vocab ? widen(static_cast<const T*>(a.bias)[first + m]) : 0.0f;
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                const int n = b * 32 + r;
                zs[n][m] = acc[b][e] + part[0][n][m] + part[1][n][m] + part[2][n][m] + bias;
            }
        }
    __syncthreads();
}

template <class T, int RB, bool TEACHER>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? 2 : 1) void narrow_forward_kernel(NarrowArgs a) {
    constexpr int R = RB * 32, kGroups = kThreads / R, kEach = kTokens / kGroups;
    __shared__ float zs[R][kPitch], part[3][R][kPitch];
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kTokens;
    const int here = static_cast<int>(min(a.vocab - first, static_cast<int64_t>(kTokens)));
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.ticket = 0;
    narrow_logits<T, RB>(a, first, zs, part);
    if (TEACHER) {
        const int k = a.entries.k;
        for (int i = threadIdx.x >> 6; i < a.rows; i += kThreads / 64)
            for (int j = threadIdx.x & 63; j < k; j += 64) {
                const int64_t v = a.entries.index[static_cast<int64_t>(i) * k + j] - first;
                if (v < 0 || v >= here) continue;
                a.entry_logit[static_cast<int64_t>(i) * k + j] = zs[i][v];
                zs[i][v] = -INFINITY;       // entries join their row later, each by itself
            }
        __syncthreads();
    }
    // row n, tokens [group * kEach, + kEach)
    const int n = threadIdx.x % R, group = threadIdx.x / R;
    const int64_t label = !TEACHER && n < a.rows ? a.entries.target[n] - first : -1;
    float z[kEach], peak = -INFINITY, sum = 0.0f, total = 0.0f;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int m = group * kEach + i;
        z[i] = zs[n][m];
        if (m >= here) z[i] = -INFINITY;
        else total += z[i];
        if (label == m && m < here) a.entry_logit[n] = z[i];
        peak = fmaxf(peak, z[i]);
    }
    const float base = peak == -INFINITY ? 0.0f : peak;
#pragma unroll
    for (int i = 0; i < kEach; ++i) sum += __builtin_amdgcn_exp2f((z[i] - base) * a.c);
    float* merge = &part[0][0][0];
    __syncthreads();
    merge[(group * 3 + 0) * R + n] = peak;
    merge[(group * 3 + 1) * R + n] = sum;
    merge[(group * 3 + 2) * R + n] = total;
    __syncthreads();
    if (group || n >= a.rows) return;
    float p = -INFINITY, s = 0.0f, t = 0.0f;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) p = fmaxf(p, merge[i * 3 * R + n]);
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
        const float more = merge[(i * 3 + 1) * R + n];
        if (more != 0.0f) s += more * __builtin_amdgcn_exp2f((merge[i * 3 * R + n] - p) * a.c);
        t += merge[(i * 3 + 2) * R + n];
    }
    const int64_t tile = static_cast<int64_t>(n) * gridDim.x + blockIdx.x;
    a.partial[tile] = make_float2(p, s);
    if (a.total) a.total[tile] = t;
}

// bf16 calls: dz as two bf16 planes, [plane][row][token] for dX and [plane][token][row] for dW.
template <int R>
struct Planes {
    uint16_t *rows, *tokens;
    int64_t plane;
    __device__ explicit Planes(const NarrowArgs& a) : rows(reinterpret_cast<uint16_t*>(a.dz)), plane(R * a.dz_stride) { tokens = rows + 2 * plane; }
};
// x in 16 bits, and what that leaves in the upper half.
__device__ inline uint32_t split(float x) {
    const uint32_t hi = to_bf16(x);
    const float left = x - widen<uint16_t>(static_cast<uint16_t>(hi));
    return hi | (fabsf(left) < INFINITY ? static_cast<uint32_t>(to_bf16(left)) << 16 : 0);      // not finite: the first plane says it
}

// The row gradient of n; 0 for rows that do not count.
__device__ inline float row_gradient(const NarrowArgs& a, int n) {
    if (n >= a.rows) return 0.0f;
    const RowState st = a.state[n];
    return st.slope == 0.0f && st.mass == 0.0f ? 0.0f : a.upstream[a.per_row ? n : 0] * (*a.reduce * a.t);
}

template <class T, int RB, bool TEACHER>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? 2 : 1) void narrow_backward_kernel(NarrowArgs a) {
    constexpr int R = RB * 32;
    __shared__ float zs[R][kPitch], part[3][R][kPitch], grad[R];
    __shared__ RowState states[R];
    const int64_t from = static_cast<int64_t>(blockIdx.x) * kTokens, first = a.first + from;
    const int here = static_cast<int>(min(a.vocab - first, static_cast<int64_t>(kTokens)));
    if (threadIdx.x < R) {
        grad[threadIdx.x] = row_gradient(a, threadIdx.x);
        states[threadIdx.x] = static_cast<int>(threadIdx.x) < a.rows ? a.state[threadIdx.x] : RowState{0.0f, 0.0f, 0.0f, 0.0f};
    }
    narrow_logits<T, RB>(a, first, zs, part);
    float (*ds)[kPitch] = part[0];
    for (int i = threadIdx.x; i < R * kTokens; i += kThreads) {
        const int n = i / kTokens, m = i % kTokens;
        const RowState st = states[n];
        float d = st.slope * __builtin_amdgcn_exp2f((zs[n][m] - st.peak_rest) * a.c) - a.uniform;
        if (!TEACHER && n < a.rows && a.entries.target[n] - first == m) d -= a.hit;
        ds[n][m] = grad[n] == 0.0f || m >= here ? 0.0f : d * grad[n];
    }
    __syncthreads();
    if (TEACHER) {
        const int k = a.entries.k;
        for (int n = threadIdx.x >> 6; n < a.rows; n += kThreads / 64)
            for (int j = threadIdx.x & 63; j < k; j += 64) {
                const int64_t at = static_cast<int64_t>(n) * k + j, v = a.entries.index[at] - first;
                if (v < 0 || v >= here || grad[n] == 0.0f) continue;
                ds[n][v] = (states[n].mass * __builtin_amdgcn_exp2f((zs[n][v] - states[n].peak) * a.c) - a.entries.p[at]) * grad[n];
            }
        __syncthreads();
    }
    if (a.d_bias && static_cast<int>(threadIdx.x) < here) {
        float s = 0.0f;
        for (int n = 0; n < a.rows; ++n) s += ds[n][threadIdx.x];
        static_cast<T*>(a.d_bias)[first + threadIdx.x] = narrow<T>(s);
    }
    if (!a.dz) return;
    if constexpr (sizeof(T) == 2) {
        Planes<R> p(a);
        for (int i = threadIdx.x; i < R * kTokens; i += kThreads) {
            const int n = i / kTokens, m = i % kTokens;
            const uint32_t v = split(ds[n][m]);
            p.rows[n * a.dz_stride + from + m] = static_cast<uint16_t>(v);
            p.rows[p.plane + n * a.dz_stride + from + m] = static_cast<uint16_t>(v >> 16);
        }
        for (int i = threadIdx.x; i < R * kTokens; i += kThreads) {
            const int m = i / R, n = i % R;
            const uint32_t v = split(ds[n][m]);
            p.tokens[(from + m) * R + n] = static_cast<uint16_t>(v);
            p.tokens[p.plane + (from + m) * R + n] = static_cast<uint16_t>(v >> 16);
        }
    } else {
        for (int i = threadIdx.x; i < R * kTokens; i += kThreads) {
            const int n = i / kTokens, m = i % kTokens;
            a.dz[n * a.dz_stride + from + m] = ds[n][m];
        }
    }
}

// Four consecutive elements of a row from column c on, zeros past the end.
__device__ inline f32x4 load_four(const float* row, int c, int cols) {
    f32x4 v;
    if (c + 4 <= cols) {
        const Some<float, 4> x = *reinterpret_cast<const Some<float, 4>*>(row + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = x.v[i];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = c + i < cols ? row[c + i] : 0.0f;
    }
    return v;
}
template <class T>
__device__ inline void store_four(T* row, int c, int cols, f32x4 v) {
    if (c + 4 <= cols) {
        Some<T, 4> x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x.v[i] = narrow<T>(v[i]);
        *reinterpret_cast<Some<T, 4>*>(row + c) = x;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i < cols) row[c + i] = narrow<T>(v[i]);
    }
}

// dW of 32 tokens, fp32: the sum over rows is the inner axis, two at a time; the waves take 128 features in turn.
template <int RB>
__device__ inline void narrow_weight_fp32(const NarrowArgs& a, int64_t unit) {
    constexpr int R = RB * 32;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, half = lane >> 5;
    const int64_t from = unit * kTokens, first = a.first + from;
    float d[R / 2];
    uint64_t live = 0;      // rows that count: the hidden states of others are zeros whatever they hold
#pragma unroll
    for (int i = 0; i < R / 2; ++i) d[i] = a.dz[(2 * i + half) * a.dz_stride + from + r];
    live = __ballot(row_gradient(a, lane) != 0.0f);
    for (int h = wave * 128; h < a.width; h += 512) {
        f32x16 acc[4];
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[c][e] = 0.0f;
#pragma unroll
        for (int i = 0; i < R / 2; ++i) {
            if (2 * i >= a.rows) break;
            const int n = 2 * i + half;
            f32x4 x = load_four(static_cast<const float*>(a.x) + static_cast<int64_t>(min(n, a.rows - 1)) * a.x_stride, h + 4 * r, a.width);
            if (!((live >> n) & 1)) x = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] = __builtin_amdgcn_mfma_f32_32x32x2f32(d[i], x[c], acc[c], 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int64_t v = first + block_m(e);
            if (v < a.vocab) store_four(static_cast<float*>(a.d_weight) + v * a.width, h + 4 * r, a.width, f32x4{acc[0][e], acc[1][e], acc[2][e], acc[3][e]});
        }
    }
}

// bf16's products take 32x32x16, whose operands hold eight elements of the inner axis a lane: F consecutive features of eight rows (of the
// weight or of the hidden states), turned about in registers, are the operands of F columns of the result each.
constexpr int F = 4;
struct Turned {
    uint32_t v[F][4];
    __device__ explicit Turned(const Some<uint16_t, F> (&x)[8]) {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            uint32_t even[F / 2], odd[F / 2];
            __builtin_memcpy(even, &x[2 * p], 2 * F);
            __builtin_memcpy(odd, &x[2 * p + 1], 2 * F);
#pragma unroll
            for (int c = 0; c < F; ++c) v[c][p] = __builtin_amdgcn_perm(odd[c / 2], even[c / 2], c & 1 ? 0x07060302u : 0x05040100u);
        }
    }
    __device__ bf16x8 operator[](int c) const {
        bf16x8 x;
        __builtin_memcpy(&x, v[c], 16);
        return x;
    }
};
__device__ inline Some<uint16_t, F> load_some(const uint16_t* row, int c, int cols) {
    if (c + F <= cols) return *reinterpret_cast<const Some<uint16_t, F>*>(row + c);
    Some<uint16_t, F> x;
#pragma unroll
    for (int i = 0; i < F; ++i) x.v[i] = c + i < cols ? row[c + i] : 0;
    return x;
}
__device__ inline bf16x8 load_eight(const uint16_t* p) { return *reinterpret_cast<const bf16x8*>(p); }

// dW of 32 tokens: the rows are the inner axis, 16 at a time; the waves take 32 F features in turn.
template <int RB>
__device__ inline void narrow_weight_bf16(const NarrowArgs& a, int64_t unit) {
    constexpr int R = RB * 32;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, half = lane >> 5;
    const int64_t from = unit * kTokens, first = a.first + from;
    const Planes<R> p(a);
    bf16x8 d[R / 16][2];
#pragma unroll
    for (int k = 0; k < R / 16; ++k)
#pragma unroll
        for (int q = 0; q < 2; ++q) d[k][q] = load_eight(p.tokens + q * p.plane + (from + r) * R + k * 16 + half * 8);
    const uint64_t live = __ballot(row_gradient(a, lane) != 0.0f);     // rows that count: the hidden states of others are zeros whatever they hold
    for (int h = wave * 32 * F; h < a.width; h += 128 * F) {
        const bool whole = h + 32 * F <= a.width;
        f32x16 acc[F];
#pragma unroll
        for (int c = 0; c < F; ++c)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[c][e] = 0.0f;
#pragma unroll
        for (int k = 0; k < R / 16; ++k) {
            if (k * 16 >= a.rows) break;
            Some<uint16_t, F> x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint16_t* row = static_cast<const uint16_t*>(a.x) + static_cast<int64_t>(min(k * 16 + half * 8 + j, a.rows - 1)) * a.x_stride;
                x[j] = whole ? *reinterpret_cast<const Some<uint16_t, F>*>(row + h + F * r) : load_some(row, h + F * r, a.width);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (!((live >> (k * 16 + half * 8 + j)) & 1)) x[j] = Some<uint16_t, F>{};
            const Turned b(x);
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int c = 0; c < F; ++c) acc[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(d[k][q], b[c], acc[c], 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int64_t v = first + block_m(e);
            if (v >= a.vocab) continue;
            uint16_t* out = static_cast<uint16_t*>(a.d_weight) + v * a.width;
            Some<uint16_t, F> y;
#pragma unroll
            for (int c = 0; c < F; ++c) y.v[c] = to_bf16(acc[c][e]);
            if (h + F * r + F <= a.width) *reinterpret_cast<Some<uint16_t, F>*>(out + h + F * r) = y;
            else
#pragma unroll
                for (int c = 0; c < F; ++c)
                    if (h + F * r + c < a.width) out[h + F * r + c] = y.v[c];
        }
    }
}

// Four features of the sums of the workgroup's waves, a block of 32 rows: merge[wave - 1][32 rows][128], then to where they go.
template <class T>
__device__ inline void narrow_merge(const NarrowArgs& a, int b, int split, int feature, const f32x16& x, const f32x16& y, const f32x16& z, const f32x16& w, float* merge) {
    const int wave = threadIdx.x >> 6, r = threadIdx.x & 31;
    __syncthreads();
    if (wave)
#pragma unroll
        for (int e = 0; e < 16; ++e) *reinterpret_cast<f32x4*>(merge + ((wave - 1) * 32 + block_m(e)) * 128 + 4 * r) = f32x4{x[e], y[e], z[e], w[e]};
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int m = block_m(e), n = b * 32 + m;
        f32x4 v = {x[e], y[e], z[e], w[e]};
#pragma unroll
        for (int i = 0; i < 3; ++i) v += *reinterpret_cast<const f32x4*>(merge + (i * 32 + m) * 128 + 4 * r);
        if (n >= a.rows) continue;
        if (a.part) {
            if (feature >= a.width) continue;
            f32x4* sum = reinterpret_cast<f32x4*>(a.part + split * a.part_plane + n * a.part_stride + feature);
            *sum = a.add ? *sum + v : v;
        } else {
            store_four(static_cast<T*>(a.d_hidden) + static_cast<int64_t>(n) * a.width, feature, a.width, v);
        }
    }
}

// dX of 32 F features over a range of tokens: 16 at a time; the waves take blocks of 32 tokens in turn.
template <int RB>
__device__ inline void narrow_hidden_bf16(const NarrowArgs& a, int64_t unit, float* merge) {
    constexpr int R = RB * 32;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, half = lane >> 5;
    const int slices = (a.width + 32 * F - 1) / (32 * F), h = static_cast<int>(unit % slices) * 32 * F, split = static_cast<int>(unit / slices);
    const int64_t begin = split * a.each, end = min(begin + a.each, a.tokens);
    const Planes<R> p(a);
    f32x16 acc[RB][F];
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int c = 0; c < F; ++c)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[b][c][e] = 0.0f;
    // Whole blocks and slices take their loads without a check, all at once.
    const bool whole = h + 32 * F <= a.width && a.first + end <= a.vocab && end - begin == a.each;
    for (int64_t v = begin + wave * 32; v < end; v += 128) {
        Some<uint16_t, F> w[2][8];
        const uint16_t* row = static_cast<const uint16_t*>(a.w) + (a.first + v + half * 8) * a.w_stride + h + F * r;
        if (whole) {
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j / 8][j % 8] = *reinterpret_cast<const Some<uint16_t, F>*>(row + (j / 8 * 16 + j % 8) * a.w_stride);
        } else {
#pragma unroll 1
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) {       // tokens past the end: the last one again, against a zero of dz
                    const int64_t at = min(a.first + v + s * 16 + half * 8 + j, a.vocab - 1);
                    const Some<uint16_t, F> x = load_some(static_cast<const uint16_t*>(a.w) + at * a.w_stride, h + F * r, a.width);
                    if (s) w[1][j] = x;
                    else w[0][j] = x;
                }
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            bf16x8 d[RB][2];
#pragma unroll
            for (int b = 0; b < RB; ++b)
#pragma unroll
                for (int q = 0; q < 2; ++q) d[b][q] = load_eight(p.rows + q * p.plane + (b * 32 + r) * a.dz_stride + v + s * 16 + half * 8);
            const Turned t(w[s]);
#pragma unroll
            for (int b = 0; b < RB; ++b)
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int c = 0; c < F; ++c) acc[b][c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(d[b][q], t[c], acc[b][c], 0, 0, 0);
        }
    }
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int g = 0; g < F; g += 4) narrow_merge<uint16_t>(a, b, split, h + F * r + g, acc[b][g], acc[b][g + 1], acc[b][g + 2], acc[b][g + 3], merge);
}

// dX of 128 features over a range of tokens, fp32: eight at a time, four to each half of a wave; the waves take blocks of 32 tokens in turn.
template <int RB>
__device__ inline void narrow_hidden_fp32(const NarrowArgs& a, int64_t unit, float* merge) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, half = lane >> 5;
    const int slices = (a.width + 127) / 128, h = static_cast<int>(unit % slices) * 128, split = static_cast<int>(unit / slices);
    const int64_t begin = split * a.each, end = min(begin + a.each, a.tokens);
    f32x16 acc[RB][4];
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[b][c][e] = 0.0f;
    const bool whole = h + 128 <= a.width && a.first + end <= a.vocab && end - begin == a.each;
    for (int64_t v = begin + wave * 32; v < end; v += 128) {
        f32x4 d[4][RB], w[4][4];
        const float* row = static_cast<const float*>(a.w) + (a.first + v + half * 4) * a.w_stride + h + 4 * r;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
#pragma unroll
            for (int b = 0; b < RB; ++b) d[q][b] = *reinterpret_cast<const f32x4*>(a.dz + (b * 32 + r) * a.dz_stride + v + q * 8 + half * 4);
            if (whole) {
#pragma unroll
                for (int t = 0; t < 4; ++t) w[q][t] = load_four(row + (q * 8 + t) * a.w_stride, 0, 4);
            } else {
#pragma unroll
                for (int t = 0; t < 4; ++t)     // tokens past the end: the last one again, against a zero of dz
                    w[q][t] = load_four(static_cast<const float*>(a.w) + min(a.first + v + q * 8 + half * 4 + t, a.vocab - 1) * a.w_stride, h + 4 * r, a.width);
            }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int b = 0; b < RB; ++b)
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[b][c] = __builtin_amdgcn_mfma_f32_32x32x2f32(d[q][b][t], w[q][t][c], acc[b][c], 0, 0, 0);
    }
#pragma unroll
    for (int b = 0; b < RB; ++b) narrow_merge<float>(a, b, split, h + 4 * r, acc[b][0], acc[b][1], acc[b][2], acc[b][3], merge);
}

template <class T, int RB>
__global__ __launch_bounds__(kThreads, 2) void narrow_grads_kernel(NarrowArgs a) {
    __shared__ __align__(16) float merge[3 * 32 * 128];
    if constexpr (sizeof(T) == 2) {
        if (blockIdx.x < a.hidden_units) narrow_hidden_bf16<RB>(a, blockIdx.x, merge);
        else narrow_weight_bf16<RB>(a, blockIdx.x - a.hidden_units);
    } else {
        if (blockIdx.x < a.hidden_units) narrow_hidden_fp32<RB>(a, blockIdx.x, merge);
        else narrow_weight_fp32<RB>(a, blockIdx.x - a.hidden_units);
    }
}

template <class A>
int launch(void (*kernel)(A), int64_t grid, const A& args, hipStream_t stream) {
    void* params[] = {const_cast<A*>(&args)};
    return hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3(static_cast<unsigned>(grid)), dim3(kThreads), params, 0, stream) == hipSuccess
               ? JABAS_OK : JABAS_ERR_LAUNCH;
}

template <class T, int RB>
int forward(const NarrowArgs& a, int64_t grid, hipStream_t stream) {
    return a.entries.index ? launch(narrow_forward_kernel<T, RB, true>, grid, a, stream) : launch(narrow_forward_kernel<T, RB, false>, grid, a, stream);
}
template <class T, int RB>
int backward(const NarrowArgs& a, int64_t grid, hipStream_t stream) {
    return a.entries.index ? launch(narrow_backward_kernel<T, RB, true>, grid, a, stream) : launch(narrow_backward_kernel<T, RB, false>, grid, a, stream);
}

}  // namespace

int64_t narrow_tiles(int64_t vocab) { return (vocab + kTokens - 1) / kTokens; }

// Token ranges of dX: 256 workgroups, one a CU beside those of dW, none with less than 128 tokens, a block for each wave. Forward and
// backward with 128, 256 and 512 workgroups: 1 row, 32317 x 1024 bf16 144, 106 and 114 us, fp32 161, 154 and 168; 16 rows fp32 170, 171 and
// 184; 8 rows, 131072 x 4096 bf16 1118, 1095 and 1119.
NarrowSplits narrow_splits(int64_t tokens, int64_t width) {
    const int64_t slices = (width + 127) / 128, most = (tokens + 127) / 128, want = (256 + slices - 1) / slices;
    const int64_t n = want < most ? want : most;
    NarrowSplits s;
    s.each = ((tokens + n - 1) / n + 127) / 128 * 128;
    s.n = static_cast<int32_t>((tokens + s.each - 1) / s.each);
    return s;
}

int launch_narrow_forward(const NarrowArgs& a, int dtype, hipStream_t stream) {
    const int64_t grid = narrow_tiles(a.vocab);
    if (dtype == JABAS_F32) return a.rows <= 32 ? forward<float, 1>(a, grid, stream) : forward<float, 2>(a, grid, stream);
    return a.rows <= 32 ? forward<uint16_t, 1>(a, grid, stream) : forward<uint16_t, 2>(a, grid, stream);
}
int launch_narrow_backward(const NarrowArgs& a, int dtype, hipStream_t stream) {
    const int64_t grid = narrow_tiles(a.tokens);
    if (dtype == JABAS_F32) return a.rows <= 32 ? backward<float, 1>(a, grid, stream) : backward<float, 2>(a, grid, stream);
    return a.rows <= 32 ? backward<uint16_t, 1>(a, grid, stream) : backward<uint16_t, 2>(a, grid, stream);
}
int launch_narrow_grads(const NarrowArgs& a, int dtype, hipStream_t stream) {
    const int64_t grid = a.hidden_units + (a.d_weight ? narrow_tiles(a.tokens) : 0);
    if (dtype == JABAS_F32) return a.rows <= 32 ? launch(narrow_grads_kernel<float, 1>, grid, a, stream) : launch(narrow_grads_kernel<float, 2>, grid, a, stream);
    return a.rows <= 32 ? launch(narrow_grads_kernel<uint16_t, 1>, grid, a, stream) : launch(narrow_grads_kernel<uint16_t, 2>, grid, a, stream);
}

}  // namespace loss
}  // namespace jabas
