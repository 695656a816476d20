// Losses of few rows (kNarrowRows at most) from hidden states and weight: what counts is to read the weight once for the logits, once for the
// hidden states' gradient, and to write its gradient once. Nothing is copied or laid out first: fragments come from memory as they lie, at
// any alignment, and there is no LDS in the inner loops, so nothing waits for a barrier.
//
// Logits: 32 tokens a workgroup, the four waves take the width's blocks of 64 in turn. Lane (r, half) holds 32 consecutive elements of
// token r: which elements of the inner axis meet in one matrix instruction is free as long as both operands agree, so each lane reads
// whole 64 or 128 bytes. bf16 through 32x32x16, fp32 through 32x32x2: its rate (16 bytes of weight per clock and CU at 32 rows) is above
// what memory gives.
// Gradients: dz in fp32, in the units of the result, so that the row gradients are exact whatever their size. Its products take
// 32x32x2 for both types: a lane holds one element of the inner axis, so operands whose rows are that axis need no transposing.
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
__global__ __launch_bounds__(kThreads) void narrow_forward_kernel(NarrowArgs a) {
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

// The row gradient of n; 0 for rows that do not count.
__device__ inline float row_gradient(const NarrowArgs& a, int n) {
    if (n >= a.rows) return 0.0f;
    const RowState st = a.state[n];
    return st.slope == 0.0f && st.mass == 0.0f ? 0.0f : a.upstream[a.per_row ? n : 0] * (*a.reduce * a.t);
}

template <class T, int RB, bool TEACHER>
__global__ __launch_bounds__(kThreads) void narrow_backward_kernel(NarrowArgs a) {
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
    for (int i = threadIdx.x; i < R * kTokens; i += kThreads) {
        const int n = i / kTokens, m = i % kTokens;
        a.dz[n * a.dz_stride + from + m] = ds[n][m];
    }
}

// Four consecutive elements of a row from column c on, zeros past the end.
template <class T>
__device__ inline f32x4 load_four(const T* row, int c, int cols) {
    f32x4 v;
    if (c + 4 <= cols) {
        const Some<T, 4> x = *reinterpret_cast<const Some<T, 4>*>(row + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = widen(x.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = c + i < cols ? widen(row[c + i]) : 0.0f;
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

// dW of 32 tokens: the sum over rows is the inner axis, two at a time; the waves take 128 features in turn.
template <class T, int RB>
__device__ inline void narrow_weight(const NarrowArgs& a, int64_t unit) {
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
            f32x4 x = load_four(static_cast<const T*>(a.x) + static_cast<int64_t>(min(n, a.rows - 1)) * a.x_stride, h + 4 * r, a.width);
            if (!((live >> n) & 1)) x = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] = __builtin_amdgcn_mfma_f32_32x32x2f32(d[i], x[c], acc[c], 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int64_t v = first + block_m(e);
            if (v < a.vocab) store_four(static_cast<T*>(a.d_weight) + v * a.width, h + 4 * r, a.width, f32x4{acc[0][e], acc[1][e], acc[2][e], acc[3][e]});
        }
    }
}

// dX of 128 features over a range of tokens: eight at a time, four to each half of a wave; the waves take blocks of 32 tokens in turn.
template <class T, int RB>
__device__ inline void narrow_hidden(const NarrowArgs& a, int64_t unit, float* merge) {
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
    for (int64_t v = begin + wave * 32; v < end; v += 128) {
        f32x4 d[4][RB], w[4][4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
#pragma unroll
            for (int b = 0; b < RB; ++b) d[q][b] = *reinterpret_cast<const f32x4*>(a.dz + (b * 32 + r) * a.dz_stride + v + q * 8 + half * 4);
#pragma unroll
            for (int t = 0; t < 4; ++t)     // tokens past the end: the last one again, against a zero of dz
                w[q][t] = load_four(static_cast<const T*>(a.w) + min(a.first + v + q * 8 + half * 4 + t, a.vocab - 1) * a.w_stride, h + 4 * r, a.width);
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
    // the four waves' sums: merge[wave - 1][32 rows][128 features], one block of rows after the other
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        __syncthreads();
        if (wave)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                *reinterpret_cast<f32x4*>(merge + ((wave - 1) * 32 + block_m(e)) * 128 + 4 * r) = f32x4{acc[b][0][e], acc[b][1][e], acc[b][2][e], acc[b][3][e]};
        __syncthreads();
        if (wave) continue;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int m = block_m(e), n = b * 32 + m;
            f32x4 v = {acc[b][0][e], acc[b][1][e], acc[b][2][e], acc[b][3][e]};
#pragma unroll
            for (int i = 0; i < 3; ++i) v += *reinterpret_cast<const f32x4*>(merge + (i * 32 + m) * 128 + 4 * r);
            if (n >= a.rows) continue;
            if (a.part) {
                if (h + 4 * r >= a.width) continue;
                f32x4* sum = reinterpret_cast<f32x4*>(a.part + split * a.part_plane + n * a.part_stride + h + 4 * r);
                *sum = a.add ? *sum + v : v;
            } else {
                store_four(static_cast<T*>(a.d_hidden) + static_cast<int64_t>(n) * a.width, h + 4 * r, a.width, v);
            }
        }
    }
}

template <class T, int RB>
__global__ __launch_bounds__(kThreads) void narrow_grads_kernel(NarrowArgs a) {
    __shared__ __align__(16) float merge[3 * 32 * 128];
    if (blockIdx.x < a.hidden_units) narrow_hidden<T, RB>(a, blockIdx.x, merge);
    else narrow_weight<T, RB>(a, blockIdx.x - a.hidden_units);
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

// Token ranges of dX: 256 workgroups, one a CU beside those of dW, none with less than 128 tokens, a block for each wave, nor with more than
// 8192, which would end after all others. Forward and backward with 128, 256 and 512 workgroups: 1 row, 32317 x 1024 bf16 176, 127 and
// 132 us, fp32 162, 152 and 166; 48 rows fp32 316, 336 and 358; 8 rows, 131072 x 4096 bf16 (16384 tokens at 256) 3014, 1908 and 1640.
NarrowSplits narrow_splits(int64_t tokens, int64_t width) {
    const int64_t slices = (width + 127) / 128, most = (tokens + 127) / 128, least = (tokens + 8191) / 8192;
    int64_t n = (256 + slices - 1) / slices;
    if (n < least) n = least;
    if (n > most) n = most;
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
