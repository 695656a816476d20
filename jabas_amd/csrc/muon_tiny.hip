// Small matrices: a workgroup takes one from its gradient to its weights, all steps in LDS.
#include "loss_core.h"
#include "muon_internal.h"
#include "muon_put.h"
#include "muon_work.h"

namespace jabas {
namespace muon {
namespace {

using loss::F16;
using loss::f16x4;
using loss::f16x8;
using loss::f32x16;
using loss::f32x4;

typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 1024, kWaves = 16;

// Halves of a row of `cols`: 16 bytes more than its elements, so that rows start four banks apart.
__host__ __device__ inline int tiny_row(int cols) { return cols + 8; }

// A matrix of LDS in two planes, `plane` halves apart.
struct Held {
    _Float16* p;
    int row, plane;
    // 32 rows from `at`, inner axis along the row: 16 of it from k
    __device__ f16x8 across(int at, int k, int q) const {
        const int lane = threadIdx.x & 63;
        return *reinterpret_cast<const f16x8*>(p + q * plane + (at + (lane & 31)) * row + k + (lane >> 5) * 8);
    }
    // 32 columns from `at`, inner axis along the columns: transposing reads
    __device__ f16x8 down(int at, int k, int q) const {
        const int lane = threadIdx.x & 63;
        const _Float16* from = p + q * plane + (k + (lane >> 5) * 8 + ((lane & 15) >> 2)) * row + at + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(from));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(from + 4 * row));
        return __builtin_bit_cast(f16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    __device__ f32x4 four(int r, int c) const {
        const f16x4 hi = *reinterpret_cast<const f16x4*>(p + r * row + c), lo = *reinterpret_cast<const f16x4*>(p + plane + r * row + c);
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = static_cast<float>(hi[e]) + static_cast<float>(lo[e]);
        return v;
    }
    __device__ void put(int r, int c, f32x4 v) const {
        f16x4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            hi[e] = static_cast<_Float16>(v[e]);
            lo[e] = static_cast<_Float16>(v[e] - static_cast<float>(hi[e]));
        }
        *reinterpret_cast<f16x4*>(p + r * row + c) = hi;
        *reinterpret_cast<f16x4*>(p + plane + r * row + c) = lo;
    }
};

// acc += (a0 + a1)(b0 + b1) without a1 b1
__device__ inline f32x16 multiply(const f16x8 (&a)[2], const f16x8 (&b)[2], f32x16 acc) {
    acc = F16::mfma(a[1], b[0], acc);
    acc = F16::mfma(a[0], b[1], acc);
    return F16::mfma(a[0], b[0], acc);
}

// LDS that a wave reads here was written by other lanes of it, or is about to be.
__device__ inline void wave_done() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The shorter side takes MB blocks of 32. X and A (then B, in its place) lie in LDS in two planes of fp16 whatever the type (22 bits, as
// the larger matrices' fp32 form; bf16's result is then off by its own rounding alone): the products are none of the time. A block of A a wave;
// X is worked on in columns of 32, each by one wave that reads all of it before it writes, so X needs no second copy.
// Bound by the way through LDS and the barriers, four a step: 64 x 64 takes 24 us, where the launches of the larger
// matrices' kernels took 60. Three sums at once, blocks under the diagonal mirrored, the inner axis shared between waves were no faster.
template <class T, int MB>
__global__ __launch_bounds__(kThreads) void tiny_kernel(TinyArgs a) {
    __shared__ __align__(16) char smem[kTinyBytes];
    __shared__ double waves[kWaves];
    Sides at;
    if (!sides_of(a.pass.w, at)) return;
    const Matrix x = matrix_of(a.pass.w, at.matrix);
    constexpr int kM = MB * 32;
    const int cols = (x.n + 31) & ~31, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const Held A{reinterpret_cast<_Float16*>(smem), tiny_row(kM), kM * tiny_row(kM)};
    const Held X{reinterpret_cast<_Float16*>(smem) + 2 * A.plane, tiny_row(cols), kM * tiny_row(cols)};

    for (int i = threadIdx.x; i < X.plane / 4; i += kThreads) reinterpret_cast<f32x4*>(X.p)[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const T* src = static_cast<const T*>(x.src);
    const Mix mix(a.pass);
    const int count = x.rows * x.cols;
    double sum = 0.0;
#pragma unroll 4
    for (int i = threadIdx.x; i < count; i += kThreads) {
        const int row = static_cast<unsigned>(i) / static_cast<unsigned>(x.cols);
        float u = element(src, row * x.src_stride + (i - row * x.cols)) * mix.scale;
        if (x.momentum) {
            const float buf = mix.buffer(u, x.momentum[i]);
            x.momentum[i] = buf;
            u = mix.update(u, buf);
        }
        sum += static_cast<double>(u) * u;
    }
    sum = sum_of_wave(sum);
    if (lane == 0) waves[wave] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += waves[w];
    const double length = sqrt(sum);
    const double factor = isfinite(length) ? a.pass.scale / fmax(length, a.pass.eps) : __builtin_nan("");
#pragma unroll 4
    for (int i = threadIdx.x; i < count; i += kThreads) {       // the elements that this thread wrote the momentum of
        const int row = static_cast<unsigned>(i) / static_cast<unsigned>(x.cols), col = i - row * x.cols;
        float u = element(src, row * x.src_stride + col) * mix.scale;
        if (x.momentum) u = mix.update(u, x.momentum[i]);
        const float v = static_cast<float>(factor * u);
        const int place = (x.tall ? col : row) * X.row + (x.tall ? row : col);
        const _Float16 hi = static_cast<_Float16>(v);
        X.p[place] = hi;
        X.p[X.plane + place] = static_cast<_Float16>(v - static_cast<float>(hi));
    }
    __syncthreads();

    const int n0 = wave / MB * 32, m0 = wave % MB * 32, r = lane & 31, m4 = (lane >> 5) * 4;        // the wave's block of A; a lane's row and first column
    const bool mine = wave < MB * MB;
    for (int k = 0; k < a.steps; ++k) {
        const TinyStep s = a.step[k];
        if (mine) {
            f32x16 acc = {};
#pragma unroll 2
            for (int d = 0; d < cols; d += 16) {
                const f16x8 f[2] = {X.across(m0, d, 0), X.across(m0, d, 1)}, g[2] = {X.across(n0, d, 0), X.across(n0, d, 1)};
                acc = multiply(f, g, acc);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) A.put(n0 + r, m0 + q * 8 + m4, f32x4{acc[q * 4], acc[q * 4 + 1], acc[q * 4 + 2], acc[q * 4 + 3]} * s.first);
        }
        __syncthreads();
        f32x4 b[4];
        if (mine) {
            f32x16 acc = {};
#pragma unroll
            for (int d = 0; d < kM; d += 16) {
                const f16x8 f[2] = {A.across(m0, d, 0), A.across(m0, d, 1)}, g[2] = {A.across(n0, d, 0), A.across(n0, d, 1)};
                acc = multiply(f, g, acc);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
                b[q] = A.four(n0 + r, m0 + q * 8 + m4) * s.second_own + f32x4{acc[q * 4], acc[q * 4 + 1], acc[q * 4 + 2], acc[q * 4 + 3]} * s.second;
        }
        __syncthreads();
        if (mine)
#pragma unroll
            for (int q = 0; q < 4; ++q) A.put(n0 + r, m0 + q * 8 + m4, b[q]);
        __syncthreads();
        const bool last = k + 1 == a.steps;
        for (int c0 = wave * 32; c0 < cols; c0 += kWaves * 32) {
            f32x16 acc[MB] = {};
#pragma unroll
            for (int d = 0; d < kM; d += 16) {
                const f16x8 f[2] = {X.down(c0, d, 0), X.down(c0, d, 1)};
#pragma unroll
                for (int j = 0; j < MB; ++j) {
                    const f16x8 g[2] = {A.across(j * 32, d, 0), A.across(j * 32, d, 1)};
                    acc[j] = multiply(f, g, acc[j]);
                }
            }
            wave_done();
#pragma unroll
            for (int j = 0; j < MB; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int row = j * 32 + r, col = c0 + q * 8 + m4;
                    const f32x4 v = X.four(row, col) * s.update_own + f32x4{acc[j][q * 4], acc[j][q * 4 + 1], acc[j][q * 4 + 2], acc[j][q * 4 + 3]} * s.update;
                    if (!last) {
                        X.put(row, col, v);
                    } else if (row < x.m) {
                        if (!x.tall) {
                            if (col < x.n) put_out<4>(a.out, a.pass.w.fanout, x, row, col, reinterpret_cast<const float*>(&v));
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (col + e < x.n) put_out<1>(a.out, a.pass.w.fanout, x, col + e, row, reinterpret_cast<const float*>(&v) + e);
                        }
                    }
                }
        }
        __syncthreads();
    }
}

template <class T>
int launch(const TinyArgs& a, int blocks, hipStream_t stream) {
    const void* kernels[] = {reinterpret_cast<const void*>(&tiny_kernel<T, 1>), reinterpret_cast<const void*>(&tiny_kernel<T, 2>),
                             reinterpret_cast<const void*>(&tiny_kernel<T, 3>), reinterpret_cast<const void*>(&tiny_kernel<T, 4>)};
    void* params[] = {const_cast<TinyArgs*>(&a)};
    return hipLaunchKernel(kernels[blocks - 1], dim3(a.pass.w.total), dim3(kThreads), params, 0, stream) == hipSuccess ? JABAS_OK : JABAS_ERR_LAUNCH;
}

}  // namespace

bool tiny_fits(int blocks, int64_t n) {
    if (blocks < 1 || blocks > 4 || n > kTinyBytes) return false;
    const int64_t rows = blocks * 32, cols = (n + 31) / 32 * 32;
    return 4 * rows * (tiny_row(static_cast<int>(rows)) + tiny_row(static_cast<int>(cols))) <= kTinyBytes;
}
int launch_tiny(const TinyArgs& a, int blocks, hipStream_t stream) {
    return a.pass.dtype == JABAS_F32 ? launch<float>(a, blocks, stream) : launch<uint16_t>(a, blocks, stream);
}

}  // namespace muon
}  // namespace jabas
