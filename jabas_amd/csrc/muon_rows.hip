// The passes over gradients and momenta of the orthogonalised update: momentum and length, then the copy that the products read.
#include "muon_internal.h"
#include "muon_work.h"

namespace jabas {
namespace muon {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <class T>
__device__ inline f32x4 quad(const T* p, int64_t i) {
    if constexpr (sizeof(T) == 4) return *reinterpret_cast<const f32x4*>(p + i);
    else {
        const uint2 v = *reinterpret_cast<const uint2*>(p + i);
        return f32x4{__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u)};
    }
}

// buf' = buf + (1 - momentum) (g - buf), written, and the sum of squares of what is to be orthogonalised, in 64 bits: in 32 a matrix of 10^7
// entries would be off by 1e-5, and entries under 1e-19 would not count.
// Bound by memory, 12 bytes an element (without momentum 2 or 4). A matrix has at most 1024 chunks: whoever needs the length adds that many up. 4 of 1024 x 1024
// and 4 of 1024 x 4096 (21 M elements) take 48 us, 5.2 TB/s; one of 4096 x 1024 10 us; twelve of 768 x 768 fp32 without momentum 7.4.
template <class T>
__global__ __launch_bounds__(256) void momentum_kernel(PassArgs a) {
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < a.n_tickets; i += gridDim.x * 256) a.tickets[i] = 0;
    Sides at;
    if (!sides_of(a.w, at)) return;
    const Matrix x = matrix_of(a.w, at.matrix);
    const T* src = static_cast<const T*>(x.src);
    const Mix mix(a);
    const int64_t count = static_cast<int64_t>(x.rows) * x.cols, begin = static_cast<int64_t>(at.tile) * x.chunk;
    const int64_t end = min(count, begin + x.chunk);
    const bool whole = x.src_stride == x.cols;
    double sum = 0.0;
    const auto take = [&](float g, int64_t i) {
        float u = g * mix.scale;
        if (x.momentum) {
            const float buf = mix.buffer(u, x.momentum[i]);
            x.momentum[i] = buf;
            u = mix.update(u, buf);
        }
        sum += static_cast<double>(u) * u;
    };
    if (whole && x.src_quads) {
        // chunks are multiples of 1024 elements; what is left of the last one goes by single elements
        const int64_t quads = begin + (end - begin) / 4 * 4;
#pragma unroll 2
        for (int64_t i = begin + threadIdx.x * 4; i < quads; i += 1024) {
            f32x4 u = quad(src, i) * mix.scale;
            if (x.momentum) {
                f32x4 buf = *reinterpret_cast<const f32x4*>(x.momentum + i);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    buf[e] = mix.buffer(u[e], buf[e]);
                    u[e] = mix.update(u[e], buf[e]);
                }
                *reinterpret_cast<f32x4*>(x.momentum + i) = buf;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += static_cast<double>(u[e]) * u[e];
        }
        if (quads + threadIdx.x < end) take(element(src, quads + threadIdx.x), quads + threadIdx.x);
    } else if (whole) {
        for (int64_t i = begin + threadIdx.x; i < end; i += 256) take(element(src, i), i);
    } else {
        for (int64_t i = begin + threadIdx.x; i < end; i += 256) {
            const uint32_t row = static_cast<uint32_t>(i / x.cols);
            take(element(src, row * x.src_stride + (i - static_cast<int64_t>(row) * x.cols)), i);
        }
    }
    __shared__ double waves[4];
    sum = sum_of_wave(sum);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) a.w.sums[x.part_at + at.tile] = (waves[0] + waves[1]) + (waves[2] + waves[3]);
}

// X = u / max(|u|, eps) as two planes of fp16 (hi + lo: 22 bits of entries down to 2^-16 of |u|, steps of 2^-38 of it below), the shorter side first, zeros to
// multiples of 64; 64 x 64 of it a workgroup. The update is made once more of gradient and momentum: as many bytes as writing and reading it would be.
// Bound by memory: 8 bytes an element in, 4 out; those matrices 51 us, 4.9 TB/s, one of 4096 x 1024 12 us. The tile goes through LDS whichever way it lies, so that
// tall matrices' rows are read and X's rows are written in full lines.
template <class T, int P>
__global__ __launch_bounds__(256) void lay_kernel(PassArgs a) {
    Sides at;
    if (!sides_of(a.w, at)) return;
    const Matrix x = matrix_of(a.w, at.matrix);
    const T* src = static_cast<const T*>(x.src);
    const Mix mix(a);
    __shared__ double waves[4];
    __shared__ float tile[kLay][kLay + 1];      // as it lies in src: [row][col]
    const int across = x.pad_n / kLay, i0 = at.tile / across * kLay, j0 = at.tile % across * kLay;
    const int r0 = x.tall ? j0 : i0, c0 = x.tall ? i0 : j0;
    {
        const int r = threadIdx.x >> 4, c = c0 + (threadIdx.x & 15) * 4;
#pragma unroll
        for (int p = 0; p < kLay / 16; ++p) {
            const int row = r0 + r + p * 16;
            f32x4 u = {0.0f, 0.0f, 0.0f, 0.0f};
            if (row < x.rows) {
                const int64_t from = row * x.src_stride + c, own = static_cast<int64_t>(row) * x.cols + c;
                if (x.src_quads && c + 4 <= x.cols) {
                    u = quad(src, from) * mix.scale;
                    if (x.momentum) {
                        const f32x4 buf = *reinterpret_cast<const f32x4*>(x.momentum + own);
#pragma unroll
                        for (int e = 0; e < 4; ++e) u[e] = mix.update(u[e], buf[e]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c + e < x.cols) {
                            u[e] = element(src, from + e) * mix.scale;
                            if (x.momentum) u[e] = mix.update(u[e], x.momentum[own + e]);
                        }
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) tile[r + p * 16][(threadIdx.x & 15) * 4 + e] = u[e];
        }
    }
    double sum = 0.0;
    for (int i = threadIdx.x; i < x.parts; i += 256) sum += a.w.sums[x.part_at + i];
    sum = sum_of_wave(sum);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = (waves[0] + waves[1]) + (waves[2] + waves[3]);
    const double length = sqrt(sum);
    // an infinity or a NaN anywhere: NaN everywhere
    const double factor = isfinite(length) ? a.scale / fmax(length, a.eps) : __builtin_nan("");
    _Float16* to = static_cast<_Float16*>(a.w.halves) + x.x_at;
#pragma unroll
    for (int p = 0; p < kLay * kLay / 8 / 256; ++p) {
        const int f = p * 256 + threadIdx.x, i = f >> 3, j = (f & 7) * 8;
        f16x8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float v = static_cast<float>(factor * (x.tall ? tile[j + e][i] : tile[i][j + e]));
            hi[e] = static_cast<_Float16>(v);
            lo[e] = static_cast<_Float16>(v - static_cast<float>(hi[e]));
        }
        const int64_t place = half_at<P>(i0 + i, j0 + j, x.pad_n);
        *reinterpret_cast<f16x8*>(to + place) = hi;
        *reinterpret_cast<f16x8*>(to + place + second_of<P>(x.x_plane)) = lo;
    }
}

template <class K>
int launch(K kernel, const PassArgs& a, hipStream_t stream) {
    void* params[] = {const_cast<PassArgs*>(&a)};
    return hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3(a.w.total), dim3(256), params, 0, stream) == hipSuccess ? JABAS_OK : JABAS_ERR_LAUNCH;
}

}  // namespace

int launch_momentum(const PassArgs& a, hipStream_t stream) {
    return a.dtype == JABAS_F32 ? launch(momentum_kernel<float>, a, stream) : launch(momentum_kernel<uint16_t>, a, stream);
}
int launch_lay(const PassArgs& a, hipStream_t stream) {
    if (a.planes == 2) return a.dtype == JABAS_F32 ? launch(lay_kernel<float, 2>, a, stream) : launch(lay_kernel<uint16_t, 2>, a, stream);
    return a.dtype == JABAS_F32 ? launch(lay_kernel<float, 1>, a, stream) : launch(lay_kernel<uint16_t, 1>, a, stream);
}

}  // namespace muon
}  // namespace jabas
