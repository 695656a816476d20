// Matrix products of the orthogonalised update: X X^T, b A + c A A and a X + B X, tiles of many matrices in one launch.
#include <math.h>

#include "loss_core.h"
#include "muon_internal.h"
#include "muon_work.h"

namespace jabas {
namespace muon {
namespace {

using loss::Core;
using loss::F16;
using loss::Operand;
using loss::f16x8;
using loss::f32x4;

__device__ inline uint16_t to_bf16(float x) {
    const uint32_t u = __float_as_uint(x);
    if ((u & 0x7fffffffu) > 0x7f800000u) return static_cast<uint16_t>((u >> 16) | 0x40);
    return static_cast<uint16_t>((u + 0x7fffu + ((u >> 16) & 1)) >> 16);
}

// Eight values and their planes.
struct Eight {
    float v[8];
    __device__ void add_planes(const _Float16* hi, const _Float16* lo, float factor) {
        const f16x8 h = *reinterpret_cast<const f16x8*>(hi);
        if (lo) {
            const f16x8 l = *reinterpret_cast<const f16x8*>(lo);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = fmaf(static_cast<float>(h[e]) + static_cast<float>(l[e]), factor, v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = fmaf(static_cast<float>(h[e]), factor, v[e]);
        }
    }
    __device__ void put_planes(_Float16* hi, _Float16* lo) const {
        f16x8 h, l;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            h[e] = static_cast<_Float16>(v[e]);
            l[e] = static_cast<_Float16>(v[e] - static_cast<float>(h[e]));
        }
        *reinterpret_cast<f16x8*>(hi) = h;
        if (lo) *reinterpret_cast<f16x8*>(lo) = l;
    }
};

// A wave's results go through LDS 32 rows of n at a time, so that a lane has consecutive elements of a row, or, read the other way, of a column:
// row r of kChunks chunks of 16 bytes, chunk k at k ^ r % kChunks.
template <class C>
struct Staged {
    static constexpr int kCols = C::kI * 32, kChunks = kCols / 4;
    float* mine;
    __device__ explicit Staged(char* smem) : mine(reinterpret_cast<float*>(smem + (threadIdx.x >> 6) * (32 * kCols * 4))) {}
    __device__ float* chunk(int r, int k) const { return mine + (r * kChunks + (k ^ (r % kChunks))) * 4; }
    __device__ void put(const C& c, int j, float factor) const {
        const int r = threadIdx.x & 31;
#pragma unroll
        for (int i = 0; i < C::kI; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = c.acc[i][j][q * 4 + e] * factor;
                *reinterpret_cast<f32x4*>(chunk(r, C::block_m(i, q * 4) >> 2)) = v;
            }
    }
    __device__ void get(int r, int col, Eight& x) const {       // columns col .. col + 7 of row r
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(chunk(r, (col >> 2) + h));
#pragma unroll
            for (int e = 0; e < 4; ++e) x.v[h * 4 + e] = v[e];
        }
    }
    __device__ void set(int r, int col, const Eight& x) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) *reinterpret_cast<f32x4*>(chunk(r, (col >> 2) + h)) = f32x4{x.v[h * 4], x.v[h * 4 + 1], x.v[h * 4 + 2], x.v[h * 4 + 3]};
    }
    __device__ float at(int r, int col) const { return chunk(r, col >> 2)[col & 3]; }
};

// LDS written by a wave is read by other lanes of it behind this.
__device__ inline void wave_done() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A = X X^T, or (SECOND) B = b A + c A A: tiles on and under the diagonal, written where they are and mirrored.
template <int P, class C, bool SECOND>
__global__ __launch_bounds__(C::kThreads) void symmetric_kernel(SymmetricArgs a) {
    __shared__ __align__(16) char smem[2 * C::kStage];
    Place at;
    if (!place_of(a.w, at)) return;
    const Matrix& x = at.x;
    int tn = static_cast<int>((sqrtf(8.0f * at.tile + 1.0f) - 1.0f) * 0.5f);        // the last row of tiles that starts at or before `tile`
    while (static_cast<uint32_t>(tn * (tn + 1)) / 2 > at.tile) --tn;
    while (static_cast<uint32_t>((tn + 1) * (tn + 2)) / 2 <= at.tile) ++tn;
    const int tm = at.tile - tn * (tn + 1) / 2, m0 = tm * C::kM, n0 = tn * C::kN, lane = threadIdx.x & 63;
    _Float16* base = static_cast<_Float16*>(a.w.halves);
    _Float16 *own = base + x.a_at, *to = own + (SECOND ? P * x.a_plane : 0);
    const Operand o = SECOND ? Operand{own, x.pad_m, x.a_plane, x.m} : Operand{base + x.x_at + a.from * 2 * x.x_plane, x.pad_n, x.x_plane, x.m};
    C c;
    c.run(o, o, m0, n0, SECOND ? x.pad_m : x.pad_n, smem, [] {}, [](int, int) { return 0.0f; });
    const Staged<C> staged(smem);
    const int wm = m0 + C::wave_m(), wn = n0 + C::wave_n();
    __syncthreads();
#pragma unroll
    for (int j = 0; j < C::kJ; ++j) {
        wave_done();
        staged.put(c, j, a.product);
        wave_done();
#pragma unroll 2
        for (int t = 0; t < C::kI * 2; ++t) {
            const int f = t * 64 + lane, r = f / (C::kI * 4), col = f % (C::kI * 4) * 8, row = wn + j * 32 + r, m = wm + col;
            if (row >= x.m || m >= x.pad_m) continue;
            Eight v;
            staged.get(r, col, v);
            const int64_t place = static_cast<int64_t>(row) * x.pad_m + m;
            if (SECOND) {
                v.add_planes(own + place, P == 2 ? own + x.a_plane + place : nullptr, a.own);
                staged.set(r, col, v);
            }
            if (m + 8 > x.m)
#pragma unroll
                for (int e = 0; e < 8; ++e) v.v[e] = m + e < x.m ? v.v[e] : 0.0f;
            v.put_planes(to + place, P == 2 ? to + x.a_plane + place : nullptr);
        }
        if (tm == tn) continue;
        wave_done();
#pragma unroll 2
        for (int t = 0; t < C::kI * 2; ++t) {       // column wm + col of the tile is row of the mirrored one
            const int f = t * 64 + lane, col = f % (C::kI * 32), r = f / (C::kI * 32) * 8, row = wm + col, m = wn + j * 32 + r;
            if (row >= x.m || m >= x.pad_m) continue;
            Eight v;
#pragma unroll
            for (int e = 0; e < 8; ++e) v.v[e] = m + e < x.m ? staged.at(r + e, col) : 0.0f;
            const int64_t place = static_cast<int64_t>(row) * x.pad_m + m;
            v.put_planes(to + place, P == 2 ? to + x.a_plane + place : nullptr);
        }
    }
}

// Where a step's last product goes: `count` (up to V) results of consecutive columns of a row of the matrix as the caller has it.
template <int V>
__device__ inline void put_out(const UpdateArgs& a, const Matrix& x, int row, int col, const float* v) {
    const int64_t place = static_cast<int64_t>(row) * x.cols + col;
    const int count = min(V, x.cols - col);
    if (!x.momentum) {
        if (a.out_dtype == JABAS_F32) {
            float* out = static_cast<float*>(x.out) + place;
            if (x.out_quads)
#pragma unroll
                for (int e = 0; e < V; e += 4) { if (e < count) *reinterpret_cast<f32x4*>(out + e) = f32x4{v[e], v[e + 1], v[e + 2], v[e + 3]}; }
            else
#pragma unroll
                for (int e = 0; e < V; ++e) { if (e < count) out[e] = v[e]; }
        } else {
            uint16_t* out = static_cast<uint16_t*>(x.out) + place;
            if (x.out_quads)
#pragma unroll
                for (int e = 0; e < V; e += 4) {
                    if (e < count)
                        *reinterpret_cast<uint2*>(out + e) = make_uint2(to_bf16(v[e]) | static_cast<uint32_t>(to_bf16(v[e + 1])) << 16,
                                                                        to_bf16(v[e + 2]) | static_cast<uint32_t>(to_bf16(v[e + 3])) << 16);
                }
            else
#pragma unroll
                for (int e = 0; e < V; ++e) { if (e < count) out[e] = to_bf16(v[e]); }
        }
        return;
    }
    const float lr = a.lr[x.group] * x.lr_factor, keep = a.keep[x.group];
    float* w = static_cast<float*>(x.out) + place;
    if (x.out_quads) {
#pragma unroll
        for (int e = 0; e < V; e += 4) {
            if (e >= count) continue;
            f32x4 now = *reinterpret_cast<const f32x4*>(w + e);
#pragma unroll
            for (int i = 0; i < 4; ++i) now[i] = fmaf(-lr, v[e + i], now[i] * keep);
            *reinterpret_cast<f32x4*>(w + e) = now;
            for (uint32_t f = 0; f < x.n_fanout; ++f) *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(a.w.fanout[x.fanout_at + f]) + place + e) = now;
        }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (e >= count) continue;
            const float now = fmaf(-lr, v[e], w[e] * keep);
            w[e] = now;
            for (uint32_t f = 0; f < x.n_fanout; ++f) reinterpret_cast<float*>(a.w.fanout[x.fanout_at + f])[place + e] = now;
        }
    }
}

// X <- a X + B X, in planes, or at the last step to the weights. X lies with its rows of k: transposing reads take it as it is.
template <int P, class C>
__global__ __launch_bounds__(C::kThreads) void update_kernel(UpdateArgs a) {
    __shared__ __align__(16) char smem[2 * C::kStage];
    Place at;
    if (!place_of(a.w, at)) return;
    const Matrix& x = at.x;
    // bands of eight tiles of m, so that tiles in flight together share their operands' rows
    const int across = (x.n + C::kM - 1) / C::kM, down = (x.m + C::kN - 1) / C::kN;
    const int band = at.tile / (8 * down), first = band * 8, height = min(8, across - first), in = at.tile - band * 8 * down;
    const int m0 = (first + in % height) * C::kM, n0 = in / height * C::kN, lane = threadIdx.x & 63;
    _Float16* base = static_cast<_Float16*>(a.w.halves);
    const _Float16* from = base + x.x_at + a.from * 2 * x.x_plane;
    _Float16* to = base + x.x_at + (1 - a.from) * 2 * x.x_plane;
    C c;
    c.run(Operand{from, x.pad_n, x.x_plane, x.pad_n}, Operand{base + x.a_at + P * x.a_plane, x.pad_m, x.a_plane, x.m}, m0, n0, x.pad_m, smem, [] {},
          [](int, int) { return 0.0f; });
    const Staged<C> staged(smem);
    const int wm = m0 + C::wave_m(), wn = n0 + C::wave_n();
    __syncthreads();
#pragma unroll
    for (int j = 0; j < C::kJ; ++j) {
        wave_done();
        staged.put(c, j, a.product);
        wave_done();
#pragma unroll 2
        for (int t = 0; t < C::kI * 2; ++t) {
            const int f = t * 64 + lane, r = f / (C::kI * 4), col = f % (C::kI * 4) * 8, row = wn + j * 32 + r, m = wm + col;
            if (row >= (a.last ? x.m : x.pad_m) || m >= x.pad_n) continue;
            const int64_t place = static_cast<int64_t>(row) * x.pad_n + m;
            Eight v;
            staged.get(r, col, v);
            v.add_planes(from + place, from + x.x_plane + place, a.own);
            if (!a.last) {
                if (row >= x.m)         // the next product takes these rows of k as well
#pragma unroll
                    for (int e = 0; e < 8; ++e) v.v[e] = 0.0f;
                v.put_planes(to + place, to + x.x_plane + place);
            } else if (x.tall) {
                staged.set(r, col, v);
            } else if (m < x.n) {
                put_out<8>(a, x, row, m, v.v);
            }
        }
        if (!a.last || !x.tall) continue;
        wave_done();
#pragma unroll 2
        for (int t = 0; t < C::kI * 4; ++t) {       // column wm + col of X is a row of the weights
            const int f = t * 64 + lane, r = f % 8 * 4, col = f / 8, row = wm + col, m = wn + j * 32 + r;
            if (row >= x.rows || m >= x.cols) continue;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = staged.at(r + e, col);
            put_out<4>(a, x, row, m, v);
        }
    }
}

template <class K, class A>
int launch(K kernel, int threads, const A& args, hipStream_t stream) {
    void* params[] = {const_cast<A*>(&args)};
    return hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3(args.w.total), dim3(threads), params, 0, stream) == hipSuccess ? JABAS_OK : JABAS_ERR_LAUNCH;
}

template <int P, int T, int WM, int WN>
int symmetric(const SymmetricArgs& a, bool second, hipStream_t stream) {
    using C = Core<F16, P, T, T, WM, WN, false, false, false, false>;
    return second ? launch(symmetric_kernel<P, C, true>, C::kThreads, a, stream) : launch(symmetric_kernel<P, C, false>, C::kThreads, a, stream);
}
template <int P, int T, int WM, int WN>
int update(const UpdateArgs& a, hipStream_t stream) {
    using C = Core<F16, P, T, T, WM, WN, true, false, false, false>;
    return launch(update_kernel<P, C>, C::kThreads, a, stream);
}

}  // namespace

int launch_symmetric(const SymmetricArgs& a, bool second, int planes, int tile, hipStream_t stream) {
    if (planes == 2) return tile == 256 ? symmetric<2, 256, 2, 4>(a, second, stream) : tile == 128 ? symmetric<2, 128, 2, 2>(a, second, stream) : symmetric<2, 64, 2, 2>(a, second, stream);
    return tile == 256 ? symmetric<1, 256, 2, 4>(a, second, stream) : tile == 128 ? symmetric<1, 128, 2, 2>(a, second, stream) : symmetric<1, 64, 2, 2>(a, second, stream);
}

int launch_update(const UpdateArgs& a, int planes, int tile, hipStream_t stream) {
    if (planes == 2) return tile == 256 ? update<2, 256, 2, 4>(a, stream) : tile == 128 ? update<2, 128, 2, 2>(a, stream) : update<2, 64, 2, 2>(a, stream);
    return tile == 256 ? update<1, 256, 2, 4>(a, stream) : tile == 128 ? update<1, 128, 2, 2>(a, stream) : update<1, 64, 2, 2>(a, stream);
}

}  // namespace muon
}  // namespace jabas
