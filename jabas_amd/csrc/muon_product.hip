// Matrix products of the orthogonalised update: X X^T, b A + c A A and a X + B X, tiles of many matrices in one launch.
#include <math.h>

#include "loss_core.h"
#include "muon_internal.h"
#include "muon_put.h"
#include "muon_work.h"

namespace jabas {
namespace muon {
namespace {

using loss::Core;
using loss::F16;
using loss::Operand;
using loss::f16x8;
using loss::f32x4;

// Eight values and their planes: fp16 each, the second what the first leaves of the value, 22 bits together. Products of two planes leave out the two seconds (2^-22
// of a product), products of one take the first alone (11 bits): fp32 matrix instructions reach an eighth of the rate (150 TFLOP/s for 1210), and three products of planes
// were off by 1.2 to 1.5e-6 from the definition where the definition in 32 bits is by 1.5 to 2.3e-6. One plane makes 1000 x 2048 in bf16 2.1e-3 where the
// result's own rounding is 1.7e-3, 4096 x 16384 1.9e-3 for 1.7e-3, at a third of the products.
template <int P>
struct Planes {
    f16x8 v[P];
};
struct Eight {
    float v[8];
    template <int P>
    __device__ void add(const Planes<P>& x, float factor) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf(static_cast<float>(x.v[0][e]) + (P == 2 ? static_cast<float>(x.v[P - 1][e]) : 0.0f), factor, v[e]);
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
    // Eights of a row are taken kGroup at a time, group g of block column j, and those of the matrix that is added to are read a group ahead.
    static constexpr int kEach = C::kI * 2, kGroup = kEach < 4 ? kEach : 4, kGroups = kEach / kGroup;
    static __device__ int row(int t) { return (t * 64 + static_cast<int>(threadIdx.x & 63)) / (C::kI * 4); }
    static __device__ int col(int t) { return (t * 64 + static_cast<int>(threadIdx.x & 63)) % (C::kI * 4) * 8; }
    static constexpr bool kEarly = C::kM < 256;         // the first group is on its way while the products are made: large tiles have no registers for it
    // Q planes of a matrix laid out for products of P
    template <int P, int Q>
    static __device__ void fetch(Planes<Q> (&x)[kGroup], int g, const _Float16* from, int64_t plane, int row0, int rows, int col0, int cols) {
#pragma unroll
        for (int t = 0; t < kGroup; ++t) {
            const int r = row0 + row(g * kGroup + t), c = col0 + col(g * kGroup + t);
#pragma unroll
            for (int q = 0; q < Q; ++q)
                if (r < rows && c < cols) x[t].v[q] = *reinterpret_cast<const f16x8*>(from + half_at<P>(r, c, cols) + q * second_of<P>(plane));
        }
    }
};

// LDS written by a wave is read by other lanes of it behind this.
__device__ inline void wave_done() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Tile `tile` of those on and under the diagonal, row by row.
__device__ inline void triangle(uint32_t tile, int& tm, int& tn) {
    int row = static_cast<int>((sqrtf(8.0f * tile + 1.0f) - 1.0f) * 0.5f);         // the last row that starts at or before `tile`
    while (static_cast<uint32_t>(row) * (row + 1) / 2 > tile) --row;
    while (static_cast<uint32_t>(row + 1) * (row + 2) / 2 <= tile) ++row;
    tn = row;
    tm = static_cast<int>(tile - static_cast<uint32_t>(row) * (row + 1) / 2);
}

// A = X X^T, or (SECOND) B = b A + c A A: tiles on and under the diagonal, written where they are and mirrored, because half the products are then enough.
// Bound by the matrix cores where tiles fill the chip's rounds: of 4096 x 16384 (bf16, tiles of 256) X X^T takes 355 us, 774 TFLOP/s counted by half, but 136 tiles
// for 256 CUs; four of 1024 x 4096 and four of 1024 x 1024 (fp32, tiles of 128) 94 us, 688 counted three times; twelve of 768 x 768 (252 tiles of 12 steps) 28 us, 592:
// a tile's start and end are about 6 us whatever its length, a launch 4.
template <int P, class C, bool SECOND>
__global__ __launch_bounds__(C::kThreads) void symmetric_kernel(SymmetricArgs a) {
    __shared__ __align__(16) char smem[C::kStages * C::kStage];
    Sides x;
    if (!sides_of(a.w, x)) return;
    int tm, tn;
    triangle(x.tile, tm, tn);
    const int m0 = tm * C::kM, n0 = tn * C::kN, lane = threadIdx.x & 63;
    _Float16* base = static_cast<_Float16*>(a.w.halves);
    _Float16 *own = base + x.a_at, *to = own + (SECOND ? P * x.a_plane : 0);
    const Operand o = SECOND ? Operand{own, stride_of<P>(x.pad_m), second_of<P>(x.a_plane), x.m}
                             : Operand{base + x.x_at + a.from * 2 * x.x_plane, stride_of<P>(x.pad_n), second_of<P>(x.x_plane), x.m};
    using S = Staged<C>;
    const int wm = m0 + C::wave_m(), wn = n0 + C::wave_n();
    Planes<P> beside[2][S::kGroup];
    const auto fetch_first = [&] { S::template fetch<P, P>(beside[0], 0, own, x.a_plane, wn, x.m, wm, x.pad_m); };
    C c;
    c.run(o, o, m0, n0, SECOND ? x.pad_m : x.pad_n, smem, [&] { if (SECOND && S::kEarly) fetch_first(); }, [](int, int) { return 0.0f; });
    const S staged(smem);
    if (SECOND && !S::kEarly) fetch_first();
    __syncthreads();
#pragma unroll
    for (int j = 0; j < C::kJ; ++j) {
        wave_done();
        staged.put(c, j, a.product);
        wave_done();
#pragma unroll
        for (int g = 0; g < S::kGroups; ++g) {
            const int now = j * S::kGroups + g, after = now + 1;
            if (SECOND && after < C::kJ * S::kGroups)
                S::template fetch<P, P>(beside[after & 1], after % S::kGroups, own, x.a_plane, wn + after / S::kGroups * 32, x.m, wm, x.pad_m);
#pragma unroll
            for (int t = 0; t < S::kGroup; ++t) {
                const int r = S::row(g * S::kGroup + t), col = S::col(g * S::kGroup + t), row = wn + j * 32 + r, m = wm + col;
                if (row >= x.m || m >= x.pad_m) continue;
                Eight v;
                staged.get(r, col, v);
                const int64_t place = half_at<P>(row, m, x.pad_m);
                if (SECOND) {
                    v.add(beside[now & 1][t], a.own);
                    staged.set(r, col, v);
                }
                if (m + 8 > x.m)
#pragma unroll
                    for (int e = 0; e < 8; ++e) v.v[e] = m + e < x.m ? v.v[e] : 0.0f;
                v.put_planes(to + place, P == 2 ? to + place + second_of<P>(x.a_plane) : nullptr);
            }
        }
        if (tm == tn) continue;
        wave_done();
#pragma unroll 2
        for (int t = 0; t < C::kI * 2; ++t) {       // column wm + col of the tile is row of the mirrored one
            const int f = t * 64 + lane, col = f / 4, r = f % 4 * 8, row = wm + col, m = wn + j * 32 + r;
            if (row >= x.m || m >= x.pad_m) continue;
            Eight v;
#pragma unroll
            for (int e = 0; e < 8; ++e) v.v[e] = m + e < x.m ? staged.at(r + e, col) : 0.0f;
            const int64_t place = half_at<P>(row, m, x.pad_m);
            v.put_planes(to + place, P == 2 ? to + place + second_of<P>(x.a_plane) : nullptr);
        }
    }
}

// Tiles of 64 x 64, for launches that leave a CU one or a few of them: what a step takes then is the way of its loads (about half a microsecond
// behind a kernel that wrote them on another die) and the chain of barrier, LDS read and product. So S stages of LDS are on their way at once, a wave
// has all it multiplies in a step in registers a step ahead, and the four waves are two halves of the inner axis by two halves of n, which reads LDS less
// than four quarters of the tile do. The halves' sums meet in LDS.
// A step of 64 of two planes takes 0.45 us with one tile a CU. Two stages leave room for four tiles a CU: a X + B X of 6 of 1024 x 4096 takes 180 us
// with them and 203 with four stages, of one of 1024 x 4096 36 and 37. 21 convolutions' matrices (43 tiles, up to 1152 long) take 11, 6 and 8 us for X X^T,
// A A and a X + B X, of which the launch and the first loads are about 4 each.
template <int P, bool TA, int S>
struct Deep {
    using C = Core<F16, P, 64, 64, 2, 2, TA, false, false, false, 2, P == 2>;
    static constexpr int kThreads = 256, kLoads = C::kLoadsA + C::kLoadsB, kHalf = C::kParts / 2, kRow = 68;    // kRow: floats of a row of sums
    static constexpr int kBytes = S * C::kStage > 64 * kRow * 4 ? S * C::kStage : 64 * kRow * 4;
    static_assert((S - 1) * kLoads < 64, "what the counter holds");

    struct Fragments {
        f16x8 a[kHalf][2][P], b[kHalf][P];
    };
    static __device__ int half() { return (threadIdx.x >> 6) & 1; }
    static __device__ int column() { return (threadIdx.x >> 7) * 32; }

    static __device__ void read(Fragments& f, const char* stage) {
#pragma unroll
        for (int k = 0; k < kHalf; ++k) {
            const int kk = half() * kHalf + k;
#pragma unroll
            for (int q = 0; q < P; ++q) {
                f.b[k][q] = C::template fragment<64, false>(stage + C::kBytesA, column(), kk, q);
#pragma unroll
                for (int i = 0; i < 2; ++i) f.a[k][i][q] = C::template fragment<64, TA>(stage, i * 32, kk, q);
            }
        }
    }
    static __device__ void multiply(const Fragments& f, loss::f32x16 (&acc)[2]) {
#pragma unroll
        for (int k = 0; k < kHalf; ++k) {
            if (P == 2) {
#pragma unroll
                for (int i = 0; i < 2; ++i) acc[i] = F16::mfma(f.a[k][i][P - 1], f.b[k][0], acc[i]);
#pragma unroll
                for (int i = 0; i < 2; ++i) acc[i] = F16::mfma(f.a[k][i][0], f.b[k][P - 1], acc[i]);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) acc[i] = F16::mfma(f.a[k][i][0], f.b[k][0], acc[i]);
        }
    }
    // Waits until at most `Behind` steps' loads are on their way, and for the other waves.
    template <int Behind>
    static __device__ void arrive() {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(Behind * kLoads) : "memory");
    }

    // The tile's sums times `factor`, row n of kRow floats, in smem. Everyone may read them when this returns.
    static __device__ float* run(const Operand& a, const Operand& b, int m0, int n0, int depth, float factor, char* smem) {
        typename C::template Source<64, TA> sa(a, m0);
        typename C::template Source<64, false> sb(b, n0);
        const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)smem));
        const auto load = [&](int stage) {
            const uint32_t to = lds + stage * C::kStage;
#pragma unroll
            for (int l = 0; l < C::kLoadsA; ++l) sa.issue(to, l);
#pragma unroll
            for (int l = 0; l < C::kLoadsB; ++l) sb.issue(to + C::kBytesA, l);
            sa.advance();
            sb.advance();
        };
        const int steps = depth / C::kStep;     // at least one
        for (int s = 0; s < min(S, steps); ++s) load(s);
        loss::f32x16 acc[2] = {};
        if (steps >= S) arrive<S - 1>();
        else arrive<0>();
        Fragments f[2];
        read(f[0], smem);
        int at = 0;
        // Step s, whose fragments are `now`.
        const auto pass = [&](int s, const Fragments& now, Fragments& next) {
            if (s + S <= steps) arrive<S - 2>();
            else arrive<0>();
            const int following = at + 1 == S ? 0 : at + 1;
            if (s + S < steps) load(at);
            read(next, smem + following * C::kStage);       // behind the last step: read, not used
            multiply(now, acc);
            at = following;
        };
        int s = 0;
        for (; s + 2 <= steps; s += 2) {
            pass(s, f[0], f[1]);
            pass(s + 1, f[1], f[0]);
        }
        if (s < steps) pass(s, f[0], f[1]);
        arrive<0>();
        float* sums = reinterpret_cast<float*>(smem);
        const int lane = threadIdx.x & 63;
        const auto quad = [&](int i, int q) { return reinterpret_cast<f32x4*>(sums + (column() + (lane & 31)) * kRow + i * 32 + q * 8 + (lane >> 5) * 4); };
        const auto value = [&](int i, int q) { return f32x4{acc[i][q * 4], acc[i][q * 4 + 1], acc[i][q * 4 + 2], acc[i][q * 4 + 3]}; };
        if (half() == 0)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) *quad(i, q) = value(i, q);
        __syncthreads();
        if (half() == 1)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) *quad(i, q) = (*quad(i, q) + value(i, q)) * factor;
        __syncthreads();
        return sums;
    }
    // Eight `t` (of two) of a thread: its row and column in the tile.
    static __device__ int row(int t) { return t * 32 + (threadIdx.x >> 3); }
    static __device__ int col() { return (threadIdx.x & 7) * 8; }
};

// A tile's sums over the parts of the inner axis that its workgroups took, added up in their order by the one that is done last; false in the others.
// The order is gfx950's, not the language's: stores and loads of the parts are atomic ones of agent scope, which this chip makes at the point that all dies share and
// not in a die's own cache; vmcnt counts stores until they have arrived there, and every wave waits for it to reach zero ahead of the barrier behind which the workgroup
// counts as done; the loads are issued when the ticket has come back. A releasing ticket with an acquiring fence in the last workgroup would say the same in the language,
// but has the die's L2 written back, and emptied, under its other workgroups: 4096 x 1024 fp32 386 us a call for 350, 1024 x 4096 bf16 257 for 222,
// 800 x 2048 fp32 233 for 218, 448 x 4096 194 for 186. 256 x 4096 (10 tiles) takes 149 us with 8 workgroups a tile and 241 with one.
template <class D>
__device__ inline bool join(float* sums, float* shares, uint32_t* ticket, int splits, uint32_t split, int64_t apart) {
    __shared__ uint32_t done;
    uint64_t* mine = reinterpret_cast<uint64_t*>(shares + split * apart);
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        const int f = t * 256 + threadIdx.x;
        __hip_atomic_store(mine + f, *reinterpret_cast<const uint64_t*>(sums + (f >> 5) * D::kRow + (f & 31) * 2), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) done = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (done + 1 != static_cast<uint32_t>(splits)) return false;
    float2 sum[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) sum[t] = make_float2(0.0f, 0.0f);
    for (int s = 0; s < splits; ++s) {
        const uint64_t* from = reinterpret_cast<const uint64_t*>(shares + s * apart);
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            const uint64_t v = __hip_atomic_load(from + t * 256 + threadIdx.x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            sum[t].x += __uint_as_float(static_cast<uint32_t>(v));
            sum[t].y += __uint_as_float(static_cast<uint32_t>(v >> 32));
        }
    }
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        const int f = t * 256 + threadIdx.x;
        *reinterpret_cast<float2*>(sums + (f >> 5) * D::kRow + (f & 31) * 2) = sum[t];
    }
    if (threadIdx.x == 0) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);      // for the next launch
    __syncthreads();
    return true;
}

template <int P, bool SECOND, int S>
__global__ __launch_bounds__(256) void symmetric_deep_kernel(SymmetricArgs a) {
    using D = Deep<P, false, S>;
    __shared__ __align__(16) char smem[D::kBytes];
    Sides x;
    if (!sides_of(a.w, x)) return;
    const int side = (x.m + 63) / 64;
    const uint32_t tiles = static_cast<uint32_t>(side) * (side + 1) / 2;
    const uint32_t split = !SECOND && x.splits > 1 ? x.tile / tiles : 0, tile = x.tile - split * tiles;
    int tm, tn;
    triangle(tile, tm, tn);
    const int m0 = tm * 64, n0 = tn * 64;
    _Float16* base = static_cast<_Float16*>(a.w.halves);
    _Float16 *own = base + x.a_at, *to = own + (SECOND ? P * x.a_plane : 0);
    const Operand o = SECOND ? Operand{own, stride_of<P>(x.pad_m), second_of<P>(x.a_plane), x.m}
                             : Operand{base + x.x_at + a.from * 2 * x.x_plane, stride_of<P>(x.pad_n), second_of<P>(x.x_plane), x.m};
    Planes<P> beside[2];            // on their way while the products are made
    if (SECOND)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int q = 0; q < P; ++q)
                beside[t].v[q] = *reinterpret_cast<const f16x8*>(own + half_at<P>(min(n0 + D::row(t), x.m - 1), min(m0 + D::col(), x.pad_m - 8), x.pad_m) + q * second_of<P>(x.a_plane));
    // this workgroup's part of the inner axis: steps of 64, of which the host gives every workgroup some
    const int whole = SECOND ? x.pad_m : x.pad_n;
    Operand part = o;
    int depth = whole;
    if (!SECOND && x.splits > 1) {
        const int first = split * (whole / 64) / x.splits * 64, last = (split + 1) * (whole / 64) / x.splits * 64;
        part.p = static_cast<const _Float16*>(o.p) + static_cast<int64_t>(first) * P;
        depth = last - first;
    }
    float* sums = D::run(part, part, m0, n0, depth, a.product, smem);
    if (!SECOND && x.splits > 1) {
        const uint32_t at = x.unit + tile;
        if (!join<D>(sums, a.shares + static_cast<int64_t>(at) * 4096, a.tickets + at, x.splits, split, static_cast<int64_t>(tiles) * 4096)) return;
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int r = D::row(t), row = n0 + r, m = m0 + D::col();
        if (row >= x.m || m >= x.pad_m) continue;
        const int64_t place = half_at<P>(row, m, x.pad_m);
        Eight v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v.v[e] = sums[r * D::kRow + D::col() + e];
        if (SECOND) {
            v.add(beside[t], a.own);
            if (tm != tn)
#pragma unroll
                for (int e = 0; e < 8; ++e) sums[r * D::kRow + D::col() + e] = v.v[e];
        }
        if (m + 8 > x.m)
#pragma unroll
            for (int e = 0; e < 8; ++e) v.v[e] = m + e < x.m ? v.v[e] : 0.0f;
        v.put_planes(to + place, P == 2 ? to + place + second_of<P>(x.a_plane) : nullptr);
    }
    if (tm == tn) return;
    if (SECOND) __syncthreads();
#pragma unroll
    for (int t = 0; t < 2; ++t) {       // column m0 + col of the tile is a row of the mirrored one
        const int col = D::row(t), r = D::col(), row = m0 + col, m = n0 + r;
        if (row >= x.m || m >= x.pad_m) continue;
        Eight v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v.v[e] = m + e < x.m ? sums[(r + e) * D::kRow + col] : 0.0f;
        const int64_t place = half_at<P>(row, m, x.pad_m);
        v.put_planes(to + place, P == 2 ? to + place + second_of<P>(x.a_plane) : nullptr);
    }
}

// Tile `tile` of across x down, in bands of eight of m, so that tiles in flight together share their operands' rows.
__device__ inline void band(uint32_t tile, int across, int down, int& tm, int& tn) {
    const int which = static_cast<int>(tile / (8u * down)), first = which * 8, height = min(8, across - first), in = static_cast<int>(tile - which * 8u * down);
    tm = first + in % height;
    tn = in / height;
}

// X <- a X + B X, in planes, or at the last step to the weights. X lies with its rows of k: transposing reads take it as it is.
// Bound by the matrix cores, and in large ones by the power that they take: 4096 x 16384 bf16 507 us, 1084 TFLOP/s (the library's plain product of that shape 1243);
// 8 of 4096 x 1024 and two of 4096 x 2048 fp32 996 counted three times (1204); one of 4096 x 1024, 256 tiles of 128, 32 us and 803.
template <int P, class C>
__global__ __launch_bounds__(C::kThreads) void update_kernel(UpdateArgs a) {
    __shared__ __align__(16) char smem[C::kStages * C::kStage];
    Sides x;
    if (!sides_of(a.w, x)) return;
    int m0, n0;
    band(x.tile, (x.n + C::kM - 1) / C::kM, (x.m + C::kN - 1) / C::kN, m0, n0);
    m0 *= C::kM;
    n0 *= C::kN;
    const int lane = threadIdx.x & 63;
    _Float16* base = static_cast<_Float16*>(a.w.halves);
    const _Float16* from = base + x.x_at + a.from * 2 * x.x_plane;
    _Float16* to = base + x.x_at + (1 - a.from) * 2 * x.x_plane;
    using S = Staged<C>;
    const int wm = m0 + C::wave_m(), wn = n0 + C::wave_n();
    Planes<2> beside[2][S::kGroup];
    const auto fetch_first = [&] { S::template fetch<P, 2>(beside[0], 0, from, x.x_plane, wn, x.m, wm, x.pad_n); };
    C c;
    c.run(Operand{from, stride_of<P>(x.pad_n), second_of<P>(x.x_plane), x.pad_n},
          Operand{base + x.a_at + P * x.a_plane, stride_of<P>(x.pad_m), second_of<P>(x.a_plane), x.m}, m0, n0, x.pad_m, smem,
          [&] { if (S::kEarly) fetch_first(); }, [](int, int) { return 0.0f; });
    const S staged(smem);
    if (!S::kEarly) fetch_first();
    __syncthreads();
#pragma unroll
    for (int j = 0; j < C::kJ; ++j) {
        wave_done();
        staged.put(c, j, a.product);
        wave_done();
#pragma unroll
        for (int g = 0; g < S::kGroups; ++g) {
            const int now = j * S::kGroups + g, after = now + 1;
            if (after < C::kJ * S::kGroups)
                S::template fetch<P, 2>(beside[after & 1], after % S::kGroups, from, x.x_plane, wn + after / S::kGroups * 32, x.m, wm, x.pad_n);
#pragma unroll
            for (int t = 0; t < S::kGroup; ++t) {
                const int r = S::row(g * S::kGroup + t), col = S::col(g * S::kGroup + t), row = wn + j * 32 + r, m = wm + col;
                if (row >= (a.last ? x.m : x.pad_m) || m >= x.pad_n) continue;
                const int64_t place = half_at<P>(row, m, x.pad_n);
                Eight v;
                if (row < x.m) {
                    staged.get(r, col, v);
                    v.add(beside[now & 1][t], a.own);
                } else {            // the next product takes these rows of k as well
#pragma unroll
                    for (int e = 0; e < 8; ++e) v.v[e] = 0.0f;
                }
                if (a.last) staged.set(r, col, v);
                else v.put_planes(to + place, to + place + second_of<P>(x.x_plane));
            }
        }
        if (!a.last) continue;
        wave_done();
        const Matrix out = matrix_of(a.w, x.matrix);
        if (out.tall) {
#pragma unroll 1
            for (int t = 0; t < C::kI * 4; ++t) {       // column wm + col of X is a row of the weights
                const int f = t * 64 + lane, r = f % 8 * 4, col = f / 8, row = wm + col, m = wn + j * 32 + r;
                if (row >= out.rows || m >= out.cols) continue;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = staged.at(r + e, col);
                put_out<4>(a.out, a.w.fanout, out, row, m, v);
            }
        } else {
#pragma unroll 1
            for (int t = 0; t < S::kEach; ++t) {
                const int r = S::row(t), col = S::col(t), row = wn + j * 32 + r, m = wm + col;
                if (row >= out.rows || m >= out.cols) continue;
                Eight v;
                staged.get(r, col, v);
                put_out<8>(a.out, a.w.fanout, out, row, m, v.v);
            }
        }
    }
}

// The same with small tiles.
template <int P, int S>
__global__ __launch_bounds__(256) void update_deep_kernel(UpdateArgs a) {
    using D = Deep<P, true, S>;
    __shared__ __align__(16) char smem[D::kBytes];
    Sides x;
    if (!sides_of(a.w, x)) return;
    int m0, n0;
    band(x.tile, (x.n + 63) / 64, (x.m + 63) / 64, m0, n0);
    m0 *= 64;
    n0 *= 64;
    _Float16* base = static_cast<_Float16*>(a.w.halves);
    const _Float16* from = base + x.x_at + a.from * 2 * x.x_plane;
    _Float16* to = base + x.x_at + (1 - a.from) * 2 * x.x_plane;
    Planes<2> beside[2];            // on their way while the products are made
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int q = 0; q < 2; ++q)
            beside[t].v[q] = *reinterpret_cast<const f16x8*>(from + half_at<P>(n0 + D::row(t), m0 + D::col(), x.pad_n) + q * second_of<P>(x.x_plane));
    float* sums = D::run(Operand{from, stride_of<P>(x.pad_n), second_of<P>(x.x_plane), x.pad_n},
                         Operand{base + x.a_at + P * x.a_plane, stride_of<P>(x.pad_m), second_of<P>(x.a_plane), x.m}, m0, n0, x.pad_m, a.product, smem);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int r = D::row(t), row = n0 + r, m = m0 + D::col();       // whole rows of the padded copy, up to pad_m and pad_n
        Eight v;
        if (row < x.m) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v.v[e] = sums[r * D::kRow + D::col() + e];
            v.add(beside[t], a.own);
        } else {                    // the next product takes these rows of k as well
#pragma unroll
            for (int e = 0; e < 8; ++e) v.v[e] = 0.0f;
        }
        if (a.last) {
#pragma unroll
            for (int e = 0; e < 8; ++e) sums[r * D::kRow + D::col() + e] = v.v[e];
        } else {
            const int64_t place = half_at<P>(row, m, x.pad_n);
            v.put_planes(to + place, to + place + second_of<P>(x.x_plane));
        }
    }
    if (!a.last) return;
    __syncthreads();
    const Matrix out = matrix_of(a.w, x.matrix);
#pragma unroll
    for (int t = 0; t < 2; ++t) {       // where X is the transpose, column m0 + D::row(t) of it is a row of the weights
        const int row = (out.tall ? m0 : n0) + D::row(t), col = (out.tall ? n0 : m0) + D::col();
        if (row >= out.rows || col >= out.cols) continue;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = out.tall ? sums[(D::col() + e) * D::kRow + D::row(t)] : sums[D::row(t) * D::kRow + D::col() + e];
        put_out<8>(a.out, a.w.fanout, out, row, col, v);
    }
}

template <class K, class A>
int launch(K kernel, int threads, const A& args, hipStream_t stream) {
    void* params[] = {const_cast<A*>(&args)};
    return hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3(args.w.total), dim3(threads), params, 0, stream) == hipSuccess ? JABAS_OK : JABAS_ERR_LAUNCH;
}

template <int P, int T, int WM, int WN, int S = 2>
int symmetric(const SymmetricArgs& a, bool second, hipStream_t stream) {
    using C = Core<F16, P, T, T, WM, WN, false, false, false, false, S, P == 2>;
    return second ? launch(symmetric_kernel<P, C, true>, C::kThreads, a, stream) : launch(symmetric_kernel<P, C, false>, C::kThreads, a, stream);
}
template <int P, int T, int WM, int WN, int S = 2>
int update(const UpdateArgs& a, hipStream_t stream) {
    using C = Core<F16, P, T, T, WM, WN, true, false, false, false, S, P == 2>;
    return launch(update_kernel<P, C>, C::kThreads, a, stream);
}

template <int P, int S>
int symmetric_deep(const SymmetricArgs& a, bool second, hipStream_t stream) {
    return second ? launch(symmetric_deep_kernel<P, true, S>, 256, a, stream) : launch(symmetric_deep_kernel<P, false, S>, 256, a, stream);
}

template <int P>
int symmetric(const SymmetricArgs& a, bool second, Kind kind, hipStream_t stream) {
    switch (kind) {
        case kSmall: return symmetric_deep<P, 4>(a, second, stream);
        case kSmallMany: return symmetric_deep<P, 2>(a, second, stream);
        case kMiddle: return symmetric<P, 128, 2, 2, 2>(a, second, stream);
        case kMiddleDeep: return symmetric<P, 128, 2, 2, 4>(a, second, stream);
        default: return symmetric<P, 256, 2, 4>(a, second, stream);
    }
}
template <int P>
int update(const UpdateArgs& a, Kind kind, hipStream_t stream) {
    switch (kind) {
        case kSmall: return launch(update_deep_kernel<P, 4>, 256, a, stream);
        case kSmallMany: return launch(update_deep_kernel<P, 2>, 256, a, stream);
        case kMiddle: return update<P, 128, 2, 2, 2>(a, stream);
        case kMiddleDeep: return update<P, 128, 2, 2, 4>(a, stream);
        default: return update<P, 256, 2, 4>(a, stream);
    }
}

}  // namespace

int launch_symmetric(const SymmetricArgs& a, bool second, int planes, Kind kind, hipStream_t stream) {
    return planes == 2 ? symmetric<2>(a, second, kind, stream) : symmetric<1>(a, second, kind, stream);
}
int launch_update(const UpdateArgs& a, int planes, Kind kind, hipStream_t stream) {
    return planes == 2 ? update<2>(a, kind, stream) : update<1>(a, kind, stream);
}

}  // namespace muon
}  // namespace jabas
