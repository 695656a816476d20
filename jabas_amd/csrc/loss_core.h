// The matrix product under the losses' kernels: a workgroup's tile of out[n][m] = sum_k a[m][k] b[n][k] in registers.
#pragma once

#include "loss_internal.h"

namespace jabas {
namespace loss {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct F16 {
    using vec = f16x8;
    static __device__ f32x16 mfma(vec a, vec b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ vec lowered(vec v) { return v * static_cast<_Float16>(1.0f / kLowScale); }
};
struct BF16 {
    using vec = bf16x8;
    static __device__ f32x16 mfma(vec a, vec b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ vec lowered(vec v) { return v; }      // one plane only
};

// Tile: kM x kN of the output, by WM x WN waves, each kI x kJ blocks of 32 x 32. P planes of an operand. An
// operand lies with its inner axis contiguous (rows of m or n), or, TA / TB, the other way round: rows of k, m or n contiguous.
// RA / RB: a's / b's second plane is kLowScale times what it stands for, so the other's first is made as much smaller for it.
//
// The inner axis goes in steps of 64 elements (two planes: 32 of each) through two stages of LDS. The loads write LDS
// themselves, 16 bytes a lane in lane order, so what keeps banks apart is which element a lane fetches:
//   contiguous inner axis, one plane: rows of 128 bytes, chunk c of row r at c ^ (r / 2 % 8); two planes, each by itself: rows of 64
//     bytes, chunk c at c ^ (r / 4 % 4). A fragment is one 16-byte read of 32 rows, 16 of them at a time over 64 banks.
//     Measured: 230 bytes per clock and CU, against 120 with r % 8;
//   rows of k: chunk c of row k at c ^ 4 (k % 4): the transposing 8-byte reads take four rows and 32 bytes of each at a time.
// The last fragments of a step are in registers before the barrier that gives its stage to the loads of the step after the
// next, and are multiplied behind it, while the next step's first fragments are read: neither the barrier nor the first read
// leaves the matrix cores waiting. Reads and loads go between the products one by one: in a row in front of them they fill the
// LDS and memory pipes and hold the products up (matrix cores busy 75 % of the cycles, 83 % so, at 16384 x 4096 x 4096).
// What bounds it then is power: the clock falls as the cores get busier (1.56 GHz there, 2.1 with LDS and memory idle). Waves of
// 128 x 128, which read LDS a third less, came out even.
// The loads are inline assembly because the compiler would wait for all of them before any later LDS read; they have no
// register outputs, and the wait in front of the barrier covers them.
template <class E, int P, int TM, int TN, int WM, int WN, bool TA, bool TB, bool RA, bool RB>
struct Core {
    static constexpr bool kTa = TA, kTb = TB;
    static constexpr int kM = TM, kN = TN, kThreads = 64 * WM * WN;
    static constexpr int kI = TM / WM / 32, kJ = TN / WN / 32;
    static constexpr int kBytesA = TM * 128, kBytesB = TN * 128, kStage = kBytesA + kBytesB;
    static constexpr int kLoadsA = TM * 8 / kThreads, kLoadsB = TN * 8 / kThreads;
    static constexpr int kStep = P == 2 ? 32 : 64;      // of the inner axis
    static constexpr int kParts = kStep / 16;
    static_assert(kLoadsA % P == 0 && kLoadsB % P == 0, "a load takes one plane");
    using vec = typename E::vec;

    f32x16 acc[kI][kJ];

    static __device__ int wave_m() { return (threadIdx.x >> 6) / WN * (TM / WM); }
    static __device__ int wave_n() { return (threadIdx.x >> 6) % WN * (TN / WN); }
    // element e of a block: m = block_m, n = 32 j + lane % 32; four consecutive e are four consecutive m
    static __device__ int block_m(int i, int e) { return i * 32 + 8 * (e >> 2) + 4 * ((threadIdx.x & 63) >> 5) + (e & 3); }

    // An operand's tile on its way: a uniform base per plane, which moves from step to step, and offsets of the lane's chunks.
    template <int T, bool TR>
    struct Source {
        static constexpr int kLoads = T * 8 / kThreads, kEach = kLoads / P;
        uint64_t base[P];
        int64_t step;
        uint32_t offset[kEach];

        __device__ Source(const Operand& o, int first) {
            const int t = threadIdx.x;
            const uint64_t p = reinterpret_cast<uint64_t>(o.p) + (TR ? 0 : 2 * static_cast<int64_t>(first) * o.stride);
#pragma unroll
            for (int q = 0; q < P; ++q) base[q] = p + 2 * q * o.plane;
            step = 2 * (TR ? kStep * o.stride : kStep);
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int f = i * kThreads + t;                 // the chunk's place in the plane's tile
                if (TR) {
                    const int k = f / (T / 8), c = (f % (T / 8)) ^ ((k & 3) << 2);
                    const int col = min(first + c * 8, o.rows - 8);        // past the end: read again, never written
                    offset[i] = 2 * (static_cast<uint32_t>(k) * static_cast<uint32_t>(o.stride) + col);
                } else {
                    const int r = P == 2 ? f >> 2 : f >> 3, c = P == 2 ? (f & 3) ^ ((r >> 2) & 3) : (f & 7) ^ ((r >> 1) & 7);
                    offset[i] = 2 * (static_cast<uint32_t>(min(first + r, o.rows - 1) - first) * static_cast<uint32_t>(o.stride) + c * 8);
                }
            }
        }
        // Load `l` of kLoads of a step. `to`: byte address in LDS of the operand's stage
        __device__ void issue(uint32_t to, int l) {
            const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x & ~63u);
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                         :: "s"(to + static_cast<uint32_t>(l * kThreads * 16) + wave * 16), "v"(offset[l % kEach]), "s"(base[l / kEach]) : "memory", "m0");
        }
        __device__ void advance() {
#pragma unroll
            for (int q = 0; q < P; ++q) base[q] += step;
        }
    };

    template <int T, bool TR>
    static __device__ vec fragment(const char* tile, int at, int kk, int plane) {
        const int lane = threadIdx.x & 63;
        if (TR) {
            const int k = (P == 2 ? plane * 32 : 0) + kk * 16 + (lane >> 5) * 8 + ((lane & 15) >> 2);
            const int m = at + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
            const int c = (m >> 3) ^ ((k & 3) << 2);
            const char* p = tile + k * (T * 2) + c * 16 + (m & 4) * 2;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + 4 * (T * 2)));
            return __builtin_bit_cast(vec, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
        const int r = at + (lane & 31), c = kk * 2 + (lane >> 5);
        if (P == 2) return *reinterpret_cast<const vec*>(tile + plane * (T * 64) + r * 64 + ((c ^ ((r >> 2) & 3)) * 16));
        return *reinterpret_cast<const vec*>(tile + r * 128 + ((c ^ ((r >> 1) & 7)) * 16));
    }

    struct Fragments {
        vec a[kI][P], b[kJ][P];
    };
    // Fragment `r` of the kReads of a part of a step, those that are multiplied first first.
    static constexpr int kReads = (kI + kJ) * P;
    static __device__ void read(Fragments& f, const char* stage, int kk, int r) {
        const int x = r / P, q = r % P;
        if (x < kJ) f.b[x][q] = fragment<TN, TB>(stage + kBytesA, wave_n() + x * 32, kk, q);
        else f.a[x - kJ][q] = fragment<TM, TA>(stage, wave_m() + (x - kJ) * 32, kk, q);
    }

    // `between(t)` runs behind product t of kProducts.
    static constexpr int kProducts = kI * kJ * (P == 2 ? 3 : 1);
    template <class Between>
    __device__ void multiply(const Fragments& f, const Between& between) {
        int t = 0;
        vec b0[kJ];
#pragma unroll
        for (int j = 0; j < kJ; ++j) b0[j] = RA ? E::lowered(f.b[j][0]) : f.b[j][0];
#pragma unroll
        for (int i = 0; i < kI; ++i) {
            const vec a0 = RB ? E::lowered(f.a[i][0]) : f.a[i][0];
#pragma unroll
            for (int j = 0; j < kJ; ++j) {
                if (P == 2) {       // (a0 + a1)(b0 + b1) without a1 b1, which is under 2^-22 of the whole
                    acc[i][j] = E::mfma(f.a[i][P - 1], b0[j], acc[i][j]);
                    between(t++);
                    acc[i][j] = E::mfma(a0, f.b[j][P - 1], acc[i][j]);
                    between(t++);
                }
                acc[i][j] = E::mfma(f.a[i][0], f.b[j][0], acc[i][j]);
                between(t++);
            }
        }
    }

    static __device__ void arrive() {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }

    // smem: 2 kStage bytes of LDS. `depth`: a multiple of 64, zeros in the operands beyond what counts. `prepare()` runs while the first
    // step's operands are on their way; the sums start from `start(i, e)`, asked behind a barrier that follows it. All waves are
    // past their reads of smem when this returns.
    template <class Prepare, class Start>
    __device__ void run(const Operand& a, const Operand& b, int m0, int n0, int depth, char* smem, const Prepare& prepare, const Start& start) {
        Source<TM, TA> sa(a, m0);
        Source<TN, TB> sb(b, n0);
        const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)smem));
        const auto load = [&](int stage, int l) {
            const uint32_t to = lds + stage * kStage;
            if (l < kLoadsA) sa.issue(to, l);
            else sb.issue(to + kBytesA, l - kLoadsA);
            if (l == kLoadsA + kLoadsB - 1) {
                sa.advance();
                sb.advance();
            }
        };
        const int steps = depth / kStep;        // at least one
        constexpr int kLoads = kLoadsA + kLoadsB;
#pragma unroll
        for (int l = 0; l < kLoads; ++l) load(0, l);
        prepare();
        arrive();
        if (steps > 1)
#pragma unroll
            for (int l = 0; l < kLoads / 2; ++l) load(1, l);
#pragma unroll
        for (int i = 0; i < kI; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float x = start(i, e);
#pragma unroll
                for (int j = 0; j < kJ; ++j) acc[i][j][e] = x;
            }
        Fragments f[2];
#pragma unroll
        for (int r = 0; r < kReads; ++r) read(f[0], smem, 0, r);
        // One step. `next`: there is another, the second half of whose loads goes between the first products; `after`: there is one more, the
        // first half of whose loads goes between the last products, behind the barrier that frees its stage.
        const auto pass = [&](int s, auto next, auto after) {
            const char* stage = smem + (s & 1) * kStage;
#pragma unroll
            for (int kk = 0; kk < kParts; ++kk) {
                const bool first = kk == 0, last = kk + 1 == kParts;
                if (last) arrive();
                __builtin_amdgcn_sched_barrier(0);
                multiply(f[kk & 1], [&](int t) {
                    const auto share = [&](int n, int at) { return min(n, at * n * 5 / (4 * kProducts)); };     // done at four fifths of the products
#pragma unroll
                    for (int r = share(kReads, t); r < share(kReads, t + 1); ++r) {       // of the next part; behind the last step: read, not used
                        if (last) read(f[0], smem + ((s + 1) & 1) * kStage, 0, r);
                        else read(f[(kk + 1) & 1], stage, kk + 1, r);
                    }
                    if (first && next())
#pragma unroll
                        for (int l = kLoads / 2 + t * (kLoads - kLoads / 2) / kProducts; l < kLoads / 2 + (t + 1) * (kLoads - kLoads / 2) / kProducts; ++l) load((s + 1) & 1, l);
                    if (last && after())
#pragma unroll
                        for (int l = t * (kLoads / 2) / kProducts; l < (t + 1) * (kLoads / 2) / kProducts; ++l) load(s & 1, l);
                    __builtin_amdgcn_sched_barrier(0);
                });
            }
        };
        const auto yes = [] { return true; };
        const auto no = [] { return false; };
        int s = 0;
        for (; s + 2 < steps; ++s) pass(s, yes, yes);
        if (s + 1 < steps) pass(s++, yes, no);
        pass(s, no, no);
    }
};

}  // namespace loss
}  // namespace jabas
