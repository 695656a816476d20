// Matrix products of the losses: logits of a tile of tokens and rows that never leave the registers (forward: their
// maxima and sums; backward: the row gradients dz), and the products of dz with the weight and the hidden states.
#include "loss_core.h"

namespace jabas {
namespace loss {
namespace {

__device__ inline float load_as_float(const void* p, int64_t i, int dtype) {
    if (dtype == JABAS_F32) return static_cast<const float*>(p)[i];
    return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(p)[i]) << 16);
}

__device__ inline uint16_t to_bf16(float x) {
    const uint32_t u = __float_as_uint(x);
    if ((u & 0x7fffffffu) > 0x7f800000u) return static_cast<uint16_t>((u >> 16) | 0x40);
    return static_cast<uint16_t>((u + 0x7fffu + ((u >> 16) & 1)) >> 16);
}

template <class C>
__host__ __device__ inline int tiles_m(int m) { return (m + C::kM - 1) / C::kM; }
template <class C>
__host__ __device__ inline int tiles_n(int n) { return (n + C::kN - 1) / C::kN; }

// Tile of a workgroup. Workgroups go round the eight dies (XCDs), each with an L2 of its own: each die takes a run of
// consecutive tiles, in bands of eight tiles of m, so that the 32 tiles in flight on a die share their operands' rows.
__device__ inline void tile_of(int block, int tm, int tn, int& m, int& n) {
    const int total = tm * tn, die = block & 7, each = total >> 3, left = total & 7;
    const int at = die * each + min(die, left) + (block >> 3);
    const int band = at / (8 * tn), first = band * 8, height = min(8, tm - first), in = at - band * 8 * tn;
    m = first + in % height;
    n = in / height;
}

// Which tokens of the tile are entries of which row: the byte of token m and row n, in the word [m / 4][n], is 1 + the entry's
// number. Built over the operands' buffers, which nobody reads any more.
template <class C>
__device__ inline void build_map(const Entries& en, const int32_t* live, char* map, int first, int n0, int rows) {
    const int t = threadIdx.x, lane = t & 63;
    for (int i = t; i < C::kM * C::kN / 16; i += C::kThreads) reinterpret_cast<u32x4*>(map)[i] = u32x4{0, 0, 0, 0};
    __syncthreads();
    constexpr int kWaves = C::kThreads / 64;
    static_assert(C::kN / kWaves <= 64, "a lane for each row of a wave");
    const int here = min(C::kN, rows - n0), wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int32_t mine = wave + kWaves * lane < here ? live[n0 + wave + kWaves * lane] : 0;
#pragma unroll 4
    for (int n = wave; n < here; n += kWaves) {
        const int32_t* index = en.index + static_cast<int64_t>(__builtin_amdgcn_readlane(mine, n / kWaves)) * en.k;
        for (int j = lane; j < en.k; j += 64) {
            const int v = index[j] - first;
            if (v >= 0 && v < C::kM) map[((v >> 2) * C::kN + n) * 4 + (v & 3)] = static_cast<char>(1 + j);
        }
    }
    __syncthreads();
}

// What a tile's logits take besides the product: the tokens' biases and, with two planes, the factors that undo the scaling of their
// rows, in LDS (kM floats each).
template <int P, class C>
__device__ inline void load_tokens(const LogitsArgs& a, int m0, float* tokens) {
    const int m = threadIdx.x;
    if (m >= C::kM) return;
    const int at = min(m0 + m, a.w.rows - 1);
    tokens[m] = a.bias ? load_as_float(a.bias, static_cast<int64_t>(a.first) + at, a.bias_dtype) : 0.0f;
    if (P == 2) tokens[C::kM + m] = a.unscale_w[at];
}

// Nothing read from memory in front of this is kept for what follows: the accumulators leave no room for it.
__device__ inline void keep_order() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
// `x` is computed here, not where it is first used.
__device__ inline void settle(float& x) { asm volatile("" : "+v"(x)); }

// The tile's logits, element e of block (i, j) of the lane. One plane: the sums start from the biases. Plain numbers: the accumulators'
// blocks of 16 registers would be copied whole for every element that changes.
template <class C>
struct Tile {
    float v[C::kI][C::kJ][16];
};
template <int P, class C, class Prepare>
__device__ inline void logits_of(const LogitsArgs& a, int rows, int m0, int n0, char* smem, float* tokens, Tile<C>& z, const Prepare& prepare) {
    const int wm = C::wave_m();
    Operand x = a.x;
    x.rows = rows;
    C c;
    c.run(a.w, x, m0, n0, a.depth, smem, [&] { load_tokens<P, C>(a, m0, tokens); prepare(); },
          [&](int i, int e) { return P == 1 ? tokens[wm + C::block_m(i, e)] : 0.0f; });
#pragma unroll
    for (int j = 0; j < C::kJ; ++j) {
        const float ux = P == 2 ? a.unscale_x[min(n0 + C::wave_n() + j * 32 + static_cast<int>(threadIdx.x & 31), rows - 1)] : 1.0f;
#pragma unroll
        for (int i = 0; i < C::kI; ++i) {
            if (P == 2) keep_order();
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int m = wm + C::block_m(i, e);
                z.v[i][j][e] = P == 2 ? c.acc[i][j][e] * ux * tokens[C::kM + m] + tokens[m] : c.acc[i][j][e];
                if (P == 2) settle(z.v[i][j][e]);
            }
        }
    }
}

// The label of row n of the call (-1: none) as a token of the tile, or -1.
template <class C>
__device__ inline int label_of(const LogitsArgs& a, int m0, int n) {
    if (n < 0) return -1;
    const int64_t label = a.entries.target[n] - a.first - m0;
    return label >= 0 && label < C::kM ? static_cast<int>(label) : -1;
}

// f(i, e) for the element of this lane's block column that is token `label` of the tile, if one is. Few waves hold one: the others
// pay a compare.
template <class C, class F>
__device__ inline void at_label(int label, const F& f) {
    const int mine = label - C::wave_m();
    if (!__any(label >= 0 && mine >= 0 && mine < C::kI * 32)) return;
    const int at = label < 0 ? -1000 : mine - 4 * ((threadIdx.x & 63) >> 5);
#pragma unroll
    for (int i = 0; i < C::kI; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (at == i * 32 + 8 * (e >> 2) + (e & 3)) f(i, e);
}

// Forward: a tile's product, then per row its maximum and the sum of 2^((z - max) c) over the tile's tokens, so that 16 bytes a row and tile
// leave the chip instead of the logits. Matrix cores bind it, and the clock they leave: 4096 x 131072 x 4096 bf16 3.2 ms, 1.38 PFLOP/s,
// cores busy 79 % of the cycles at 1.65 GHz; with an inner axis of 768 to 1024 the start and the exponentials of a tile weigh more:
// 4099 x 50001 x 768 bf16 328 us, 0.96; 1280 x 32317 x 1024 fp32 287 us, 0.88 (three products).
template <class E, int P, class C, bool TEACHER>
__global__ __launch_bounds__(C::kThreads) void logits_forward_kernel(LogitsArgs a) {
    __shared__ __align__(16) char smem[2 * C::kStage];
    __shared__ float tokens[P * C::kM];
    const int rows = *a.rows.live, across = tiles_m<C>(a.w.rows);
    if (static_cast<int>(blockIdx.x) >= across * tiles_n<C>(rows)) return;
    int tm, tn;
    tile_of(blockIdx.x, across, tiles_n<C>(rows), tm, tn);
    const int m0 = tm * C::kM, n0 = tn * C::kN, lane = threadIdx.x & 63;
    const int wm = C::wave_m(), wn = C::wave_n();
    int row[C::kJ], label[C::kJ];       // rows of the call and their labels, asked for while the first operands are on their way
    Tile<C> z;
    logits_of<P>(a, rows, m0, n0, smem, tokens, z, [&] {
#pragma unroll
        for (int j = 0; j < C::kJ; ++j) {
            const int n = n0 + wn + j * 32 + (lane & 31);
            row[j] = n < rows ? a.rows.map[n] : -1;
            label[j] = TEACHER ? -1 : label_of<C>(a, m0, row[j]);
        }
    });
    float peak[C::kJ], sum[C::kJ], total[C::kJ];
    if (m0 + C::kM > a.w.rows) {        // tokens past the end
#pragma unroll
        for (int i = 0; i < C::kI; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const bool in = m0 + wm + C::block_m(i, e) < a.w.rows;
#pragma unroll
                for (int j = 0; j < C::kJ; ++j)
                    if (!in) z.v[i][j][e] = -INFINITY;
            }
    }
    if (TEACHER) build_map<C>(a.entries, a.rows.map, smem, a.first + m0, n0, rows);
#pragma unroll
    for (int j = 0; j < C::kJ; ++j) {
        const int nl = wn + j * 32 + (lane & 31), n = row[j];
        total[j] = 0.0f;
        if (TEACHER) {          // entries join their row later, each by itself
#pragma unroll
            for (int i = 0; i < C::kI; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t hits = reinterpret_cast<const uint32_t*>(smem)[((wm + C::block_m(i, q * 4)) >> 2) * C::kN + nl];
                    if (hits)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t hit = (hits >> (8 * e)) & 0xff;
                            if (hit) {
                                a.entry_logit[static_cast<int64_t>(n) * a.entries.k + hit - 1] = z.v[i][j][q * 4 + e];
                                z.v[i][j][q * 4 + e] = -INFINITY;
                            }
                        }
                }
        } else {
            at_label<C>(label[j], [&](int i, int e) { a.entry_logit[n] = z.v[i][j][e]; });
            if (a.total) {
#pragma unroll
                for (int i = 0; i < C::kI; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) total[j] += m0 + C::kM <= a.w.rows || m0 + wm + C::block_m(i, e) < a.w.rows ? z.v[i][j][e] : 0.0f;
                total[j] += __shfl_xor(total[j], 32);
            }
        }
        peak[j] = -INFINITY;
#pragma unroll
        for (int i = 0; i < C::kI; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) peak[j] = fmaxf(peak[j], z.v[i][j][e]);
        peak[j] = fmaxf(peak[j], __shfl_xor(peak[j], 32));
        const float base = peak[j] == -INFINITY ? 0.0f : peak[j];
        sum[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < C::kI; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) sum[j] += __builtin_amdgcn_exp2f((z.v[i][j][e] - base) * a.c);
        sum[j] += __shfl_xor(sum[j], 32);
    }
    // the waves that share rows: [wave of m][row of the tile]
    constexpr int kWaves = C::kM / (C::kI * 32);
    float* merge = reinterpret_cast<float*>(smem);
    __syncthreads();
    if (lane < 32)
#pragma unroll
        for (int j = 0; j < C::kJ; ++j) {
            float* at = merge + (wm / (C::kI * 32)) * C::kN + wn + j * 32 + lane;
            at[0] = peak[j];
            at[kWaves * C::kN] = sum[j];
            at[2 * kWaves * C::kN] = total[j];
        }
    __syncthreads();
    const int nl = threadIdx.x, n = n0 + nl;
    if (nl >= C::kN || n >= rows) return;
    float p = merge[nl], s = 0.0f, t = 0.0f;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) p = fmaxf(p, merge[w * C::kN + nl]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const float part = merge[(kWaves + w) * C::kN + nl];
        if (part != 0.0f) s += part * __builtin_amdgcn_exp2f((merge[w * C::kN + nl] - p) * a.c);
        t += merge[(2 * kWaves + w) * C::kN + nl];
    }
    const int64_t at = static_cast<int64_t>(a.first / C::kM + tm) * a.x.rows + n;
    a.partial[at] = make_float2(p, s);
    if (a.total) a.total[at] = t;
}

// Sums over 32 lanes of 32 values a lane, half of them handed over at every step: lane l ends with the sum of value l % 32 in
// v[0].
template <int HALF>
__device__ inline void scatter_sum(float (&v)[32]) {
    const bool upper = threadIdx.x & HALF;
#pragma unroll
    for (int i = 0; i < HALF; ++i) {
        const float give = upper ? v[i] : v[i + HALF], keep = upper ? v[i + HALF] : v[i];
        v[i] = keep + __shfl_xor(give, HALF);
    }
    if constexpr (HALF > 1) scatter_sum<HALF / 2>(v);
}

// Backward: the same product, and dz = slope 2^((z - peak) c) - what the label or the entries take off, written once as fp16 through LDS, 16
// bytes a lane. db's sums over a tile's rows are taken here, in 32 bits, where dz is still exact. Bound by the matrix cores
// as the forward pass: 4096 x 16384 x 4096 bf16 442 us, 1.25 PFLOP/s; 1280 x 32317 x 1024 fp32 317 us, 0.80.
template <class E, int P, class C, bool TEACHER>
__global__ __launch_bounds__(C::kThreads) void logits_backward_kernel(LogitsArgs a) {
    __shared__ __align__(16) char smem[2 * C::kStage];
    __shared__ float tokens[P * C::kM];
    const int rows = *a.rows.live, across = tiles_m<C>(a.w.rows);
    if (static_cast<int>(blockIdx.x) >= across * tiles_n<C>(rows)) return;
    int tm, tn;
    tile_of(blockIdx.x, across, tiles_n<C>(rows), tm, tn);
    const int m0 = tm * C::kM, n0 = tn * C::kN, lane = threadIdx.x & 63;
    const int wm = C::wave_m(), wn = C::wave_n();
    int row[C::kJ], label[C::kJ];       // as in the forward pass
    Tile<C> z;
    logits_of<P>(a, rows, m0, n0, smem, tokens, z, [&] {
#pragma unroll
        for (int j = 0; j < C::kJ; ++j) {
            const int n = n0 + wn + j * 32 + (lane & 31);
            row[j] = n < rows ? a.rows.map[n] : -1;
            label[j] = TEACHER ? -1 : label_of<C>(a, m0, row[j]);
        }
    });
    if (TEACHER) build_map<C>(a.entries, a.rows.map, smem, a.first + m0, n0, rows);
#pragma unroll
    for (int j = 0; j < C::kJ; ++j) {
        keep_order();
        const int nl = wn + j * 32 + (lane & 31), n = row[j];
        const float scale = TEACHER && n >= 0 ? kDzScale * a.down[n] : kDzScale, uniform = TEACHER ? 0.0f : a.uniform * kDzScale;
        const RowState st = n >= 0 ? a.state[n] : RowState{0.0f, 0.0f, 0.0f, 0.0f};
        const bool counts = !(st.slope == 0.0f && st.mass == 0.0f);
        const float slope = st.slope * scale;
#pragma unroll
        for (int i = 0; i < C::kI; ++i) {
            if (P == 2) keep_order();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint32_t hits = TEACHER ? reinterpret_cast<const uint32_t*>(smem)[((wm + C::block_m(i, q * 4)) >> 2) * C::kN + nl] : 0;
                float d[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) d[e] = fmaf(slope, __builtin_amdgcn_exp2f((z.v[i][j][q * 4 + e] - st.peak_rest) * a.c), -uniform);
                if (TEACHER && hits)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t hit = (hits >> (8 * e)) & 0xff;
                        if (hit)
                            d[e] = (st.mass * __builtin_amdgcn_exp2f((z.v[i][j][q * 4 + e] - st.peak) * a.c) -
                                    a.entries.p[static_cast<int64_t>(n) * a.entries.k + hit - 1]) * scale;
                    }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    z.v[i][j][q * 4 + e] = d[e];
                    if (P == 2) settle(z.v[i][j][q * 4 + e]);
                }
            }
        }
        if (!TEACHER) at_label<C>(label[j], [&](int i, int e) { z.v[i][j][e] -= a.hit * scale; });
        if (__any(!counts)) {
#pragma unroll
            for (int i = 0; i < C::kI; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) z.v[i][j][e] = counts ? z.v[i][j][e] : 0.0f;
        }
    }
    if (m0 + C::kM > a.w.rows) {        // tokens past the end
#pragma unroll
        for (int i = 0; i < C::kI; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const bool in = m0 + wm + C::block_m(i, e) < a.w.rows;
#pragma unroll
                for (int j = 0; j < C::kJ; ++j)
                    if (!in) z.v[i][j][e] = 0.0f;
            }
    }
    if (a.db) {      // sums over this tile's rows: within the wave, then over the waves that share tokens
        __syncthreads();
        float* merge = reinterpret_cast<float*>(smem);
        float g[C::kJ];
#pragma unroll
        for (int j = 0; j < C::kJ; ++j) {
            g[j] = row[j] >= 0 ? a.row_grad[row[j]] * (1.0f / kDzScale) : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < C::kI; i += 2) {
            float v[32];
#pragma unroll
            for (int x = 0; x < 32; ++x) {
                v[x] = 0.0f;
#pragma unroll
                for (int j = 0; j < C::kJ; ++j) v[x] += z.v[i + (x >> 4)][j][x & 15] * g[j];
            }
            scatter_sum<16>(v);
            merge[wn / (C::kJ * 32) * C::kM + wm + C::block_m(i + ((lane & 31) >> 4), lane & 15)] = v[0];
        }
        __syncthreads();
        const int m = threadIdx.x;
        if (m < C::kM && m0 + m < a.w.rows) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < C::kN / (C::kJ * 32); ++w) s += merge[w * C::kM + m];
            a.db[static_cast<int64_t>(tn) * a.w.rows + m0 + m] = s;
        }
    }
    if (!a.dz) return;
    const int pad_rows = (rows + kDepth - 1) / kDepth * kDepth;
    __syncthreads();
    // The wave's part of dz through LDS, so that lanes write 16 consecutive bytes of a row: row n of kChunks chunks, chunk k at k ^ n % kChunks.
    constexpr int kRows = C::kJ * 32, kChunks = C::kI * 32 / 8;
    char* mine = smem + (threadIdx.x >> 6) * (kRows * kChunks * 16);
    if (P == 2) {       // both planes of an element in the register that held it
#pragma unroll
        for (int j = 0; j < C::kJ; ++j)
#pragma unroll
            for (int i = 0; i < C::kI; ++i) {
                keep_order();
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const _Float16 hi = static_cast<_Float16>(z.v[i][j][e]);
                    const _Float16 lo = static_cast<_Float16>((z.v[i][j][e] - static_cast<float>(hi)) * kLowScale);
                    z.v[i][j][e] = __uint_as_float(__builtin_bit_cast(uint16_t, hi) | static_cast<uint32_t>(__builtin_bit_cast(uint16_t, lo)) << 16);
                    settle(z.v[i][j][e]);
                }
            }
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
#pragma unroll
        for (int j = 0; j < C::kJ; ++j)
#pragma unroll
            for (int i = 0; i < C::kI; ++i) {
                keep_order();
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    f16x4 h;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float v = z.v[i][j][q * 4 + e];
                        h[e] = P == 2 ? __builtin_bit_cast(_Float16, static_cast<uint16_t>(__float_as_uint(v) >> (16 * p))) : static_cast<_Float16>(v);
                    }
                    const int r = j * 32 + (lane & 31), m = C::block_m(i, q * 4);
                    *reinterpret_cast<f16x4*>(mine + (r * kChunks + ((m >> 3) ^ (r % kChunks))) * 16 + (m & 4) * 2) = h;
                }
            }
        uint16_t* out = static_cast<uint16_t*>(a.dz) + p * a.dz_plane;
#pragma unroll 4
        for (int x = 0; x < kRows * kChunks / 64; ++x) {
            const int f = x * 64 + lane, r = f / kChunks, k = f % kChunks;
            const u32x4 v = *reinterpret_cast<const u32x4*>(mine + (r * kChunks + (k ^ (r % kChunks))) * 16);
            const int n = n0 + wn + r, m = m0 + wm + k * 8;
            if (n < pad_rows && m < a.pad_tokens) *reinterpret_cast<u32x4*>(out + static_cast<int64_t>(n) * a.dz_stride + m) = v;
        }
    }
}

// Results of four consecutive m of a row.
__device__ inline void put_four(const Job& a, int n, int m, f32x4 v) {
    const int here = min(4, a.m - m);
    if (a.live_n) n = a.rows.map[n];
    if (a.row_scale) v *= a.row_scale[n];
    const int64_t at = static_cast<int64_t>(n) * a.out_stride + m;
    if (a.out_dtype == JABAS_F32) {
        float* out = static_cast<float*>(a.out) + at;
        if (a.out_aligned) *reinterpret_cast<f32x4*>(out) = v;
        else
            for (int e = 0; e < here; ++e) out[e] = v[e];
    } else {
        uint16_t* out = static_cast<uint16_t*>(a.out) + at;
        const uint16_t h[4] = {to_bf16(v[0]), to_bf16(v[1]), to_bf16(v[2]), to_bf16(v[3])};
        if (a.out_aligned) *reinterpret_cast<uint64_t*>(out) = h[0] | static_cast<uint64_t>(h[1]) << 16 | static_cast<uint64_t>(h[2]) << 32 | static_cast<uint64_t>(h[3]) << 48;
        else
            for (int e = 0; e < here; ++e) out[e] = h[e];
    }
}

__device__ inline int live_or(const Job& a, int32_t is_live, int otherwise) { return is_live ? *a.rows.live : otherwise; }

template <class C>
__device__ inline void run_job(const Job& a, int unit, char* smem) {
    const int n_here = live_or(a, a.live_n, a.n), depth = (live_or(a, a.live_depth, a.depth) + kDepth - 1) / kDepth * kDepth;
    const int tiles = tiles_m<C>(a.m) * tiles_n<C>(n_here), split = unit / tiles;
    int tm, tn;
    tile_of(unit - split * tiles, tiles_m<C>(a.m), tiles_n<C>(n_here), tm, tn);
    const int m0 = tm * C::kM, n0 = tn * C::kN, lane = threadIdx.x & 63;
    Operand x = a.a, y = a.b;
    const int k0 = split * a.each;
    x.p = static_cast<const uint16_t*>(x.p) + (C::kTa ? k0 * x.stride : k0);
    y.p = static_cast<const uint16_t*>(y.p) + (C::kTb ? k0 * y.stride : k0);
    if (a.live_n) y.rows = n_here;
    C c;
    if (k0 < depth) {
        c.run(x, y, m0, n0, min(a.each, depth - k0), smem, [] {}, [](int, int) { return 0.0f; });
    } else {        // fewer rows count than the splits were made for
#pragma unroll
        for (int i = 0; i < C::kI; ++i)
#pragma unroll
            for (int j = 0; j < C::kJ; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) c.acc[i][j][e] = 0.0f;
    }
    const int wm = C::wave_m(), wn = C::wave_n();
    float scale = a.scale;
    if (a.unscale0) scale *= *a.unscale0;
    const float second = a.unscale1 ? *a.unscale1 : 1.0f;
    float* part = a.part ? a.part + split * a.part_plane : nullptr;
    // 32 rows of the wave at a time through LDS: row n of kChunks 16-byte chunks, chunk k at k ^ n % kChunks
    constexpr int kChunks = C::kI * 32 / 4;
    float* mine = reinterpret_cast<float*>(smem + (threadIdx.x >> 6) * (32 * kChunks * 16));
    __syncthreads();
#pragma unroll
    for (int j = 0; j < C::kJ; ++j) {
#pragma unroll
        for (int i = 0; i < C::kI; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = c.acc[i][j][q * 4 + e] * scale * second;    // the pieces of a sum have scales of their own
                const int r = lane & 31, m = C::block_m(i, q * 4);
                *reinterpret_cast<f32x4*>(mine + (r * kChunks + ((m >> 2) ^ (r % kChunks))) * 4) = v;
            }
#pragma unroll
        for (int x = 0; x < 32 * kChunks / 64; ++x) {
            const int f = x * 64 + lane, r = f / kChunks, k = f % kChunks;
            f32x4 v = *reinterpret_cast<const f32x4*>(mine + (r * kChunks + (k ^ (r % kChunks))) * 4);
            const int n = n0 + wn + j * 32 + r, m = m0 + wm + k * 4;
            if (n >= n_here || m >= a.m) continue;
            if (a.unscale_m) v *= *reinterpret_cast<const f32x4*>(a.unscale_m + m);
            if (part) {
                float* sum = part + static_cast<int64_t>(n) * a.part_stride + m;       // rows padded to four
                if (!a.first) v += *reinterpret_cast<const f32x4*>(sum);
                if (a.keep) {
                    *reinterpret_cast<f32x4*>(sum) = v;
                    continue;
                }
            }
            put_four(a, n, m, v);
        }
    }
}

// dW and dX of a piece in one launch, the longer units first, so that neither's last round leaves CUs idle. dz is the right operand of
// both: rows of k for dW, through transposing reads, and as it lies for dX. Bound by the matrix cores: 4096 x 16384 x 4096 bf16
// 926 us, 1.19 PFLOP/s (dW and dX alone take the same each); 1280 x 32317 x 1024 fp32 498 us, 1.02.
template <class CW, class CH>
__global__ __launch_bounds__(CW::kThreads) void grads_kernel(GradArgs a) {
    static_assert(CW::kStage == CH::kStage && CW::kThreads == CH::kThreads, "one launch shape");
    __shared__ __align__(16) char smem[2 * CW::kStage];
    const int units_w = tiles_m<CW>(a.w.m) * tiles_n<CW>(a.w.n) * a.w.splits;
    const int units_h = tiles_m<CH>(a.h.m) * tiles_n<CH>(live_or(a.h, a.h.live_n, a.h.n)) * a.h.splits;
    const int block = blockIdx.x, lead = a.h_first ? units_h : units_w;
    if (block >= units_w + units_h) return;
    if ((block < lead) == (a.h_first != 0)) run_job<CH>(a.h, a.h_first ? block : block - lead, smem);
    else run_job<CW>(a.w, a.h_first ? block - lead : block, smem);
}

// Bound by memory: 5120 rows x 1024 from 5 splits 13 us, 1600 x 1024 from 4 9 us.
__global__ __launch_bounds__(256) void join_splits_kernel(Job a) {
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int quads = (a.m + 3) / 4, n = static_cast<int>(at / quads), m = static_cast<int>(at % quads) * 4;
    if (n >= live_or(a, a.live_n, a.n)) return;
    const float* part = a.part + n * a.part_stride + m;
    f32x4 v = *reinterpret_cast<const f32x4*>(part);
    for (int i = 1; i < a.splits; ++i) v += *reinterpret_cast<const f32x4*>(part + i * a.part_plane);
    put_four(a, n, m, v);
}

template <class K, class A>
int launch(K kernel, int64_t grid, int threads, const A& args, hipStream_t stream) {
    void* params[] = {const_cast<A*>(&args)};
    return hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3(static_cast<unsigned>(grid)), dim3(threads), params, 0, stream) == hipSuccess
               ? JABAS_OK : JABAS_ERR_LAUNCH;
}

template <class E, int P, int TM, int TN, int WM, int WN>
int logits(const LogitsArgs& a, bool backward, hipStream_t stream) {
    using C = Core<E, P, TM, TN, WM, WN, false, false, P == 2, false>;
    const int64_t grid = static_cast<int64_t>(tiles_m<C>(a.w.rows)) * tiles_n<C>(a.x.rows);
    if (a.entries.index)
        return backward ? launch(logits_backward_kernel<E, P, C, true>, grid, C::kThreads, a, stream) : launch(logits_forward_kernel<E, P, C, true>, grid, C::kThreads, a, stream);
    return backward ? launch(logits_backward_kernel<E, P, C, false>, grid, C::kThreads, a, stream) : launch(logits_forward_kernel<E, P, C, false>, grid, C::kThreads, a, stream);
}

int logits(const LogitsArgs& a, int planes, bool large, bool backward, hipStream_t stream) {
    if (planes == 2) return large ? logits<F16, 2, 256, 256, 2, 4>(a, backward, stream) : logits<F16, 2, 128, 128, 2, 2>(a, backward, stream);
    return large ? logits<BF16, 1, 256, 256, 2, 4>(a, backward, stream) : logits<BF16, 1, 128, 128, 2, 2>(a, backward, stream);
}

template <int P, int TM, int TN, int WM, int WN>
int grads(const GradArgs& a, hipStream_t stream) {
    using CW = Core<F16, P, TM, TN, WM, WN, false, true, false, P == 2>;
    using CH = Core<F16, P, TM, TN, WM, WN, P == 2, false, P == 2, P == 2>;
    const int64_t grid = static_cast<int64_t>(tiles_m<CW>(a.w.m)) * tiles_n<CW>(a.w.n) * a.w.splits + static_cast<int64_t>(tiles_m<CH>(a.h.m)) * tiles_n<CH>(a.h.n) * a.h.splits;
    return launch(grads_kernel<CW, CH>, grid, CW::kThreads, a, stream);
}

struct Sizes { int m, n; };
// Tiles of the gradients' products. Small ones where a side is one of them, and for less than 12e9 products of either: forward and
// backward, small and large, 256 x 32317 x 1024 fp32 548 and 579 us, bf16 206 and 200; 6400 x 1000 x 768 fp32 252 and 278, bf16 143
// and 150; 1600 x 8192 x 1024 fp32 476 and 463, bf16 205 and 198; 512 x 32317 x 1024 bf16 292 and 277; 128 x 16384 x 1024 fp32 257 and 280.
bool large_grads(int64_t features, int64_t tokens, int64_t rows) {
    return features > 128 && rows > 128 && static_cast<double>(features) * tokens * rows >= 12e9;
}
Sizes grads_tile(bool large) { return large ? Sizes{256, 256} : Sizes{128, 128}; }

}  // namespace

// A CU holds one workgroup of a large tile or two of a small one, whose round takes 0.6 of a large one's, or 0.55 behind fp32's backward
// pass, whose large tile runs out of registers (112 bytes a lane go to scratch memory, 56 with entries; 48 in fp32's forward pass). Forward, then forward and backward, small and large, by 1024: 512 x 16384 (128 large tiles)
// fp32 106 and 118 us; 512 x 32317 (254) fp32 185 and 170, 710 and 669, bf16 64.7 and 56.6, 286 and 274; 640 x 32317 (381) 231 and 237,
// 829 and 876, 79 and 83, 341 and 349; 1280 x 32317 (635) 345 and 331, 1266 and 1286, 124 and 118, 496 and 491; 5120 x 32317 (2540) 1072
// and 962, 4143 and 3988, 386 and 344, 1521 and 1430. 256 x 128 was no faster than the better of the two at any of these.
bool large_tiles(int64_t tokens, int64_t rows, int planes, bool backward) {
    const auto rounds = [&](int64_t tile, int64_t slots) { return ((tokens + tile - 1) / tile * ((rows + tile - 1) / tile) + slots - 1) / slots; };
    return rounds(128, 512) * (planes == 2 && backward ? 0.55 : 0.6) >= rounds(256, 256);
}
int logits_tile(bool large) { return large ? 256 : 128; }

int launch_logits_forward(const LogitsArgs& a, int planes, bool large, hipStream_t stream) { return logits(a, planes, large, false, stream); }
int launch_logits_backward(const LogitsArgs& a, int planes, bool large, hipStream_t stream) { return logits(a, planes, large, true, stream); }

// Time, in steps of a tile, that `slots` workgroups take for `na` units of length `la`, then `nb` of length `lb`, each taken by whoever is
// free first. Workgroups that get free together are counted together.
namespace {
double makespan(int slots, int64_t na, double la, int64_t nb, double lb) {
    struct Group { double free; int64_t n; } g[64] = {{0.0, slots}};
    int groups = 1;
    double end = 0.0;
    for (int kind = 0; kind < 2; ++kind) {
        int64_t left = kind ? nb : na;
        const double length = kind ? lb : la;
        while (left > 0) {
            int at = 0;
            for (int i = 1; i < groups; ++i)
                if (g[i].free < g[at].free) at = i;
            if (groups == 1 && left > 8 * g[0].n) {     // whole rounds of one kind
                const int64_t rounds = left / g[0].n - 4;
                g[0].free += rounds * length;
                left -= rounds * g[0].n;
                continue;
            }
            const int64_t take = left < g[at].n ? left : g[at].n;
            const double until = g[at].free + length;
            left -= take;
            if (until > end) end = until;
            if (take == g[at].n) {
                g[at].free = until;
            } else {
                g[at].n -= take;
                if (groups == 64) return end + left * length / slots;
                g[groups++] = {until, take};
            }
            for (int i = 0; i < groups; ++i)            // those that are free at one time, together
                for (int j = i + 1; j < groups; ++j)
                    if (g[i].free == g[j].free) {
                        g[i].n += g[j].n;
                        g[j--] = g[--groups];
                    }
        }
    }
    return end;
}
}  // namespace

// The split that the model above says ends first. A unit costs its steps of 64 elements and kUnit more for its start and its results; fp32
// sums that are written, read and joined cost what their bytes take of the chip's bandwidth (a step of a 256 x 256 tile is 1.8 us at
// 1.2 PFLOP/s, in which HBM moves 9 MB). Forward and backward,
// fp32, without splits and with those chosen: 100 x 16384 x 1024 615 and 250 us, 256 x 32317 2201 and 581, 1600 x 32317 2896 and 1637,
// 6400 x 32317 5288 and 5365; none of 2, 4, 8 or 16 splits of dX alone is over 4 % faster than the choice, bf16 included.
Splits choose_splits(int64_t features, int64_t tokens, int64_t rows, bool w, bool h, bool many_pieces, int planes) {
    const bool large = large_grads(features, tokens, rows);
    const Sizes t = grads_tile(large);
    const int slots = large ? 256 : 512;
    const double kUnit = 6.0, bytes_per_step = (large ? 9e6 : 4.5e6) * (planes == 2 ? 3 : 1);
    const int64_t fm = (features + t.m - 1) / t.m, tw = w ? fm * ((tokens + t.n - 1) / t.n) : 0, th = h ? fm * ((rows + t.n - 1) / t.n) : 0;
    const double kw = (rows + 63) / 64, kh = (tokens + 63) / 64;
    Splits best = {1, 1};
    double least = 0.0;
    static const int kTries[] = {1, 2, 3, 4, 5, 6, 8, 12, 16};
    for (int sw : kTries)
        for (int sh : kTries) {
            if (sw > (w && tw < 2 * slots ? 4 : 1) || sh > (h && th < 2 * slots ? 16 : 1) || (sw > 1 && kw / sw < 4) || (sh > 1 && kh / sh < 4)) continue;
            const double lw = kw / sw + kUnit, lh = kh / sh + kUnit;
            double time = lh > lw ? makespan(slots, th * sh, lh, tw * sw, lw) : makespan(slots, tw * sw, lw, th * sh, lh);
            const double sums_w = sw > 1 ? 4.0 * features * tokens * sw * 2 : 0.0;
            const double sums_h = sh > 1 || many_pieces ? 4.0 * features * rows * sh * 2 : 0.0;
            time += (sums_w + sums_h) / bytes_per_step;
            if ((sw == 1 && sh == 1) || time < least * 0.98) {
                least = time;
                best = {sw, sh};
            }
        }
    return best;
}

int launch_grads(GradArgs& a, int planes, hipStream_t stream) {
    const int64_t features = a.w.m > a.h.m ? a.w.m : a.h.m;
    a.h_first = !a.w.m || (a.h.m && a.h.each > a.w.each);
    const bool large = large_grads(features, a.w.m ? a.w.n : a.h.depth, a.h.m ? a.h.n : a.w.depth);
    if (planes == 2) return large ? grads<2, 256, 256, 2, 4>(a, stream) : grads<2, 128, 128, 2, 2>(a, stream);
    return large ? grads<1, 256, 256, 2, 4>(a, stream) : grads<1, 128, 128, 2, 2>(a, stream);
}

int launch_join_splits(const Job& j, hipStream_t stream) {
    return launch(join_splits_kernel, (static_cast<int64_t>((j.m + 3) / 4) * j.n + 255) / 256, 256, j, stream);
}

// ------------------------------------------------------------------ layout of operands
namespace {

constexpr int kLayThreads = 256;

// The power of two that takes `peak` to [2^14, 2^15): both planes of an element then fit fp16, elements down to 2^-16
// of the largest keep 22 bits, and smaller ones are off by 2^-40 of it at most. With a second plane that is raised by kLowScale they are off by
// 2^-51: the weight's is, because the backward pass takes a piece of it by one scale for the product that sums over the tokens, and a weight
// of 1e6 among others of 0.03 would leave their logits at 4e-5 where the forward pass, a scale per token, has them at 1e-7. What it costs is
// one more multiplication of the other operand's fragments: 1600 x 32317 x 1024 1.5 % of a pass.
__device__ inline int scale_exponent(float peak) {
    if (!(peak > 0.0f)) return 0;
    int e = static_cast<int>((__float_as_uint(peak) >> 23) & 0xff) - 126;
    return min(max(15 - e, -126), 126);
}
__device__ inline float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

__device__ inline float finite_size(float x) {
    const float s = fabsf(x);
    return s < INFINITY ? s : 0.0f;     // infinities and NaN do not set the scale
}

__device__ inline float wave_max(float x) {
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) x = fmaxf(x, __shfl_xor(x, i));
    return x;
}

// Eight elements of a row from column c on, zeros past the end; any alignment.
struct __attribute__((packed, aligned(2))) Eight16 { uint16_t v[8]; };
struct __attribute__((packed, aligned(4))) Eight32 { float v[8]; };
__device__ inline void load_eight(const LayArgs& a, int64_t row, int c, float (&v)[8]) {
    const int64_t at = row * a.in_stride + c;
    if (c + 8 <= a.cols) {
        if (a.in_dtype == JABAS_F32) {
            const Eight32 x = *reinterpret_cast<const Eight32*>(static_cast<const float*>(a.in) + at);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = x.v[i];
        } else {
            const Eight16 x = *reinterpret_cast<const Eight16*>(static_cast<const uint16_t*>(a.in) + at);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(static_cast<uint32_t>(x.v[i]) << 16);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < a.cols ? load_as_float(a.in, at + i, a.in_dtype) : 0.0f;
    }
}

__device__ inline void store_eight(const LayArgs& a, int64_t row, int c, const float (&v)[8]) {
    _Float16* p = static_cast<_Float16*>(a.out) + row * a.out_stride + c;
    f16x8 hi, lo;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        hi[i] = static_cast<_Float16>(v[i]);
        const float f = static_cast<float>(hi[i]);
        lo[i] = static_cast<_Float16>(fabsf(f) < INFINITY ? (v[i] - f) * a.low : 0.0f);
    }
    *reinterpret_cast<f16x8*>(p) = hi;
    if (a.planes == 2) *reinterpret_cast<f16x8*>(p + a.out_plane) = lo;
}

__device__ inline float row_keeps(const LayArgs& a, int row) {
    if (a.row_mask && load_as_float(a.row_mask, row, a.in_dtype) == -INFINITY) {
        const int token = a.first + row;
        if (!((a.named[token >> 5] >> (token & 31)) & 1)) return 0.0f;
    }
    return a.row_factor ? a.row_factor[row] : 1.0f;
}

// Row r that is laid out: rows and places.
__device__ inline int rows_of(const LayArgs& a) { return a.live.live ? *a.live.live : a.rows; }
__device__ inline int row_of(const LayArgs& a, int r) { return a.live.map ? a.live.map[r] : r; }

// The tokens that a row of the call has a dz of its own for, whatever rules them out, by one wave.
__device__ inline void name_tokens(const LayArgs& a, int row, int lane) {
    const auto name = [&](int64_t token) {
        if (token >= 0 && token < a.vocab) atomicOr(a.name + (token >> 5), 1u << (token & 31));
    };
    if (!a.entries.index) {
        if (lane == 0) name(a.entries.target[row]);
        return;
    }
    const int64_t first = static_cast<int64_t>(row) * a.entries.k;
    for (int j = lane; j < a.entries.k; j += 64)
        if (a.entries.p[first + j] != 0.0f) name(a.entries.index[first + j]);
}

// The largest of the partial maxima, for every thread of the workgroup.
__device__ inline float join_parts(const float* parts) {
    __shared__ float merge[kLayThreads / 64];
    static_assert(kMaxParts % kLayThreads == 0, "as many partial maxima per thread");
    float peak = 0.0f;
#pragma unroll
    for (int i = 0; i < kMaxParts; i += kLayThreads) peak = fmaxf(peak, parts[i + threadIdx.x]);
    peak = wave_max(peak);
    if ((threadIdx.x & 63) == 0) merge[threadIdx.x >> 6] = peak;
    __syncthreads();
    return fmaxf(fmaxf(merge[0], merge[1]), fmaxf(merge[2], merge[3]));
}

// One wave per row: padded, and scaled by the row's own power of two, or all by one. Bound by memory: 32317 x 1024 fp32, 132 MB read and as
// much written, 50 us (5.3 TB/s); a row's second read comes from the caches.
__global__ __launch_bounds__(kLayThreads) void lay_rows_kernel(LayArgs a) {
    const int place = blockIdx.x * (kLayThreads / 64) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (a.parts) {
        const int e = scale_exponent(join_parts(a.parts));
        if (place >= a.pad_rows) return;
        const float scale = place < a.rows ? row_keeps(a, place) * power_of_two(e) : 0.0f;
        float v[8];
        for (int c = lane * 8; c < a.pad; c += 512) {
            if (scale != 0.0f) load_eight(a, place, c, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = scale != 0.0f ? v[i] * scale : 0.0f;
            store_eight(a, place, c, v);
        }
        if (lane == 0 && place < a.rows) a.unscale[place] = power_of_two(-e);
        if (lane == 0 && place == 0) *a.unscale_all = power_of_two(-e);
        return;
    }
    if (place >= a.rows) return;
    const int row = row_of(a, place);
    if (place >= rows_of(a)) {
        if (!a.zero) return;
        const int64_t bytes = static_cast<int64_t>(a.cols) * (a.in_dtype == JABAS_F32 ? 4 : 2);
        uint16_t* out = reinterpret_cast<uint16_t*>(static_cast<char*>(a.zero) + row * bytes);
        for (int64_t i = lane; i < bytes / 2; i += 64) out[i] = 0;
        return;
    }
    if (a.name) name_tokens(a, row, lane);
    if (a.planes == 0) {
        const uint16_t* in = static_cast<const uint16_t*>(a.in) + static_cast<int64_t>(row) * a.in_stride;
        uint16_t* out = static_cast<uint16_t*>(a.out) + static_cast<int64_t>(place) * a.out_stride;
        for (int c = lane * 8; c < a.pad; c += 512) {
            Eight16 x;
            if (c + 8 <= a.cols) x = *reinterpret_cast<const Eight16*>(in + c);
            else
                for (int i = 0; i < 8; ++i) x.v[i] = c + i < a.cols ? in[c + i] : 0;
            u32x4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = x.v[2 * i] | static_cast<uint32_t>(x.v[2 * i + 1]) << 16;
            *reinterpret_cast<u32x4*>(out + c) = v;
        }
        return;
    }
    float peak = 0.0f, v[8];
    for (int c = lane * 8; c < a.cols; c += 512) {
        load_eight(a, row, c, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) peak = fmaxf(peak, finite_size(v[i]));
    }
    const int e = scale_exponent(wave_max(peak));
    const float scale = power_of_two(e);
    for (int c = lane * 8; c < a.pad; c += 512) {
        load_eight(a, row, c, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= scale;
        store_eight(a, place, c, v);
    }
    if (lane == 0) a.unscale[place] = power_of_two(-e);
}

// The largest size of each column, in kPeakParts parts of the rows. A wave takes 512 columns of eight rows at a time; bound by its few rounds of
// loads: 5120 x 1024 bf16 9 us. One scale per feature instead of one for all costs dW's product and its layout 8 us a pass there.
constexpr int kPeakWaves = 16;
__global__ __launch_bounds__(64 * kPeakWaves) void column_peaks_kernel(LayArgs a) {
    __shared__ float merge[kPeakWaves][512];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, first = blockIdx.y * 512, c = first + lane * 8, rows = rows_of(a);
    constexpr int kOnTheirWay = 8;
    const int apart = gridDim.x * kPeakWaves;
    float peak[8] = {};
    if (c < a.cols)
        for (int place = blockIdx.x * kPeakWaves + wave; place < rows; place += kOnTheirWay * apart) {
            float v[kOnTheirWay][8], f[kOnTheirWay];
            int row[kOnTheirWay];
#pragma unroll
            for (int u = 0; u < kOnTheirWay; ++u) row[u] = row_of(a, min(place + u * apart, rows - 1));       // past the end: the last again
#pragma unroll
            for (int u = 0; u < kOnTheirWay; ++u) {
                load_eight(a, row[u], c, v[u]);
                f[u] = row_keeps(a, row[u]);
            }
#pragma unroll
            for (int u = 0; u < kOnTheirWay; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) peak[i] = fmaxf(peak[i], f[u] == 0.0f ? 0.0f : finite_size(v[u][i] * f[u]));
        }
#pragma unroll
    for (int i = 0; i < 8; ++i) merge[wave][i * 64 + lane] = peak[i];
    __syncthreads();
    const int x = threadIdx.x, at = first + (x & 63) * 8 + (x >> 6);
    if (x >= 512 || at >= a.cols) return;
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < kPeakWaves; ++i) top = fmaxf(top, merge[i][x]);
    a.peaks[blockIdx.x * a.peak_stride + at] = top;
}

// Bound by memory: 134 MB in 22 us (6.1 TB/s).
__global__ __launch_bounds__(kLayThreads) void absmax_kernel(LayArgs a) {
    __shared__ float merge[kLayThreads / 64];
    const int lane = threadIdx.x & 63;
    float peak = 0.0f, v[8];
    const int rows = rows_of(a);
    for (int place = blockIdx.x * (kLayThreads / 64) + (threadIdx.x >> 6); place < rows; place += gridDim.x * (kLayThreads / 64)) {
        const int row = row_of(a, place);
        const float f = row_keeps(a, row);
        if (f == 0.0f) continue;
        for (int c = lane * 8; c < a.cols; c += 512) {
            load_eight(a, row, c, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) peak = fmaxf(peak, finite_size(v[i] * f));
        }
    }
    peak = wave_max(peak);
    if (lane == 0) merge[threadIdx.x >> 6] = peak;
    __syncthreads();
    if (threadIdx.x == 0) a.parts[blockIdx.x] = fmaxf(fmaxf(merge[0], merge[1]), fmaxf(merge[2], merge[3]));
}

// 64 x 64 elements through LDS: out[col][row], one scale for all of them or (peaks) one per column, which is a row of the product. Bound by memory: 16384 x 4096 bf16 to fp16 44 us (6.1 TB/s).
__global__ __launch_bounds__(kLayThreads) void lay_columns_kernel(LayArgs a) {
    __shared__ float tile[64][65], peaks[kLayThreads / 64][64];
    const int t = threadIdx.x, r0 = blockIdx.x * 64, c0 = blockIdx.y * 64, rows = rows_of(a), pad = (rows + 63) / 64 * 64;
    if (r0 >= pad && r0) return;        // the first writes the scales, whatever there is to lay out
    float v[8];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int r = x * 32 + (t >> 3), c = (t & 7) * 8;
        const int row = r0 + r < rows ? row_of(a, r0 + r) : 0;
        const float f = r0 + r < rows ? row_keeps(a, row) : 0.0f;
        if (f != 0.0f) load_eight(a, row, c0 + c, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) tile[r][c + i] = f != 0.0f ? v[i] * f : 0.0f;
    }
    float whole = 0.0f;
    if (a.peaks) {
        const int c = c0 + (t & 63);
        float peak = 0.0f;
#pragma unroll
        for (int i = 0; i < kPeakParts; i += kLayThreads / 64) peak = fmaxf(peak, c < a.cols ? a.peaks[(i + (t >> 6)) * a.peak_stride + c] : 0.0f);
        peaks[t >> 6][t & 63] = peak;
        __syncthreads();
    } else {
        whole = join_parts(a.parts);        // its barrier stands behind the writes of `tile` too
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int c = x * 32 + (t >> 3), r = (t & 7) * 8;
        if (c0 + c >= a.cols) continue;
        const int e = scale_exponent(a.peaks ? fmaxf(fmaxf(peaks[0][c], peaks[1][c]), fmaxf(peaks[2][c], peaks[3][c])) : whole);
        const float scale = power_of_two(e);
        if (r0 + r == 0 && (a.peaks || c0 + c == 0)) a.unscale[c0 + c] = power_of_two(-e);
        if (r0 + r >= pad) continue;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = tile[r + i][c] * scale;
        store_eight(a, c0 + c, r0 + r, v);
    }
}

}  // namespace

int launch_lay_rows(const LayArgs& a, hipStream_t stream) {
    if (!a.parts) return launch(lay_rows_kernel, (a.rows + 3) / 4, kLayThreads, a, stream);
    const int status = launch(absmax_kernel, kMaxParts, kLayThreads, a, stream);
    return status != JABAS_OK ? status : launch(lay_rows_kernel, (a.pad_rows + 3) / 4, kLayThreads, a, stream);
}

int launch_lay_columns(const LayArgs& a, hipStream_t stream) {
    void* params[] = {const_cast<LayArgs*>(&a)};
    const hipError_t error = a.peaks ? hipLaunchKernel(reinterpret_cast<const void*>(column_peaks_kernel), dim3(kPeakParts, (a.cols + 511) / 512), dim3(64 * kPeakWaves), params, 0, stream)
                                     : hipLaunchKernel(reinterpret_cast<const void*>(absmax_kernel), dim3(kMaxParts), dim3(kLayThreads), params, 0, stream);
    if (error != hipSuccess) return JABAS_ERR_LAUNCH;
    return hipLaunchKernel(reinterpret_cast<const void*>(lay_columns_kernel), dim3(a.pad / 64, (a.cols + 63) / 64), dim3(kLayThreads), params, 0, stream) == hipSuccess
               ? JABAS_OK : JABAS_ERR_LAUNCH;
}

}  // namespace loss
}  // namespace jabas
