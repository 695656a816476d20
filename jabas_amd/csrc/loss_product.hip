// Matrix products of the losses: logits of a tile of tokens and rows that never leave the registers (forward: their
// maxima and sums; backward: the row gradients dz), and the products of dz with the weight and the hidden states.
#include "loss_internal.h"

namespace jabas {
namespace loss {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct F16 {
    using vec = f16x8;
    static __device__ f32x16 mfma(vec a, vec b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
struct BF16 {
    using vec = bf16x8;
    static __device__ f32x16 mfma(vec a, vec b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};

__device__ inline f16x8 lowered(f16x8 v) { return v * static_cast<_Float16>(1.0f / kLowScale); }
__device__ inline bf16x8 lowered(bf16x8 v) { return v; }     // one plane only

constexpr int kThreads = 256;               // four waves, each a quarter (64 x 64) of the tile
constexpr int kChunks = kTile * 8 / kThreads;   // 16-byte chunks of one operand's tile per thread

__device__ inline float load_as_float(const void* p, int64_t i, int dtype) {
    if (dtype == JABAS_F32) return static_cast<const float*>(p)[i];
    return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(p)[i]) << 16);
}

__device__ inline uint16_t to_bf16(float x) {
    const uint32_t u = __float_as_uint(x);
    if ((u & 0x7fffffffu) > 0x7f800000u) return static_cast<uint16_t>((u >> 16) | 0x40);
    return static_cast<uint16_t>((u + 0x7fffu + ((u >> 16) & 1)) >> 16);
}

__device__ inline void store_as(void* p, int64_t i, int dtype, float v) {
    if (dtype == JABAS_F32) static_cast<float*>(p)[i] = v;
    else static_cast<uint16_t*>(p)[i] = to_bf16(v);
}

// A row of a staged tile is 128 bytes, eight chunks of 16: one plane of 64 elements, or two planes of 32. Chunk c of row r
// lies at chunk c ^ (r & 7): lanes that read the same chunk of eight rows then touch all banks once.
template <int P>
__device__ inline const u32x4* chunk_address(const Operand& o, int row, int chunk, int step) {
    row = row < o.rows ? row : o.rows - 1;          // rows past the end are read again, never written
    const uint16_t* p = static_cast<const uint16_t*>(o.p) + static_cast<int64_t>(row) * o.stride;
    if (P == 2) p += (chunk >> 2) * o.plane + step * 32 + (chunk & 3) * 8;
    else p += step * 64 + chunk * 8;
    return reinterpret_cast<const u32x4*>(p);
}

// acc[i][j]: 32 x 32 blocks of out[m][n] = sum_k a[m][k] b[n][k] over this wave's 64 x 64. Element e of a block is
// m = 8 (e / 4) + 4 (lane / 32) + e % 4, n = lane % 32.
// Two planes: (a0 + a1)(b0 + b1) without a1 b1, which is under 2^-22 of the whole. kRaised: a's second plane is kept
// larger by kLowScale, so b0 is made as much smaller for it.
template <class E, int P, bool kRaised>
__device__ inline void product(const Operand& a, const Operand& b, int m0, int n0, int depth, char* smem, f32x16 (&acc)[2][2]) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
    constexpr int kBytes = kTile * 128;
    u32x4 ra[kChunks], rb[kChunks];
    const int steps = depth / (P == 2 ? 32 : 64);
    auto fetch = [&](int s) {
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const int at = i * kThreads + t;
            ra[i] = *chunk_address<P>(a, m0 + (at >> 3), at & 7, s);
            rb[i] = *chunk_address<P>(b, n0 + (at >> 3), at & 7, s);
        }
    };
    auto stage = [&](int buf) {
        char* base = smem + buf * 2 * kBytes;
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const int at = i * kThreads + t, row = at >> 3, c = (at & 7) ^ (row & 7);
            *reinterpret_cast<u32x4*>(base + row * 128 + c * 16) = ra[i];
            *reinterpret_cast<u32x4*>(base + kBytes + row * 128 + c * 16) = rb[i];
        }
    };
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    fetch(0);
    stage(0);
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
        if (s + 1 < steps) fetch(s + 1);
        const char* base = smem + (s & 1) * 2 * kBytes;
        auto read = [&](int row, int chunk) {
            return *reinterpret_cast<const typename E::vec*>(base + row * 128 + ((chunk ^ (row & 7)) * 16));
        };
        const int r = lane & 31, h = lane >> 5;
        if (P == 1) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                typename E::vec fa[2], fb[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    fa[i] = read(wm + i * 32 + r, kk * 2 + h);
                    fb[i] = read(kTile + wn + i * 32 + r, kk * 2 + h);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[i][j] = E::mfma(fa[i], fb[j], acc[i][j]);
            }
        } else {
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                typename E::vec fa[2][2], fb[2][2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        fa[i][q] = read(wm + i * 32 + r, q * 4 + kk * 2 + h);
                        fb[i][q] = read(kTile + wn + i * 32 + r, q * 4 + kk * 2 + h);
                    }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        acc[i][j] = E::mfma(fa[i][1], kRaised ? lowered(fb[j][0]) : fb[j][0], acc[i][j]);
                        acc[i][j] = E::mfma(fa[i][0], fb[j][1], acc[i][j]);
                        acc[i][j] = E::mfma(fa[i][0], fb[j][0], acc[i][j]);
                    }
            }
        }
        if (s + 1 < steps) stage((s + 1) & 1);
        __syncthreads();
    }
}

__device__ inline int block_m(int i, int e, int lane) { return i * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3); }

constexpr int kMapStride = kTile + 4;       // bytes of a row of the entry map: lanes of 32 rows read 32 banks

// Which tokens of the tile are entries of which row: byte [row][token] is 1 + the entry's number. Built over the
// operands' buffers, which nobody reads any more.
__device__ inline void build_map(const Entries& en, char* map, int first, int n0, int rows) {
    const int t = threadIdx.x;
    for (int i = t; i < kTile * kMapStride / 4; i += kThreads) reinterpret_cast<uint32_t*>(map)[i] = 0;
    __syncthreads();
    const int here = min(kTile, rows - n0) * en.k;
    for (int i = t; i < here; i += kThreads) {
        const int n = i / en.k, j = i - n * en.k;
        const int v = en.index[static_cast<int64_t>(n0) * en.k + i] - first;
        if (v >= 0 && v < kTile) map[n * kMapStride + v] = static_cast<char>(1 + j);
    }
    __syncthreads();
}

__device__ inline void wave_range(int& wm, int& wn) {
    const int wave = threadIdx.x >> 6;
    wm = (wave >> 1) * 64;
    wn = (wave & 1) * 64;
}

// The tile's logits out of the accumulators: scaling undone, bias added.
template <int P>
__device__ inline void logits_of(const LogitsArgs& a, int m0, int n0, f32x16 (&acc)[2][2]) {
    const int lane = threadIdx.x & 63;
    int wm, wn;
    wave_range(wm, wn);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int m = min(m0 + wm + block_m(i, e, lane), a.w.rows - 1);
            const float b = a.bias ? load_as_float(a.bias, static_cast<int64_t>(a.first) + m, a.bias_dtype) : 0.0f;
            const float uw = P == 2 ? a.unscale_w[m] : 1.0f;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float z = acc[i][j][e];
                if (P == 2) z = z * a.unscale_x[min(n0 + wn + j * 32 + (lane & 31), a.x.rows - 1)] * uw;
                acc[i][j][e] = z + b;
            }
        }
}

template <class E, int P>
__global__ __launch_bounds__(kThreads) void logits_forward_kernel(LogitsArgs a) {
    __shared__ __align__(16) char smem[4 * kTile * 128];
    const int tiles_m = (a.w.rows + kTile - 1) / kTile;
    const int tm = blockIdx.x % tiles_m, tn = blockIdx.x / tiles_m;
    const int m0 = tm * kTile, n0 = tn * kTile, lane = threadIdx.x & 63;
    f32x16 acc[2][2];
    product<E, P, false>(a.w, a.x, m0, n0, a.depth, smem, acc);
    logits_of<P>(a, m0, n0, acc);
    int wm, wn;
    wave_range(wm, wn);
    const bool teacher = a.entries.index != nullptr;
    if (teacher) build_map(a.entries, smem, a.first + m0, n0, a.x.rows);
    float peak[2], sum[2], total[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int nl = wn + j * 32 + (lane & 31), n = n0 + nl;
        const bool row = n < a.x.rows;
        const int64_t label = !teacher && row ? a.entries.target[n] - a.first - m0 : -1;
        peak[j] = -INFINITY;
        total[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int ml = wm + block_m(i, q * 4, lane);
                const uint32_t hits = teacher ? *reinterpret_cast<const uint32_t*>(smem + nl * kMapStride + ml) : 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float z = acc[i][j][q * 4 + e];
                    const bool in = m0 + ml + e < a.w.rows;
                    if (in) total[j] += z;
                    const uint32_t hit = (hits >> (8 * e)) & 0xff;
                    if (hit) a.entry_logit[static_cast<int64_t>(n) * a.entries.k + hit - 1] = z;
                    if (in && label == ml + e) a.entry_logit[n] = z;
                    acc[i][j][q * 4 + e] = in && !hit ? z : -INFINITY;     // entries join their row later, each by itself
                    peak[j] = fmaxf(peak[j], acc[i][j][q * 4 + e]);
                }
            }
        peak[j] = fmaxf(peak[j], __shfl_xor(peak[j], 32));
        const float base = peak[j] == -INFINITY ? 0.0f : peak[j];
        sum[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) sum[j] += __builtin_amdgcn_exp2f((acc[i][j][e] - base) * a.c);
        sum[j] += __shfl_xor(sum[j], 32);
        total[j] += __shfl_xor(total[j], 32);
    }
    __syncthreads();
    float* merge = reinterpret_cast<float*>(smem);       // [3][128] of the waves that hold the upper half of the tile's tokens
    if (wm != 0 && lane < 32) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int nl = wn + j * 32 + lane;
            merge[nl] = peak[j];
            merge[kTile + nl] = sum[j];
            merge[2 * kTile + nl] = total[j];
        }
    }
    __syncthreads();
    if (wm == 0 && lane < 32) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int nl = wn + j * 32 + lane, n = n0 + nl;
            const float p2 = merge[nl], s2 = merge[kTile + nl];
            const float p = fmaxf(peak[j], p2);
            float s = 0.0f;
            if (sum[j] != 0.0f) s += sum[j] * __builtin_amdgcn_exp2f((peak[j] - p) * a.c);
            if (s2 != 0.0f) s += s2 * __builtin_amdgcn_exp2f((p2 - p) * a.c);
            if (n < a.x.rows) {
                const int64_t at = static_cast<int64_t>(a.first_tile + tm) * a.x.rows + n;
                a.partial[at] = make_float2(p, s);
                if (a.total) a.total[at] = total[j] + merge[2 * kTile + nl];
            }
        }
    }
}

template <class E, int P>
__global__ __launch_bounds__(kThreads) void logits_backward_kernel(LogitsArgs a) {
    __shared__ __align__(16) char smem[4 * kTile * 128];
    const int tiles_m = (a.pad_tokens + kTile - 1) / kTile;
    const int tm = blockIdx.x % tiles_m, tn = blockIdx.x / tiles_m;
    const int m0 = tm * kTile, n0 = tn * kTile, lane = threadIdx.x & 63;
    f32x16 acc[2][2];
    product<E, P, false>(a.w, a.x, m0, n0, a.depth, smem, acc);
    logits_of<P>(a, m0, n0, acc);
    int wm, wn;
    wave_range(wm, wn);
    const bool teacher = a.entries.index != nullptr;
    if (teacher) build_map(a.entries, smem, a.first + m0, n0, a.x.rows);
    float grad[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int nl = wn + j * 32 + (lane & 31), n = n0 + nl;
        const bool row = n < a.x.rows;
        const RowState st = row ? a.state[n] : RowState{0.0f, 0.0f, 0.0f, 0.0f};
        const bool counts = !(st.slope == 0.0f && st.mass == 0.0f);
        const int64_t label = !teacher && row ? a.entries.target[n] - a.first - m0 : -1;
        grad[j] = row ? a.row_grad[n] : 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int ml = wm + block_m(i, q * 4, lane);
                const uint32_t hits = teacher ? *reinterpret_cast<const uint32_t*>(smem + nl * kMapStride + ml) : 0;
                float d[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float z = acc[i][j][q * 4 + e];
                    const uint32_t hit = (hits >> (8 * e)) & 0xff;
                    if (hit) d[e] = st.mass * __builtin_amdgcn_exp2f((z - st.peak) * a.c) - a.entries.p[static_cast<int64_t>(n) * a.entries.k + hit - 1];
                    else d[e] = st.slope * __builtin_amdgcn_exp2f((z - st.peak_rest) * a.c) - a.uniform;
                    if (label == ml + e) d[e] -= a.hit;
                    if (!counts || m0 + ml + e >= a.w.rows) d[e] = 0.0f;
                    acc[i][j][q * 4 + e] = d[e];
                }
                f16x4 hi, lo;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float v = d[e] * kDzScale;
                    hi[e] = static_cast<_Float16>(v);
                    if (P == 2) lo[e] = static_cast<_Float16>((v - static_cast<float>(hi[e])) * kLowScale);
                }
                _Float16* dz = static_cast<_Float16*>(a.dz) + static_cast<int64_t>(n) * a.dz_stride + m0 + ml;
                _Float16* dzt = static_cast<_Float16*>(a.dzt) + static_cast<int64_t>(m0 + ml) * a.dzt_stride + n;
                if (a.dz && row && m0 + ml < a.pad_tokens) {
                    *reinterpret_cast<f16x4*>(dz) = hi;
                    if (P == 2) *reinterpret_cast<f16x4*>(dz + a.dz_plane) = lo;
                }
                if (a.dzt && n < a.pad_rows) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (m0 + ml + e < a.w.rows) {
                            dzt[e * a.dzt_stride] = hi[e];
                            if (P == 2) dzt[e * a.dzt_stride + a.dzt_plane] = lo[e];
                        }
                }
            }
    }
    if (a.db) {      // sums over this tile's rows: within the wave, then over the two waves that share tokens
        __syncthreads();
        float* merge = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float s = acc[i][0][e] * grad[0] + acc[i][1][e] * grad[1];
#pragma unroll
                for (int x = 1; x < 32; x <<= 1) s += __shfl_xor(s, x);
                if ((lane & 31) == 0) merge[(wn ? kTile : 0) + wm + block_m(i, e, lane)] = s;
            }
        __syncthreads();
        const int m = threadIdx.x;
        if (m < kTile && m0 + m < a.w.rows) a.db[static_cast<int64_t>(tn) * a.w.rows + m0 + m] = merge[m] + merge[kTile + m];
    }
}

template <int P>
__global__ __launch_bounds__(kThreads) void out_kernel(OutArgs a) {
    __shared__ __align__(16) char smem[4 * kTile * 128];
    const int tiles_m = (a.a.rows + kTile - 1) / kTile;
    const int tm = blockIdx.x % tiles_m, tn = blockIdx.x / tiles_m;
    const int m0 = tm * kTile, n0 = tn * kTile, lane = threadIdx.x & 63;
    f32x16 acc[2][2];
    product<F16, P, P == 2>(a.a, a.b, m0, n0, a.depth, smem, acc);
    int wm, wn;
    wave_range(wm, wn);
    float scale = a.scale;
    if (a.unscale0) scale *= *a.unscale0;
    const float second = a.unscale1 ? *a.unscale1 : 1.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int m = m0 + wm + block_m(i, e, lane);
            if (m >= a.a.rows) continue;
            const float rs = a.row_scale ? a.row_scale[m] : 1.0f;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int n = n0 + wn + j * 32 + (lane & 31);
                if (n >= a.b.rows) continue;
                float v = acc[i][j][e] * scale * second;        // the pieces of a sum have scales of their own
                if (a.acc) {
                    float* sum = a.acc + static_cast<int64_t>(m) * a.b.rows + n;
                    if (!a.first) v += *sum;
                    if (!a.last) {
                        *sum = v;
                        continue;
                    }
                }
                // a row that does not count is zero even where its neighbours' scale is not finite
                v = rs == 0.0f ? 0.0f : v * rs;
                store_as(a.out, static_cast<int64_t>(m) * a.out_stride + n, a.out_dtype, v);
            }
        }
}

inline int tiles(int64_t n) { return static_cast<int>((n + kTile - 1) / kTile); }

inline int launched() { return hipGetLastError() == hipSuccess ? JABAS_OK : JABAS_ERR_LAUNCH; }

template <class K, class A>
int launch(K kernel, unsigned grid, const A& args, hipStream_t stream) {
    void* params[] = {const_cast<A*>(&args)};
    return hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3(grid), dim3(kThreads), params, 0, stream) == hipSuccess ? JABAS_OK : JABAS_ERR_LAUNCH;
}

}  // namespace

int launch_logits_forward(const LogitsArgs& a, int planes, hipStream_t stream) {
    const unsigned grid = static_cast<unsigned>(tiles(a.w.rows)) * tiles(a.x.rows);
    return planes == 2 ? launch(logits_forward_kernel<F16, 2>, grid, a, stream) : launch(logits_forward_kernel<BF16, 1>, grid, a, stream);
}

int launch_logits_backward(const LogitsArgs& a, int planes, hipStream_t stream) {
    const unsigned grid = static_cast<unsigned>(tiles(a.pad_tokens)) * tiles(a.pad_rows);
    return planes == 2 ? launch(logits_backward_kernel<F16, 2>, grid, a, stream) : launch(logits_backward_kernel<BF16, 1>, grid, a, stream);
}

int launch_out(const OutArgs& a, int planes, hipStream_t stream) {
    const unsigned grid = static_cast<unsigned>(tiles(a.a.rows)) * tiles(a.b.rows);
    return planes == 2 ? launch(out_kernel<2>, grid, a, stream) : launch(out_kernel<1>, grid, a, stream);
}

// ------------------------------------------------------------------ layout of operands
namespace {

constexpr int kLayThreads = 256;

// The power of two that takes `peak` to [2^14, 2^15): both planes of an element then fit fp16, and elements down to
// 2^-24 of the largest keep 22 bits.
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

__device__ inline void put_planes(_Float16* p, int64_t plane, int planes, float v) {
    const _Float16 hi = static_cast<_Float16>(v);
    p[0] = hi;
    if (planes == 2) {
        const float f = static_cast<float>(hi);
        p[plane] = static_cast<_Float16>(fabsf(f) < INFINITY ? v - f : 0.0f);
    }
}

__device__ inline float row_keeps(const LayArgs& a, int row) {
    if (a.row_mask && load_as_float(a.row_mask, row, a.in_dtype) == -INFINITY) return 0.0f;
    return a.row_factor ? a.row_factor[row] : 1.0f;
}

// One wave per row: padded, and scaled by the row's own power of two.
__global__ __launch_bounds__(kLayThreads) void lay_rows_kernel(LayArgs a) {
    const int row = blockIdx.x * (kLayThreads / 64) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= a.rows) return;
    const int64_t at = static_cast<int64_t>(row) * a.in_stride;
    if (a.planes == 0) {
        uint16_t* out = static_cast<uint16_t*>(a.out) + static_cast<int64_t>(row) * a.out_stride;
        for (int c = lane; c < a.pad; c += 64) out[c] = c < a.cols ? static_cast<const uint16_t*>(a.in)[at + c] : 0;
        return;
    }
    float peak = 0.0f;
    for (int c = lane; c < a.cols; c += 64) peak = fmaxf(peak, finite_size(load_as_float(a.in, at + c, a.in_dtype)));
    const int e = scale_exponent(wave_max(peak));
    const float scale = power_of_two(e);
    _Float16* out = static_cast<_Float16*>(a.out) + static_cast<int64_t>(row) * a.out_stride;
    for (int c = lane; c < a.pad; c += 64)
        put_planes(out + c, a.out_plane, a.planes, c < a.cols ? load_as_float(a.in, at + c, a.in_dtype) * scale : 0.0f);
    if (lane == 0) a.unscale[row] = power_of_two(-e);
}

__global__ __launch_bounds__(kLayThreads) void absmax_kernel(LayArgs a) {
    __shared__ float merge[kLayThreads / 64];
    float peak = 0.0f;
    for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float f = row_keeps(a, row);
        if (f == 0.0f) continue;
        float here = 0.0f;
        for (int c = threadIdx.x; c < a.cols; c += kLayThreads)
            here = fmaxf(here, finite_size(load_as_float(a.in, static_cast<int64_t>(row) * a.in_stride + c, a.in_dtype) * f));
        peak = fmaxf(peak, here);
    }
    peak = wave_max(peak);
    if ((threadIdx.x & 63) == 0) merge[threadIdx.x >> 6] = peak;
    __syncthreads();
    if (threadIdx.x == 0) a.parts[blockIdx.x] = fmaxf(fmaxf(merge[0], merge[1]), fmaxf(merge[2], merge[3]));
}

// 64 x 64 elements through LDS: out[col][row].
__global__ __launch_bounds__(kLayThreads) void lay_columns_kernel(LayArgs a) {
    __shared__ float tile[64][65];
    __shared__ float merge[kLayThreads / 64];
    const int t = threadIdx.x, r0 = blockIdx.x * 64, c0 = blockIdx.y * 64;
    float peak = wave_max(a.parts[t]);
    static_assert(kMaxParts == kLayThreads, "a partial maximum per thread");
    if ((t & 63) == 0) merge[t >> 6] = peak;
    for (int i = t; i < 64 * 64; i += kLayThreads) {
        const int r = i >> 6, c = i & 63;
        float v = 0.0f;
        if (r0 + r < a.rows && c0 + c < a.cols) {
            const float f = row_keeps(a, r0 + r);
            if (f != 0.0f) v = load_as_float(a.in, static_cast<int64_t>(r0 + r) * a.in_stride + c0 + c, a.in_dtype) * f;
        }
        tile[r][c] = v;
    }
    __syncthreads();
    peak = fmaxf(fmaxf(merge[0], merge[1]), fmaxf(merge[2], merge[3]));
    const int e = scale_exponent(peak);
    const float scale = power_of_two(e);
    if (t == 0 && blockIdx.x == 0 && blockIdx.y == 0) *a.unscale = power_of_two(-e);
    for (int i = t; i < 64 * 64; i += kLayThreads) {
        const int c = i >> 6, r = i & 63;
        if (c0 + c < a.cols && r0 + r < a.pad)
            put_planes(static_cast<_Float16*>(a.out) + static_cast<int64_t>(c0 + c) * a.out_stride + r0 + r, a.out_plane, a.planes, tile[r][c] * scale);
    }
}

}  // namespace

int launch_lay_rows(const LayArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL(lay_rows_kernel, dim3((a.rows + 3) / 4), dim3(kLayThreads), 0, stream, a);
    return launched();
}

int launch_lay_columns(const LayArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL(absmax_kernel, dim3(kMaxParts), dim3(kLayThreads), 0, stream, a);
    hipLaunchKernelGGL(lay_columns_kernel, dim3((a.pad + 63) / 64, (a.cols + 63) / 64), dim3(kLayThreads), 0, stream, a);
    return launched();
}

}  // namespace loss
}  // namespace jabas
