// Where the results of the orthogonalised update go.
#pragma once

#include "muon_internal.h"

namespace jabas {
namespace muon {

typedef float quad_t __attribute__((ext_vector_type(4)));

__device__ inline uint16_t to_bf16(float x) {
    const uint32_t u = __float_as_uint(x);
    if ((u & 0x7fffffffu) > 0x7f800000u) return static_cast<uint16_t>((u >> 16) | 0x40);
    return static_cast<uint16_t>((u + 0x7fffu + ((u >> 16) & 1)) >> 16);
}

// Where a step's last product goes: `count` (up to V) results of consecutive columns of a row of the matrix as the caller has it.
template <int V>
__device__ inline void put_out(const Out& a, const uint64_t* fanout, const Matrix& x, int row, int col, const float* v) {
    const int64_t place = static_cast<int64_t>(row) * x.cols + col;
    const int count = min(V, x.cols - col);
    if (!x.momentum) {
        if (a.dtype == JABAS_F32) {
            float* out = static_cast<float*>(x.out) + place;
            if (V >= 4 && x.out_quads)
#pragma unroll
                for (int e = 0; e < V; e += 4) { if (e < count) *reinterpret_cast<quad_t*>(out + e) = quad_t{v[e], v[e + 1], v[e + 2], v[e + 3]}; }
            else
#pragma unroll
                for (int e = 0; e < V; ++e) { if (e < count) out[e] = v[e]; }
        } else {
            uint16_t* out = static_cast<uint16_t*>(x.out) + place;
            if (V >= 4 && x.out_quads)
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
    if (V >= 4 && x.out_quads) {
#pragma unroll
        for (int e = 0; e < V; e += 4) {
            if (e >= count) continue;
            quad_t now = *reinterpret_cast<const quad_t*>(w + e);
#pragma unroll
            for (int i = 0; i < 4; ++i) now[i] = fmaf(-lr, v[e + i], now[i] * keep);
            *reinterpret_cast<quad_t*>(w + e) = now;
            for (uint32_t f = 0; f < x.n_fanout; ++f) *reinterpret_cast<quad_t*>(reinterpret_cast<float*>(fanout[x.fanout_at + f]) + place + e) = now;
        }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (e >= count) continue;
            const float now = fmaf(-lr, v[e], w[e] * keep);
            w[e] = now;
            for (uint32_t f = 0; f < x.n_fanout; ++f) reinterpret_cast<float*>(fanout[x.fanout_at + f])[place + e] = now;
        }
    }
}

}  // namespace muon
}  // namespace jabas
