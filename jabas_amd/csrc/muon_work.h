// What a workgroup of the orthogonalised update works on, and what it makes of a gradient.
#pragma once

#include "muon_internal.h"

namespace jabas {
namespace muon {

// A list's tables are not written while a launch reads them: through the constant address space they are uniform loads.
template <class T>
using Fixed = const __attribute__((address_space(4))) T;

// What a product needs of a matrix.
struct Sides {
    uint32_t matrix, tile;
    int32_t m, n, pad_m, pad_n;
    int64_t x_at, a_at, x_plane, a_plane;
    uint32_t unit;
    int32_t splits;
    __device__ void pad() {
        pad_m = (m + kPad - 1) / kPad * kPad;
        pad_n = (n + kPad - 1) / kPad * kPad;
        x_plane = static_cast<int64_t>(pad_m) * pad_n;
        a_plane = static_cast<int64_t>(pad_m) * pad_m;
    }
};

// Workgroups go round the eight dies (XCDs), each with an L2 of its own. A list's slots are laid out for that by the host; of a batch
// each die takes a run of consecutive tiles.
__device__ inline bool sides_of(const Work& w, Sides& at) {
    const uint32_t block = blockIdx.x;
    if (block >= w.total) return false;
    if (w.table) {
        Fixed<Slot>& s = *(Fixed<Slot>*)(w.slots + block);
        at.matrix = s.matrix;
        at.tile = s.tile;
        at.m = s.m;
        at.n = s.n;
        at.x_at = s.x_at;
        at.a_at = s.a_at;
        at.unit = s.unit;
        at.splits = s.splits;
    } else {
        const uint32_t die = block & 7, each = w.total >> 3, left = w.total & 7;
        const uint32_t slot = die * each + min(die, left) + (block >> 3);
        at.matrix = slot / w.per;
        at.tile = slot - at.matrix * w.per;
        at.m = w.one.m;
        at.n = w.one.n;
        at.x_at = w.one.x_at + at.matrix * w.x_step;
        at.a_at = w.one.a_at + at.matrix * w.a_step;
        at.unit = at.matrix * w.per;
        at.splits = w.splits;
    }
    at.pad();
    return true;
}

// Everything about matrix `i`.
__device__ inline Matrix matrix_of(const Work& w, uint32_t i) {
    if (!w.table) {
        Matrix x = w.one;
        x.src = static_cast<const char*>(w.one.src) + i * w.src_step;
        x.out = static_cast<char*>(w.one.out) + i * w.out_step;
        x.x_at += i * w.x_step;
        x.a_at += i * w.a_step;
        x.part_at += i * w.part_step;
        return x;
    }
    Fixed<Matrix>& t = *(Fixed<Matrix>*)(w.table + i);
    Matrix x;
    x.src = t.src;
    x.momentum = t.momentum;
    x.out = t.out;
    x.src_stride = t.src_stride;
    x.x_at = t.x_at;
    x.a_at = t.a_at;
    x.part_at = t.part_at;
    x.x_plane = t.x_plane;
    x.a_plane = t.a_plane;
    x.rows = t.rows;
    x.cols = t.cols;
    x.m = t.m;
    x.n = t.n;
    x.pad_m = t.pad_m;
    x.pad_n = t.pad_n;
    x.tall = t.tall;
    x.src_quads = t.src_quads;
    x.out_quads = t.out_quads;
    x.parts = t.parts;
    x.chunk = t.chunk;
    x.group = t.group;
    x.lr_factor = t.lr_factor;
    x.n_fanout = t.n_fanout;
    x.fanout_at = t.fanout_at;
    return x;
}

template <class T>
__device__ inline float element(const T* p, int64_t i) {
    if constexpr (sizeof(T) == 4) return p[i];
    else return __uint_as_float(static_cast<uint32_t>(p[i]) << 16);
}
// Momentum and update of an element.
struct Mix {
    float momentum, fresh, scale;
    int nesterov;
    __device__ explicit Mix(const PassArgs& a) : momentum(a.momentum), fresh(a.fresh), scale(1.0f), nesterov(a.nesterov) {
        if (a.grad_scale) {
            const float c = *a.grad_scale;
            if (c < 1.0f) scale = c;        // a NaN is no bound
        }
    }
    __device__ float buffer(float g, float buf) const { return fmaf(fresh, g - buf, buf); }
    __device__ float update(float g, float buf) const { return nesterov ? fmaf(momentum, buf - g, g) : buf; }
};

__device__ inline double sum_of_wave(double x) {
#pragma unroll
    for (int i = 32; i; i >>= 1) x += __shfl_xor(x, i);
    return x;
}

}  // namespace muon
}  // namespace jabas
