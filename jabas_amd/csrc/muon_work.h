// What a workgroup of the orthogonalised update works on, and what it makes of a gradient.
#pragma once

#include "muon_internal.h"

namespace jabas {
namespace muon {

struct Place {
    Matrix x;
    uint32_t tile;
};

// Workgroups go round the eight dies (XCDs), each with an L2 of its own. A list's slots are laid out for that by the host; of a batch
// each die takes a run of consecutive tiles.
__device__ inline bool place_of(const Work& w, Place& at) {
    const uint32_t block = blockIdx.x;
    if (block >= w.total) return false;
    if (w.table) {
        const Slot s = w.slots[block];
        at.x = w.table[__builtin_amdgcn_readfirstlane(s.matrix)];
        at.tile = __builtin_amdgcn_readfirstlane(s.tile);
        return true;
    }
    const uint32_t die = block & 7, each = w.total >> 3, left = w.total & 7;
    const uint32_t slot = die * each + min(die, left) + (block >> 3), i = slot / w.per;
    at.tile = slot - i * w.per;
    at.x = w.one;
    at.x.src = static_cast<const char*>(w.one.src) + i * w.src_step;
    at.x.out = static_cast<char*>(w.one.out) + i * w.out_step;
    at.x.x_at += i * w.x_step;
    at.x.a_at += i * w.a_step;
    at.x.part_at += i * w.part_step;
    return true;
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
