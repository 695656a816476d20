// What a workgroup of the orthogonalised update works on.
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

}  // namespace muon
}  // namespace jabas
