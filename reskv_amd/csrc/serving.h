// Shared by the serving kernels: which packed sequence an item of work belongs to.
#pragma once

#include "common.h"

namespace reskv {

struct Item {
    int seq;    // -1: behind the last sequence's items
    int index;  // item within the sequence
};

// Item t of the items that sequences 0, 1, .. bring one after the other, count(s) each.
// Called by whole waves; 64 sequences per turn, one per lane.
template <class Count>
__device__ __forceinline__ Item find_item(int t, int sequences, Count count) {
    const int lane = lane_id();
    int base = 0;
    for (int s0 = 0; s0 < sequences; s0 += kWave) {
        const int mine = s0 + lane < sequences ? count(s0 + lane) : 0;
        int sum = mine;  // inclusive
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) {
            const int below = __shfl_up(sum, d);
            if (lane >= d) sum += below;
        }
        const uint64_t past = ballot(sum > t - base);
        if (past != 0) {
            const int who = __builtin_ctzll(past);
            return {__builtin_amdgcn_readfirstlane(s0 + who),
                    __builtin_amdgcn_readfirstlane(t - base - (__shfl(sum, who) - __shfl(mine, who)))};
        }
        base += __builtin_amdgcn_readlane(sum, kWave - 1);
    }
    return {-1, __builtin_amdgcn_readfirstlane(t - base)};
}

// The rows of sequence s, clamped into [0, rows) whatever the offsets hold.
struct Rows {
    int first, count;
};
__device__ __forceinline__ Rows sequence_rows(const int32_t* offsets, int s, int rows) {
    const int a = min(max(offsets[s], 0), rows), b = min(max(offsets[s + 1], a), rows);
    return {a, b - a};
}

}  // namespace reskv
