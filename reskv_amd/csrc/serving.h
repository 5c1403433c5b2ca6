// Shared by the serving kernels: which packed sequence an item of work belongs to.
#pragma once

#include "common.h"

namespace reskv {

// Sum and maximum over the wave, and inclusive sums in lane order, on DPP row operations: a few
// cycles each, where a shuffle through the LDS takes a hundred and a kernel's start waits for a dozen.
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ int dpp_int(int v) {  // lanes without a source get 0
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_sum_int(int v) {
    v += dpp_int<0xB1>(v);
    v += dpp_int<0x4E>(v);
    v += dpp_int<0x141>(v);
    v += dpp_int<0x140>(v);
    return (__builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16)) +
           (__builtin_amdgcn_readlane(v, 32) + __builtin_amdgcn_readlane(v, 48));
}
__device__ __forceinline__ int wave_max_int(int v) {
    v = max(v, dpp_int<0xB1>(v));
    v = max(v, dpp_int<0x4E>(v));
    v = max(v, dpp_int<0x141>(v));
    v = max(v, dpp_int<0x140>(v));
    return max(max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
               max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}
__device__ __forceinline__ int wave_scan_int(int v) {
    v += dpp_int<0x111>(v);       // row_shr 1, 2, 4, 8
    v += dpp_int<0x112>(v);
    v += dpp_int<0x114>(v);
    v += dpp_int<0x118>(v);
    v += dpp_int<0x142, 0xA>(v);  // a row's last lane to the next row
    v += dpp_int<0x143, 0xC>(v);  // lane 31 to the upper half
    return v;
}

constexpr long kLaunchThreads = 1L << 32;  // a launch has fewer: the grid is counted in threads, in 32 bits

struct Item {
    int seq;    // -1: behind the last sequence's items
    int index;  // item within the sequence
};

// Item t of the items that sequences 0, 1, .. bring one after the other, count(s) each.
// Called by whole waves with one t; 64 sequences per turn, one per lane.
template <class Count>
__device__ __forceinline__ Item find_item(int t, int sequences, Count count) {
    const int lane = lane_id();
    int base = 0;
    for (int s0 = 0; s0 < sequences; s0 += kWave) {
        const int mine = s0 + lane < sequences ? count(s0 + lane) : 0;
        const int sum = wave_scan_int(mine);
        const uint64_t past = ballot(sum > t - base);
        if (past != 0) {
            const int who = __builtin_ctzll(past);
            return {s0 + who, t - base - (__builtin_amdgcn_readlane(sum, who) - __builtin_amdgcn_readlane(mine, who))};
        }
        base += __builtin_amdgcn_readlane(sum, kWave - 1);
    }
    return {-1, t - base};
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
