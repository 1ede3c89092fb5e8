// Row groups as the grouped products see them: ranges from device offsets, and the table that maps a tile
// number to its group.
#pragma once

#include "rows.cuh"

namespace spmm_b200 {

// Rows [begin, end) of group g, kept inside [0, rows] whatever the offsets hold; a bad pair is recorded.
struct GroupRange {
    int begin, end;
};
__device__ __forceinline__ GroupRange group_range(const int* __restrict__ offsets, int g, int rows, DeviceErrorRecord* err) {
    if (!offsets) return {g, g + 1};  // every row a group of its own
    const int b = __ldg(offsets + g), e = __ldg(offsets + g + 1);
    if (b < 0 || e < b || e > rows) record_device_error(err, SPMM_ERR_BAD_INDEX, g);
    const int begin = max(0, min(b, rows));
    return {begin, max(begin, min(e, rows))};
}

// start[g] = number of row tiles (tile rows each) of the groups before g, start[groups] = all of them. Called by every
// thread of the block; ends with a barrier.
__device__ __forceinline__ void build_tile_table(int* start, const int* __restrict__ offsets, int groups, int rows, int tile,
                                                 DeviceErrorRecord* err) {
    for (int g = threadIdx.x; g < groups; g += blockDim.x) {
        const GroupRange r = group_range(offsets, g, rows, err);
        start[g + 1] = (r.end - r.begin + tile - 1) / tile;
    }
    if (threadIdx.x == 0) start[0] = 0;
    __syncthreads();
    if (threadIdx.x < 32) {
        int run = 0;
        for (int base = 0; base < groups; base += 32) {
            const int g = base + threadIdx.x;
            int v = g < groups ? start[g + 1] : 0;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const int u = __shfl_up_sync(0xffffffffu, v, d);
                if (static_cast<int>(threadIdx.x) >= d) v += u;
            }
            if (g < groups) start[g + 1] = run + v;
            run += __shfl_sync(0xffffffffu, v, 31);
        }
    }
    __syncthreads();
}

// The group of row tile m < start[groups].
__device__ __forceinline__ int tile_group(const int* start, int groups, int m) {
    int lo = 0, hi = groups;  // start[lo] <= m < start[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (start[mid] <= m) lo = mid;
        else hi = mid;
    }
    return lo;
}

}  // namespace spmm_b200
