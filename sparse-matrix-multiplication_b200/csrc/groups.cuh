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

// The matrix of group g: g itself, or which[g], -1 for none (negative or, recorded, past `matrices`).
__device__ __forceinline__ int group_matrix(const int* __restrict__ which, int g, int matrices, DeviceErrorRecord* err) {
    if (!which) return g;
    const int i = __ldg(which + g);
    if (i >= matrices) record_device_error(err, SPMM_ERR_BAD_INDEX, g);
    return i < 0 || i >= matrices ? -1 : i;
}

// start[g] = sum of count(0) .. count(g - 1), start[groups] = all of them; counts are at most 2^24. Offsets out of order can
// overlap and so count rows more than once: sums past 2^30 stay above it without being exact, and callers take no more
// entries than groups without overlap have (most_tiles). Called by every thread of the block; ends with a barrier.
template <class Count>
__device__ __forceinline__ void build_table(int* start, int groups, Count count) {
    for (int g = threadIdx.x; g < groups; g += blockDim.x) start[g + 1] = count(g);
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
            run = min(run + __shfl_sync(0xffffffffu, v, 31), 1 << 30);
        }
    }
    __syncthreads();
}

// The table of row tiles (tile rows each).
__device__ __forceinline__ void build_tile_table(int* start, const int* __restrict__ offsets, int groups, int rows, int tile,
                                                 DeviceErrorRecord* err) {
    build_table(start, groups, [&](int g) {
        const GroupRange r = group_range(offsets, g, rows, err);
        return (r.end - r.begin + tile - 1) / tile;
    });
}

// Row tiles (of `tile` rows) that groups in order have at most.
__host__ __device__ __forceinline__ int most_tiles(int groups, int rows, int tile) { return rows / tile + (groups < rows ? groups : rows); }

// The group of entry m, 0 <= m < start[groups].
__device__ __forceinline__ int tile_group(const int* start, int groups, int m) {
    int lo = 0, hi = groups;  // start[lo] <= m < start[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (start[mid] <= m) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Adapter requests of one row are multiplied on CUDA cores, also in a batch with longer ones: a tensor-core tile of one row
// costs as much as one of 128.
__device__ __forceinline__ bool is_single(const GroupRange& r) { return r.end - r.begin == 1; }

// Partial sums of x[p] a[which[g]]^T (grouped_mm.cu), for lora.cu: parts[s][p][0 .. rank) for each of up to most_splits ranges
// of K, on the tensor cores; groups of one row have their whole sum in parts[0]. Rows of groups without a matrix are not
// written. Operands on 16-byte boundaries, rank and K multiples of 8.
struct PartialProducts {
    const int* offsets;
    const int* which;
    int groups, rows, matrices, rank, K, dtype;
    const void* x;
    long long ldx;
    const void* a;
    float* parts;
    int* singles;  // the number of groups of one row, the number of ranges, and those groups in order (2 + groups ints)
    int most_splits;
};
int partial_products(const PartialProducts& p, cudaStream_t s, DeviceState* st);

}  // namespace spmm_b200
