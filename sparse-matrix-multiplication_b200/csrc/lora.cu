// Low-rank adapters of many requests at once: out_p = base_p + s_i B_i (A_i x_p), i = the adapter of p's request.
//
// Two launches: shrink u_p = A_i x_p (rank values a row, FP32 in the workspace), expand out_p = base_p + s_i B_i u_p.
// Three forms of each: a few rows a request (CUDA cores, latency), many (tcgen05, the rows' bytes), any alignment. The last shares
// nothing between rows: 8200 mixed rows, N = K = 4096, rank 4 228 us (rank 8 by tcgen05 54), rank 64 and N = 4095 7.1 ms (65).

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <cstdint>

#include "groups.cuh"
#include "tcgen05.cuh"

namespace spmm_b200 {
namespace {

constexpr int kMaxRank = 256;

struct LoraArgs {
    int adapters, rank, N, K;
    const uint16_t* __restrict__ a;
    const uint16_t* __restrict__ b;
    const float* __restrict__ scale;
    const int* __restrict__ offsets;
    const int* __restrict__ adapter;
    int requests, rows;
    const uint16_t* __restrict__ x;
    long long ldx;
    const uint16_t* base;  // may be out itself
    long long ldbase;
    uint16_t* out;
    long long ldout;
    float* u;
    DeviceErrorRecord* err;
};

// The request of row p (-1: none): the last one that begins at or before p, if p is inside it.
__device__ __forceinline__ int request_of(const LoraArgs& a, int p) {
    if (!a.offsets) return p;
    int lo = 0, hi = a.requests;  // offsets[lo] <= p < offsets[hi] if p is in any
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (__ldg(a.offsets + mid) <= p) lo = mid;
        else hi = mid;
    }
    return __ldg(a.offsets + lo) <= p && p < __ldg(a.offsets + lo + 1) ? lo : -1;
}

// A request's adapter, -1 for none.
__device__ __forceinline__ int adapter_of(const LoraArgs& a, int r, DeviceErrorRecord* err) {
    const int i = __ldg(a.adapter + r);
    if (i >= a.adapters) record_device_error(err, SPMM_ERR_BAD_INDEX, r);
    return i < 0 || i >= a.adapters ? -1 : i;
}

// Bad offsets and adapters of all requests, those without rows too, to the record: by one block.
__device__ __forceinline__ void record_bad_requests(const LoraArgs& a) {
    for (int r = threadIdx.x; r < a.requests; r += blockDim.x) {
        if (a.offsets) group_range(a.offsets, r, a.rows, a.err);
        adapter_of(a, r, a.err);
    }
}

// ------------------------------------------------------------------ any alignment: one block a row

template <int DT>
__global__ void __launch_bounds__(256) lora_shrink_any_kernel(LoraArgs a) {
    grid_dependency_wait();
    allow_dependent_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int p = blockIdx.x; p < a.rows; p += gridDim.x) {
        const int r = request_of(a, p);
        const int i = r < 0 ? -1 : adapter_of(a, r, nullptr);
        if (i < 0) continue;
        for (int q = warp; q < a.rank; q += 8) {
            const uint16_t* row = a.a + (static_cast<long long>(i) * a.rank + q) * a.K;
            float s = 0.f;
            for (int k = lane; k < a.K; k += 32)
                s = fmaf(half_bits_to_float<DT>(__ldg(row + k)), half_bits_to_float<DT>(__ldg(a.x + p * a.ldx + k)), s);
#pragma unroll
            for (int d = 16; d > 0; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
            if (lane == 0) a.u[static_cast<long long>(p) * a.rank + q] = s;
        }
    }
}

template <int DT>
__global__ void __launch_bounds__(256) lora_expand_any_kernel(LoraArgs a) {
    __shared__ float u[kMaxRank];
    grid_dependency_wait();
    allow_dependent_launch();
    if (blockIdx.x == 0) record_bad_requests(a);
    for (int p = blockIdx.x; p < a.rows; p += gridDim.x) {
        const int r = request_of(a, p);
        if (r < 0) continue;
        const int i = adapter_of(a, r, nullptr);
        __syncthreads();
        if (i >= 0)
            for (int q = threadIdx.x; q < a.rank; q += 256) u[q] = a.u[static_cast<long long>(p) * a.rank + q];
        __syncthreads();
        const float s = i >= 0 && a.scale ? __ldg(a.scale + i) : 1.f;
        for (int n = threadIdx.x; n < a.N; n += 256) {
            float d = 0.f;
            if (i >= 0) {
                const uint16_t* row = a.b + (static_cast<long long>(i) * a.N + n) * a.rank;
                for (int q = 0; q < a.rank; ++q) d = fmaf(half_bits_to_float<DT>(__ldg(row + q)), u[q], d);
                d *= s;
            }
            if (a.base) {
                const float b = half_bits_to_float<DT>(a.base[p * a.ldbase + n]);
                d = i >= 0 ? b + d : b;
            }
            a.out[p * a.ldout + n] = float_to_half_bits<DT>(d);
        }
    }
}

// ------------------------------------------------------------------ few rows a request: CUDA cores
//
// With a row or a few to a request nothing is reused: the adapters' bytes bound the work, at single tokens its latency.
// Shrink: a block takes a row and four ranks, all its loads in flight at once. Expand: a thread takes one output, its
// row of b and its base are under way before the kernel waits for the shrink.

constexpr int kRanksPerBlock = 4;

template <int DT>
__global__ void __launch_bounds__(256) lora_shrink_rows_kernel(LoraArgs a, int rank_blocks) {
    __shared__ float sums[8][kRanksPerBlock];
    grid_dependency_wait();
    allow_dependent_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int p = blockIdx.x / rank_blocks, q0 = (blockIdx.x - p * rank_blocks) * kRanksPerBlock;
    const int r = request_of(a, p);
    const int i = r < 0 ? -1 : adapter_of(a, r, nullptr);
    if (i < 0) return;
    const uint4* x = reinterpret_cast<const uint4*>(a.x + p * a.ldx);
    const uint4* rows = reinterpret_cast<const uint4*>(a.a + (static_cast<long long>(i) * a.rank + q0) * a.K);
    const int nvec = a.K / 8;
    float s[kRanksPerBlock] = {};
#pragma unroll 2
    for (int c = threadIdx.x; c < nvec; c += 256) {
        const uint4 xv = __ldg(x + c);
        uint4 v[kRanksPerBlock];
#pragma unroll
        for (int q = 0; q < kRanksPerBlock; ++q) v[q] = __ldg(rows + static_cast<long long>(q) * nvec + c);  // rank is a multiple of 8
#pragma unroll
        for (int q = 0; q < kRanksPerBlock; ++q) s[q] = dot8<DT>(xv, v[q], s[q]);
    }
#pragma unroll
    for (int q = 0; q < kRanksPerBlock; ++q) {
#pragma unroll
        for (int d = 16; d > 0; d /= 2) s[q] += __shfl_xor_sync(0xffffffffu, s[q], d);
        if (lane == 0) sums[warp][q] = s[q];
    }
    __syncthreads();
    if (threadIdx.x < kRanksPerBlock) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) t += sums[w][threadIdx.x];
        a.u[static_cast<long long>(p) * a.rank + q0 + threadIdx.x] = t;
    }
}

template <int DT>
__global__ void __launch_bounds__(256) lora_expand_rows_kernel(LoraArgs a, int col_blocks) {
    constexpr int kAhead = 2;  // vectors of b's row that are loaded before the wait
    __shared__ __align__(16) float u[kMaxRank];
    // Reached only behind the shrink of the same call, which has itself waited for everything before it and writes
    // nothing but u: the rest may be read before this kernel's own wait.
    allow_dependent_launch();
    if (blockIdx.x == 0) record_bad_requests(a);
    const int p = blockIdx.x / col_blocks, n = (blockIdx.x - p * col_blocks) * 256 + threadIdx.x;
    const int r = request_of(a, p);
    const int i = r < 0 ? -1 : adapter_of(a, r, nullptr);
    const bool mine = r >= 0 && n < a.N;
    const uint4* row = reinterpret_cast<const uint4*>(a.b + (static_cast<long long>(max(i, 0)) * a.N + n) * a.rank);
    const int nvec = a.rank / 8;
    uint4 v[kAhead];
    float base = 0.f, scale = 1.f;
    if (mine) {
        if (i >= 0) {
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (k < nvec) v[k] = __ldg(row + k);
            if (a.scale) scale = __ldg(a.scale + i);
        }
        if (a.base) base = half_bits_to_float<DT>(a.base[p * a.ldbase + n]);
    }
    grid_dependency_wait();
    if (i >= 0)
        for (int q = threadIdx.x; q < a.rank; q += 256) u[q] = a.u[static_cast<long long>(p) * a.rank + q];
    __syncthreads();
    if (!mine) return;
    float d = 0.f;
    if (i >= 0) {
        const auto add = [&](const uint4& w, int k) {
            float f[8];
            RowVec<DT, 16>::unpack(w, f);
#pragma unroll
            for (int e = 0; e < 8; ++e) d = fmaf(f[e], u[8 * k + e], d);
        };
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (k < nvec) add(v[k], k);
#pragma unroll 4
        for (int k = kAhead; k < nvec; ++k) add(__ldg(row + k), k);
        d = a.base ? fmaf(d, scale, base) : d * scale;
    } else {
        d = base;
    }
    a.out[p * a.ldout + n] = float_to_half_bits<DT>(d);
}

// ------------------------------------------------------------------ many rows a request: tcgen05
//
// Shrink is the grouped product's kernel on 128-row tiles of the requests, its sum over K cut so that few tiles still
// fill the GPU (partial_products; FP32 parts in the workspace). Expand moves base and out (2 x rows x N) and computes
// little: a persistent block holds u of a 128-row tile in shared memory and streams b and base past it.
//   warp 0        TMA: b (TN features x rank) and the base tile (128 x TN) into a ring of stages, with what they are
//   warp 1        MMA: D = u b^T in TMEM, two accumulators
//   warps 2..17   D * scale + base (from the stage) -> 32-byte stores, two sets of eight on alternate stages
//   warps 18..21  the next row tile's u: the parts' sum as two 16-bit terms, hi + lo, K-major under the 128-byte swizzle
// Requests of one row come behind the tiles through the same ring: a stage is then as many of b's column tiles as it
// holds, and the epilogue warps take the dot products with u from it on CUDA cores (lanes loading b themselves took 17 us
// where the 100 single rows of a mixed batch now take 4).
// The MMA needs 16-bit u. In BF16 it takes three terms of eight bits each, which are u's FP32 value exactly: for three times
// the MMAs of one, which still run under the copies. The third, for which shared memory has no room, is in TMEM. In FP16 two
// terms leave 2^-22; they have neither the range nor the small steps of FP32, so a row of u is held with a power of two taken
// out, its largest element in [2^14, 2^15), and the epilogue puts it back.

constexpr int kTileM = 128;
constexpr int kSetWarps = 8;
constexpr int kEpilogueWarps = 2 * kSetWarps;
constexpr int kExpandThreads = (2 + kEpilogueWarps + 4) * 32;
constexpr int kSmallRows = 32;  // tiles with no more rows load a base box of this many

template <int RB>  // rank in blocks of 64
struct ExpandLayout {
    static constexpr int kTn = RB == 4 ? 64 : 128;
    static constexpr int kU = 2 * RB * 16384;                 // first terms' blocks, second's: 128 rows x 64 each
    static constexpr int kThird = RB * 32;                    // TMEM columns of the third terms (BF16), behind the accumulators
    static constexpr int kUs = RB == 1 ? 2 : 1;
    static constexpr int kB = RB * kTn * 128;
    static constexpr int kBase = kTn / 64 * 16384;            // 64-column blocks of 128 rows
    static constexpr int kStage = kB + kBase;
    // A single row's stage: column tiles of b, then the row's base, then (1 KB on) u in FP32.
    static constexpr int kSingle = RB == 1 ? 2 : 1;
    static constexpr int kSingleBase = kSingle * kB;
    static constexpr int kStages = RB == 1 ? 3 : (RB == 2 ? 2 : 1);
    static constexpr int kStage0 = kUs * kU;
    static constexpr int kBars = kStage0 + kStages * kStage;  // full[], empty[], u_full[2], u_empty[2], acc_full[2], acc_empty[2], drain, u_first
    static constexpr int kInfo = kBars + 8 * (2 * kStages + 10);  // StageInfo[kStages]
    // Powers of two taken out of u's rows, of kUs + 2 units: u of a unit is made once the MMAs of the unit kUs before it are
    // done, when the epilogue may still be at the last tile of that one and, if it has a single tile, of the one before it.
    static constexpr int kScales = 4;
    static constexpr int kExp = kInfo + 32 * kStages;  // int8_t[kScales][kTileM]
    static constexpr int kSlot = kExp + kScales * kTileM;
    static constexpr int kTable = kSlot + 8;
    static constexpr int kFixed = kTable + 1024;
    static constexpr int tmem_columns(int dtype) {
        const int used = 2 * kTn + (dtype == SPMM_DTYPE_BF16 ? kUs * kThird : 0);
        return used <= 128 ? 128 : (used <= 256 ? 256 : 512);
    }
};

struct ExpandArgs {
    LoraArgs l;
    const int* singles;  // from the shrink: the number of requests of one row, of parts, and those requests
    int ntiles;        // column tiles
};

// A run of column tiles of one row tile. A block takes an equal, contiguous range of all (row tile, column tile) pairs,
// row tiles outermost: at most one column tile more than any other, and u made once for each row tile that it meets.
struct Unit {
    int i;             // adapter, -1 none
    int row, rows;     // first row, rows of the tile
    int nt0, nt1;      // column tiles
};

// What a stage holds, from the producer, which runs ahead: finding a unit is a search and three loads that depend on
// one another, 1400 cycles that the other roles do not wait for.
struct StageInfo {
    int rows;          // 0: no more stages
    int row, i, nt;
    float scale;
    int16_t first, last;  // tile of its unit
    int tile;          // a tile for the tensor cores: 1 + the place of its unit's powers of two; else 0
    int singles;       // column tiles from nt on of a request of one row, else 0
};

// The unit that begins at pair t of the block's range, which ends before pair `end`.
__device__ __forceinline__ Unit unit_of(const ExpandArgs& e, const int* start, int t, int end) {
    const int m = t / e.ntiles;
    const int r = tile_group(start, e.l.requests, m);
    const GroupRange g = group_range(e.l.offsets, r, e.l.rows, nullptr);
    Unit x;
    x.row = g.begin + (m - start[r]) * kTileM;
    x.rows = min(kTileM, g.end - x.row);
    x.i = adapter_of(e.l, r, nullptr);
    x.nt0 = t - m * e.ntiles;
    x.nt1 = min(e.ntiles, end - m * e.ntiles);
    return x;
}

// u of one unit as three BF16 terms, by `warps` warps, a multiple of four, of which this is the `w`-th. A warp stores to its own
// quarter of the TMEM lanes, 16 rows x 32 ranks at a time: four lanes read and write a row's pieces side by side.
template <int RB>
__device__ __forceinline__ void make_u_bf16(const ExpandArgs& e, const Unit& x, uint8_t* u, uint32_t third, int w, int warps) {
    const LoraArgs& a = e.l;
    const int lane = threadIdx.x & 31, q = (threadIdx.x >> 5) & 3;
    const long long stride = static_cast<long long>(a.rows) * a.rank;
    const int splits = e.singles[1], halves = (a.rank + 31) / 32 * 2;  // what lies past the rank is zero
    tc_fence_after();  // the MMAs that read what was there before
    for (int k = w / 4; k < halves; k += warps / 4) {
        const int lane0 = 32 * q + 16 * (k & 1), row = lane0 + lane / 4, col = 32 * (k >> 1) + 4 * (lane & 3);
        if (lane0 >= x.rows) continue;
        float f[2][2][4] = {};  // of ranks col and col + 16, of rows row and row + 8
        if (row < x.rows && col < a.rank) {
            // All of a part's loads in flight together; what does not exist is the first again, and not used.
            const float* src = a.u + static_cast<long long>(x.row + row) * a.rank + col;
            const int right = col + 16 < a.rank ? 16 : 0, down = row + 8 < x.rows ? 8 * a.rank : 0;
#pragma unroll 4
            for (int s = 0; s < splits; ++s) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float4 v = *reinterpret_cast<const float4*>(src + s * stride + (c & 1) * down + (c >> 1) * right);
                    float(&g)[4] = f[c >> 1][c & 1];
                    g[0] += v.x, g[1] += v.y, g[2] += v.z, g[3] += v.w;
                }
            }
            if (!right) {
#pragma unroll
                for (int i = 0; i < 8; ++i) f[1][i / 4][i % 4] = 0.f;
            }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            uint32_t terms[3][2][2];
#pragma unroll
            for (int t = 0; t < 3; ++t) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // The upper halves of two words: what is cut off is exact in FP32, and nothing of an infinity or NaN.
                    float &even = f[c][i / 2][2 * (i & 1)], &odd = f[c][i / 2][2 * (i & 1) + 1];
                    const uint32_t lo = __float_as_uint(even), hi = __float_as_uint(odd);
                    terms[t][i / 2][i & 1] = __byte_perm(lo, hi, 0x7632);
                    even = fabsf(even) < INFINITY ? even - __uint_as_float(lo & 0xffff0000u) : 0.f;
                    odd = fabsf(odd) < INFINITY ? odd - __uint_as_float(hi & 0xffff0000u) : 0.f;
                }
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint4* piece = swizzled_piece(u + (t * RB + col / 64) * 16384, row + 8 * h, col / 8 % 8 + 2 * c);
                    reinterpret_cast<uint2*>(piece)[lane & 1] = make_uint2(terms[t][h][0], terms[t][h][1]);
                }
            }
            __syncwarp();
            tmem_st_16x8(third + 16 * (k >> 1) + 8 * c + (static_cast<uint32_t>(lane0) << 16), terms[2]);
        }
    }
    tmem_st_wait();
    tc_fence_before();
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
}

// u of one unit as two FP16 terms, by `warps` warps of which this is the `w`-th. A row's pieces of 8 ranks to consecutive lanes; the
// parts' loads of a piece are in flight together.
template <int RB>
__device__ __forceinline__ void make_u_f16(const ExpandArgs& e, const Unit& x, uint8_t* hi, int8_t* exponents, int w, int warps) {
    constexpr int DT = SPMM_DTYPE_F16;
    const LoraArgs& a = e.l;
    const int pieces = (a.rank + 15) / 16 * 2;  // the last may lie past the rank and is zero
    int lanes = 2;                              // that a row takes
    while (lanes < pieces) lanes *= 2;
    const int lane = threadIdx.x & 31, piece = lane & (lanes - 1), per_warp = 32 / lanes;
    const int splits = e.singles[1];
    const float* parts = a.u + static_cast<long long>(x.row) * a.rank;
    const long long stride = static_cast<long long>(a.rows) * a.rank;
    for (int row0 = w * per_warp; row0 < x.rows; row0 += warps * per_warp) {
        const int row = row0 + lane / lanes;
        float f[8] = {};
        if (row < x.rows && 8 * piece < a.rank) {
            const float* src = parts + static_cast<long long>(row) * a.rank + 8 * piece;
#pragma unroll 4
            for (int s = 0; s < splits; ++s) {
                const float4 lo = *reinterpret_cast<const float4*>(src + s * stride), hi4 = *reinterpret_cast<const float4*>(src + s * stride + 4);
                f[0] += lo.x, f[1] += lo.y, f[2] += lo.z, f[3] += lo.w;
                f[4] += hi4.x, f[5] += hi4.y, f[6] += hi4.z, f[7] += hi4.w;
            }
        }
        float most = 0.f;  // of the finite ones
#pragma unroll
        for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(f[j]) < INFINITY ? fabsf(f[j]) : 0.f);
        for (int d = lanes / 2; d > 0; d /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
        // Sums of products of FP16 values are 0 or between 2^-48 and 2^56: -62 <= exponent <= 42.
        const int exponent = most > 0.f ? static_cast<int>(__float_as_uint(most) >> 23) - 127 - 14 : 0;
        const float down = __uint_as_float(static_cast<uint32_t>(127 - exponent) << 23);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= down;
        if (piece == 0 && row < x.rows) exponents[row] = static_cast<int8_t>(exponent);
        if (row >= x.rows || piece >= pieces) continue;
        const uint4 top = RowVec<DT, 16>::pack(f);
        float g[8];
        RowVec<DT, 16>::unpack(top, g);
        // An infinity or NaN is hi's alone, or lo would undo it.
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = fabsf(g[j]) < INFINITY ? f[j] - g[j] : 0.f;
        const int at = row * 128 + piece / 8 * 16384 + (((piece % 8) ^ (row & 7)) << 4);
        *reinterpret_cast<uint4*>(hi + at) = top;
        *reinterpret_cast<uint4*>(hi + RB * 16384 + at) = RowVec<DT, 16>::pack(g);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
}

// One row's outputs from a stage of b's column tiles, by one of a set's warps: 8 lanes to a feature, 4 features a step.
// Gives the stage back once it is in registers.
template <int DT, int RB>
__device__ __forceinline__ void single_dots(const LoraArgs& a, const StageInfo& x, uint8_t* stage, int w, uint32_t empty,
                                            uint32_t acc_empty) {
    using L = ExpandLayout<RB>;
    constexpr int kSteps = L::kTn / kSetWarps / 4, kSums = L::kSingle * kSteps;  // of a column tile, of the stage
    static_assert(kSums <= 8, "a lane of the eight keeps each sum");
    const int lane = threadIdx.x & 31, piece = lane & 7;
    // The lane that keeps sum k has the feature of step k % kSteps of column tile k / kSteps.
    const int local = (piece / kSteps) * L::kTn + (w * kSteps + piece % kSteps) * 4 + lane / 8;
    float base = 0.f, d[kSums] = {};
    if (a.base) base = half_bits_to_float<DT>(reinterpret_cast<const uint16_t*>(stage + L::kSingleBase)[local % (L::kSingle * L::kTn)]);
    if (x.i >= 0) {
        const float* u = reinterpret_cast<const float*>(stage + L::kSingleBase + 1024);
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            const int q = 64 * b + 8 * piece;
            float4 lo = {}, hi = {};
            if (q < a.rank) lo = *reinterpret_cast<const float4*>(u + q), hi = *reinterpret_cast<const float4*>(u + q + 4);
#pragma unroll
            for (int k = 0; k < kSums; ++k) {  // of a tile that the stage does not have, too: those sums are not stored
                float f[8];
                RowVec<DT, 16>::unpack(*swizzled_piece(stage + k / kSteps * L::kB + b * L::kTn * 128, (w * kSteps + k % kSteps) * 4 + lane / 8, piece), f);
                d[k] = fmaf(f[0], lo.x, fmaf(f[1], lo.y, fmaf(f[2], lo.z, fmaf(f[3], lo.w, d[k]))));
                d[k] = fmaf(f[4], hi.x, fmaf(f[5], hi.y, fmaf(f[6], hi.z, fmaf(f[7], hi.w, d[k]))));
            }
        }
    }
    __syncwarp();
    if (lane == 0) {
        mbar_arrive_count(empty, 1);
        mbar_arrive_count(acc_empty, 1);
    }
    float mine = 0.f;
#pragma unroll
    for (int o = 4; o > 0; o /= 2) {
#pragma unroll
        for (int k = 0; k < kSums; ++k) d[k] += __shfl_xor_sync(0xffffffffu, d[k], o);
    }
#pragma unroll
    for (int k = 0; k < kSums; ++k) mine = piece == k ? d[k] : mine;
    const int n = x.nt * L::kTn + local;
    if (piece < kSums && piece / kSteps < x.singles && n < a.N)
        a.out[x.row * a.ldout + n] = float_to_half_bits<DT>(x.i >= 0 ? fmaf(mine, x.scale, base) : base);
    __syncwarp();
}

template <int DT, int RB>
__global__ void __launch_bounds__(kExpandThreads, 1)
    lora_expand_tc_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_base,
                          const __grid_constant__ CUtensorMap map_base_small, ExpandArgs e) {
    using L = ExpandLayout<RB>;
    constexpr int kStages = L::kStages, kTn = L::kTn, kUs = L::kUs;
    const LoraArgs& a = e.l;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_addr(smem_raw);
    uint8_t* base = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    const uint32_t sbase = smem_addr(base);
    const uint32_t full0 = sbase + L::kBars, empty0 = full0 + 8 * kStages, u_full0 = empty0 + 8 * kStages, u_empty0 = u_full0 + 16,
                   acc_full0 = u_empty0 + 16, acc_empty0 = acc_full0 + 16, drain = acc_empty0 + 16, u_first = drain + 8;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base + L::kSlot);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    StageInfo* infos = reinterpret_cast<StageInfo*>(base + L::kInfo);
    int8_t* exponents = reinterpret_cast<int8_t*>(base + L::kExp);
    int* start = reinterpret_cast<int*>(base + L::kTable);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, kSetWarps);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(u_full0 + 8 * s, 4);
            mbar_init(u_empty0 + 8 * s, 1);
            mbar_init(acc_full0 + 8 * s, 1);
            mbar_init(acc_empty0 + 8 * s, kSetWarps);
        }
        mbar_init(drain, 1);
        mbar_init(u_first, kExpandThreads / 32 - 2);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetch_tensormap(&map_b);
        if (a.base) prefetch_tensormap(&map_base);
    }
    if (warp == 1) tmem_alloc(smem_addr(tmem_slot), L::tmem_columns(DT));
    // The shrink itself waited for everything before it, and writes nothing but the parts: the first stages' b and base are
    // loaded while it runs. Every role waits for its end before a bounded wait that could cover it.
    allow_dependent_launch();
    build_table(start, a.requests, [&](int r) {
        const GroupRange g = group_range(a.offsets, r, a.rows, blockIdx.x == 0 ? a.err : nullptr);
        return is_single(g) ? 0 : (g.end - g.begin + kTileM - 1) / kTileM;
    });
    const long long pairs = static_cast<long long>(min(start[a.requests], most_tiles(a.requests, a.rows, kTileM))) * e.ntiles;
    const int begin = static_cast<int>(pairs * blockIdx.x / gridDim.x), end = static_cast<int>(pairs * (blockIdx.x + 1) / gridDim.x);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // u of a unit: into buffer `buf`, `order`-th of the block's units with an adapter.
    const auto make_u = [&](const Unit& x, int buf, int order, int w, int warps) {
        if constexpr (DT == SPMM_DTYPE_BF16) make_u_bf16<RB>(e, x, base + buf * L::kU, tmem + 2 * kTn + buf * L::kThird, w, warps);
        else make_u_f16<RB>(e, x, base + buf * L::kU, exponents + order % L::kScales * kTileM, w, warps);
    };
    // The first unit with an adapter has its u made by every warp but the first two: nothing else can begin without it.
    if (warp >= 2) {
        grid_dependency_wait();
        for (int t = begin; t < end;) {
            const Unit x = unit_of(e, start, t, end);
            t += x.nt1 - x.nt0;
            if (x.i < 0) continue;
            make_u(x, 0, 0, warp - 2, kExpandThreads / 32 - 2);
            if (lane == 0) mbar_arrive_count(u_first, 1);
            break;
        }
    }

    if (warp == 0) {
        // ---------------- producer
        if (elect_one()) {
            int it = 0, nu = 0;
            bool ok = true;
            // The next stage, once it is free, with its description; its copies follow.
            const auto claim = [&](const StageInfo& info) {
                const int s = it % kStages;
                if (it == kStages) grid_dependency_wait();
                ok = mbar_wait(empty0 + 8 * s, ((it / kStages) & 1u) ^ 1u, abort_flag);
                if (ok) {
                    infos[s] = info;
                    ++it;
                }
                return s;
            };
            for (int t = begin; ok && t < end;) {
                const Unit x = unit_of(e, start, t, end);
                t += x.nt1 - x.nt0;
                const bool small = x.rows <= kSmallRows;
                const float scale = x.i >= 0 && a.scale ? __ldg(a.scale + x.i) : 1.f;
                const int tile = x.i >= 0 ? 1 + nu++ % L::kScales : 0;
                for (int nt = x.nt0; nt < x.nt1; ++nt) {
                    const int s = claim({x.rows, x.row, x.i, nt, scale, nt == x.nt0, nt == x.nt1 - 1, tile, 0});
                    if (!ok) break;
                    const uint32_t bar = full0 + 8 * s, sb = sbase + L::kStage0 + s * L::kStage, sbs = sb + L::kB;
                    const int n0 = nt * kTn, blocks = min(kTn / 64, (a.N - n0 + 63) / 64);
                    mbar_arrive_expect_tx(bar, static_cast<uint32_t>(x.i >= 0 ? L::kB : 0) + (a.base ? blocks * (small ? kSmallRows * 128 : 16384) : 0));
                    if (x.i >= 0)
                        for (int k = 0; k < RB; ++k) tma_load_3d(sb + k * kTn * 128, &map_b, bar, 64 * k, n0, x.i);
                    if (a.base)
                        for (int k = 0; k < blocks; ++k)
                            tma_load_2d(sbs + k * 16384, small ? &map_base_small : &map_base, bar, n0 + 64 * k, x.row);
                }
            }
            grid_dependency_wait();  // the list is the shrink's
            const int pieces = (e.ntiles + L::kSingle - 1) / L::kSingle;
            const long long items = static_cast<long long>(e.singles[0]) * pieces;
            const long long last = items * (blockIdx.x + 1) / gridDim.x;
            int m = -1;
            StageInfo info{};
            for (long long k = items * blockIdx.x / gridDim.x; ok && k < last; ++k) {
                if (k / pieces != m) {
                    m = static_cast<int>(k / pieces);
                    const int r = e.singles[2 + m];
                    info.rows = 1;
                    info.row = group_range(a.offsets, r, a.rows, nullptr).begin;
                    info.i = adapter_of(a, r, nullptr);
                    info.scale = info.i >= 0 && a.scale ? __ldg(a.scale + info.i) : 1.f;
                }
                info.nt = static_cast<int>(k - static_cast<long long>(m) * pieces) * L::kSingle;
                info.singles = min(L::kSingle, e.ntiles - info.nt);
                const int s = claim(info);
                if (!ok) break;
                const uint32_t bar = full0 + 8 * s, sb = sbase + L::kStage0 + s * L::kStage;
                const uint32_t bytes = a.base ? 2 * min(info.singles * kTn, a.N - info.nt * kTn) : 0;
                mbar_arrive_expect_tx(bar, bytes + (info.i >= 0 ? info.singles * L::kB + 4 * a.rank : 0));
                if (a.base) bulk_load(sb + L::kSingleBase, a.base + info.row * a.ldbase + info.nt * kTn, bytes, bar);
                if (info.i >= 0) {
                    bulk_load(sb + L::kSingleBase + 1024, a.u + static_cast<long long>(info.row) * a.rank, 4 * a.rank, bar);
                    for (int j = 0; j < info.singles; ++j)
                        for (int b = 0; b < RB; ++b)
                            tma_load_3d(sb + j * L::kB + b * kTn * 128, &map_b, bar, 64 * b, (info.nt + j) * kTn, info.i);
                }
            }
            for (int k = 0; ok && k < 2; ++k) {  // the end, for either set of epilogue warps
                const int s = claim({});
                if (ok) mbar_arrive_count(full0 + 8 * s, 1);
            }
            if (!ok) {
                *abort_flag = 1;
                record_device_error(a.err, SPMM_ERR_TIMEOUT, 21);
            }
            for (int i = max(0, it - kStages); i < it; ++i) {
                const unsigned long long t0 = global_ns();
                while (!mbar_try_wait(full0 + 8 * (i % kStages), (i / kStages) & 1u) && global_ns() - t0 < kWaitNs) {
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer
        if (elect_one()) {
            const uint32_t idesc = instr_desc_f16(DT, kTn, false, false);
            const int slices = (a.rank + 15) / 16;
            int nu = 0;
            bool ok = true;
            grid_dependency_wait();
            // Stage `it` goes to epilogue set it & 1 with accumulator it & 1, whether or not it is a tile: so a set sees every
            // phase of its barriers, in order.
            for (int it = 0, ends = 0; ends < 2; ++it) {
                const int s = it % kStages, ub = nu % kUs, buf = it & 1;
                ok = mbar_wait(full0 + 8 * s, (it / kStages) & 1u, abort_flag) &&
                     mbar_wait(acc_empty0 + 8 * buf, ((it >> 1) & 1u) ^ 1u, abort_flag);
                if (!ok) break;
                const StageInfo x = infos[s];
                if (!x.tile) {
                    ends += x.rows == 0;
                    mbar_arrive_count(acc_full0 + 8 * buf, 1);
                    continue;
                }
                ok = !x.first || (nu == 0 ? mbar_wait(u_first, 0, abort_flag) : mbar_wait(u_full0 + 8 * ub, ((nu - (ub == 0)) / kUs) & 1u, abort_flag));
                if (!ok) break;
                tc_fence_after();
                const uint32_t su = sbase + ub * L::kU, sb = sbase + L::kStage0 + s * L::kStage;
                const uint32_t acc = tmem + buf * kTn;
                for (int t = 0; t < 2; ++t)
                    for (int k = 0; k < slices; ++k) {
                        const uint64_t da = smem_desc(su + (t * RB + k / 4) * 16384 + 32 * (k % 4), 16, 1024, kSwizzle128);
                        const uint64_t db = smem_desc(sb + k / 4 * kTn * 128 + 32 * (k % 4), 16, 1024, kSwizzle128);
                        umma_f16(acc, da, db, idesc, t + k > 0 ? 1u : 0u);
                    }
                if constexpr (DT == SPMM_DTYPE_BF16) {
                    for (int k = 0; k < slices; ++k)
                        umma_f16_tmem_a(acc, tmem + 2 * kTn + ub * L::kThird + 8 * k, smem_desc(sb + k / 4 * kTn * 128 + 32 * (k % 4), 16, 1024, kSwizzle128), idesc, 1u);
                }
                umma_commit(acc_full0 + 8 * buf);
                if (x.last) {
                    umma_commit(u_empty0 + 8 * ub);
                    ++nu;
                }
            }
            if (!ok) {
                *abort_flag = 1;
                record_device_error(a.err, SPMM_ERR_TIMEOUT, 22);
            }
        }
        __syncwarp();
    } else if (warp < 2 + kEpilogueWarps) {
        // ---------------- epilogue: two sets of eight warps take alternate stages; in a set two warps a lane quarter
        const int set = (warp - 2) / kSetWarps, w = (warp - 2) % kSetWarps, q = warp & 3, half = w / 4;
        const bool sectors = (reinterpret_cast<uintptr_t>(a.out) | static_cast<uintptr_t>(a.ldout * 2)) % 32 == 0;
        bool ok = true;
        for (int it = set;; it += 2) {
            const int s = it % kStages;
            uint8_t* stage = base + L::kStage0 + s * L::kStage;
            // The stage's own barrier too, for the copies' writes; its phase cannot pass before this set gives the stage back.
            ok = __all_sync(0xffffffffu, mbar_wait(acc_full0 + 8 * set, (it >> 1) & 1u, abort_flag) &&
                                             mbar_wait(full0 + 8 * s, (it / kStages) & 1u, abort_flag));
            if (!ok) break;
            tc_fence_after();
            const StageInfo x = infos[s];
            if (x.singles) {
                single_dots<DT, RB>(a, x, stage, w, empty0 + 8 * s, acc_empty0 + 8 * set);
                continue;
            }
            const int cols = min(kTn, a.N - x.nt * kTn), row = q * 32 + lane;
            uint16_t* out = a.out + (x.row + row) * a.ldout + x.nt * kTn;
            float up = 1.f;
            if (DT == SPMM_DTYPE_F16 && x.tile) up = __uint_as_float(static_cast<uint32_t>(127 + exponents[(x.tile - 1) * kTileM + row]) << 23);
            if (q * 32 < x.rows) {
                // 32 columns at a time, half of a 64-column block (16 KB of the stage).
                for (int c0 = half * 32; c0 < cols; c0 += 64) {
                    uint4 o[4] = {};
                    if (a.base) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) o[c] = *swizzled_piece(stage + L::kB + c0 / 64 * 16384, row, 4 * half + c);
                    }
                    if (x.tile) {
                        uint32_t v[32];
                        tmem_ld32(tmem + set * kTn + c0 + (static_cast<uint32_t>(q * 32) << 16), v);
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            float f[8];
                            RowVec<DT, 16>::unpack(o[c], f);
#pragma unroll
                            for (int k = 0; k < 8; ++k) f[k] = fmaf(DT == SPMM_DTYPE_F16 ? __uint_as_float(v[8 * c + k]) * up : __uint_as_float(v[8 * c + k]), x.scale, f[k]);
                            o[c] = RowVec<DT, 16>::pack(f);
                        }
                    }
                    if (row < x.rows) {
                        uint4* at = reinterpret_cast<uint4*>(out + c0);
                        if (sectors && c0 + 32 <= cols) {
                            store_32(at, o[0], o[1]);
                            store_32(at + 2, o[2], o[3]);
                        } else {
#pragma unroll
                            for (int c = 0; c < 4; ++c)
                                if (c0 + 8 * c < cols) at[c] = o[c];
                        }
                    }
                    __syncwarp();
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive_count(empty0 + 8 * s, 1);
                mbar_arrive_count(acc_empty0 + 8 * set, 1);
            }
            if (x.rows == 0) break;
        }
        if (!ok && lane == 0) {
            *abort_flag = 1;
            record_device_error(a.err, SPMM_ERR_TIMEOUT, 23);
        }
    } else {
        // ---------------- u of the units behind the first
        int nu = 0;
        bool ok = true;
        for (int t = begin; ok && t < end;) {
            const Unit x = unit_of(e, start, t, end);
            t += x.nt1 - x.nt0;
            if (x.i < 0) continue;
            const int ub = nu % kUs;
            if (nu > 0) {
                ok = __all_sync(0xffffffffu, mbar_wait_sum(u_empty0 + 8 * ub, ((nu / kUs) & 1u) ^ 1u, abort_flag, kUs * e.ntiles));
                if (!ok) break;
                make_u(x, ub, nu, warp - 2 - kEpilogueWarps, 4);
                if (lane == 0) mbar_arrive_count(u_full0 + 8 * ub, 1);
            }
            ++nu;
        }
        if (!ok && lane == 0) {
            *abort_flag = 1;
            record_device_error(a.err, SPMM_ERR_TIMEOUT, 24);
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        // The last commits' arrivals, and after a timeout the MMAs in flight, end before the block gives up its TMEM.
        if (elect_one()) {
            umma_commit(drain);
            const unsigned long long t0 = global_ns();
            while (!mbar_try_wait(drain, 0) && global_ns() - t0 < kWaitNs) {
            }
        }
        __syncwarp();
        tmem_dealloc(tmem, L::tmem_columns(DT));
    }
}

template <int DT, int RB>
int expand_launch(const CUtensorMap& mb, const CUtensorMap& ms, const CUtensorMap& small, const ExpandArgs& e, cudaStream_t s,
                  DeviceState* st) {
    using L = ExpandLayout<RB>;
    static std::atomic<unsigned long long> attr_set{0};
    const unsigned long long bit = st->device < 64 ? 1ull << st->device : 0ull;
    if (!bit || !(attr_set.load(std::memory_order_acquire) & bit)) {
        SPMM_CUDA_TRY(cudaFuncSetAttribute(lora_expand_tc_kernel<DT, RB>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           L::kFixed + 4 * (SPMM_MAX_GROUPS + 1)));
        attr_set.fetch_or(bit, std::memory_order_acq_rel);
    }
    const size_t smem = L::kFixed + 4 * (static_cast<size_t>(e.l.requests) + 1);
    return launch_dependent(lora_expand_tc_kernel<DT, RB>, dim3(st->sm_count), dim3(kExpandThreads), smem, s, mb, ms, small, e);
}

template <int DT>
int expand(const ExpandArgs& e0, int64_t mtiles, cudaStream_t s, DeviceState* st) {
    ExpandArgs e = e0;
    const LoraArgs& a = e.l;
    const int rb = a.rank <= 64 ? 1 : (a.rank <= 128 ? 2 : 4);
    const int tn = rb == 4 ? 64 : 128;
    e.ntiles = (a.N + tn - 1) / tn;
    if (mtiles * e.ntiles > INT32_MAX) return SPMM_ERR_TOO_LARGE;
    CUtensorMap mb, ms{}, small{};
    const uint64_t N = a.N, rank = a.rank, rows = a.rows;
    SPMM_TRY(encode_3d(&mb, a.b, {rank, N, static_cast<uint64_t>(a.adapters)}, {rank * 2, N * rank * 2}, {64, static_cast<uint32_t>(tn), 1},
                       CU_TENSOR_MAP_SWIZZLE_128B));
    if (a.base) {
        SPMM_TRY(encode_2d(&ms, a.base, N, rows, a.ldbase * 2, 64, kTileM, CU_TENSOR_MAP_SWIZZLE_128B));
        SPMM_TRY(encode_2d(&small, a.base, N, rows, a.ldbase * 2, 64, kSmallRows, CU_TENSOR_MAP_SWIZZLE_128B));
    }
    if (rb == 1) return expand_launch<DT, 1>(mb, ms, small, e, s, st);
    if (rb == 2) return expand_launch<DT, 2>(mb, ms, small, e, s, st);
    return expand_launch<DT, 4>(mb, ms, small, e, s, st);
}

// ------------------------------------------------------------------ host

// How a call runs, by its sizes alone (the lengths are on the device). `fits`: 16-byte boundaries throughout.
struct Shape {
    bool rows;         // CUDA cores, a few rows a request
    int most_splits;   // parts of u
    int64_t mtiles;
};

Shape shape_of(const spmm_lora_view& l, int32_t requests, int32_t rows) {
    Shape h{};
    const int64_t K = l.K;
    // Few rows a request, and the form with the smaller estimate in ns: rows, each with its adapter through L2 (5.2 TB/s) and its
    // blocks' share, or tiles, a start and each request's column tiles (half of one where no request has more than one row).
    // Four rows a request at most: beyond them the requests are rarely all short, and a long one costs the row form most.
    // Measured, us, rows and tiles, BF16, N = K = 4096: 32 single rows, rank 16 4.9, 16.4; 256 single rows, rank 16 20, 31, rank 64
    // 58, 42; 256 requests of 2, rank 16 35, 81, rank 64 109, 87; a prompt of 380 and 128 single rows, rank 16 33, 27, rank 64 106, 34;
    // 2000 single rows, rank 8 117, 249, rank 64 430, 256.
    const int64_t vectors = static_cast<int64_t>(l.rank) * (static_cast<int64_t>(l.N) + K);
    const int64_t rows_ns = rows * (vectors / 2600 + l.rank / 4 + l.N / 256);
    const int64_t tiles_ns = 12000 + requests * ((static_cast<int64_t>(l.N) + 127) / 128) * (rows <= requests ? 4 : 8);
    h.rows = rows <= 4 * static_cast<int64_t>(requests) && rows_ns <= tiles_ns;
    h.mtiles = most_tiles(requests, rows, kTileM);
    // Ranges of the sum over K, from which the shrink chooses: enough that few tiles fill the GPU, each at least 4 steps of 64.
    h.most_splits = h.rows ? 1 : static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({8, 1184 / std::max<int64_t>(1, h.mtiles), K / 256})));
    return h;
}

bool fits16(const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; }

int check_view(const spmm_lora_view* l, int32_t requests, int32_t rows) {
    if (!l || l->adapters < 0 || l->rank < 0 || l->N < 0 || l->K < 0 || requests < 0 || rows < 0) return SPMM_ERR_INVALID_ARG;
    if (l->dtype != SPMM_DTYPE_F16 && l->dtype != SPMM_DTYPE_BF16) return SPMM_ERR_INVALID_ARG;
    if (l->rank > kMaxRank || requests > SPMM_MAX_GROUPS || rows > INT32_MAX - 256 || l->N > (1 << 24) || l->K > (1 << 24))
        return SPMM_ERR_TOO_LARGE;
    return SPMM_OK;
}

int check_operand(const void* p, int64_t ld, int64_t cols) {
    if (!p || ld < cols || ld > (INT64_C(1) << 32)) return SPMM_ERR_INVALID_ARG;
    return reinterpret_cast<uintptr_t>(p) % 2 ? SPMM_ERR_MISALIGNED : SPMM_OK;
}

}  // namespace
}  // namespace spmm_b200

using namespace spmm_b200;

extern "C" {

int spmm_lora_workspace_size(const spmm_lora_view* l, int32_t requests, int32_t rows, size_t* bytes) {
    SPMM_TRY(check_view(l, requests, rows));
    if (!bytes) return SPMM_ERR_INVALID_ARG;
    const Shape h = shape_of(*l, requests, rows);
    *bytes = sizeof(float) * static_cast<size_t>(rows) * l->rank * h.most_splits + (h.rows ? 0 : sizeof(int) * (2 + static_cast<size_t>(requests)));
    return SPMM_OK;
}

int spmm_lora(const spmm_lora_view* l, const int32_t* offsets, const int32_t* adapter, int32_t requests, int32_t rows, const void* x,
              int64_t ldx, const void* base, int64_t ldbase, void* out, int64_t ldout, void* ws, size_t ws_bytes, void* stream) {
    size_t need = 0;
    SPMM_TRY(spmm_lora_workspace_size(l, requests, rows, &need));
    if (!offsets && requests != rows) return SPMM_ERR_INVALID_ARG;
    const bool some = rows > 0 && requests > 0 && l->N > 0;
    const bool adds = some && l->adapters > 0 && l->rank > 0;
    if (some) {
        if (!adapter) return SPMM_ERR_INVALID_ARG;
        if (!words_fit(offsets, adapter, l->scale)) return SPMM_ERR_MISALIGNED;
        SPMM_TRY(check_operand(out, ldout, l->N));
        if (base) SPMM_TRY(check_operand(base, ldbase, l->N));
        if (base == out && ldbase != ldout) return SPMM_ERR_INVALID_ARG;
    }
    if (adds) {
        SPMM_TRY(check_operand(l->b, l->rank, l->rank));
        if (l->K > 0) {
            SPMM_TRY(check_operand(l->a, l->K, l->K));
            SPMM_TRY(check_operand(x, ldx, l->K));
        }
        if (need > 0 && (!ws || ws_bytes < need)) return SPMM_ERR_INVALID_ARG;
        if (reinterpret_cast<uintptr_t>(ws) % 256) return SPMM_ERR_MISALIGNED;
    }
    DeviceState* st = nullptr;
    SPMM_TRY(current_device_state(&st));
    if (!some) return SPMM_OK;
    LoraArgs a{};
    a.adapters = l->adapters;
    a.rank = l->rank;
    a.N = l->N;
    a.K = l->K;
    a.a = static_cast<const uint16_t*>(l->a);
    a.b = static_cast<const uint16_t*>(l->b);
    a.scale = l->scale;
    a.offsets = offsets;
    a.adapter = adapter;
    a.requests = requests;
    a.rows = rows;
    a.x = static_cast<const uint16_t*>(x);
    a.ldx = ldx;
    a.base = static_cast<const uint16_t*>(base);
    a.ldbase = ldbase;
    a.out = static_cast<uint16_t*>(out);
    a.ldout = ldout;
    a.u = static_cast<float*>(ws);
    a.err = st->err;
    const cudaStream_t s = as_stream(stream);
    const bool bf16 = l->dtype == SPMM_DTYPE_BF16;
    const bool fits = adds && st->cc_major == 10 && l->K > 0 && l->K % 8 == 0 && l->N % 8 == 0 && l->rank % 8 == 0 && fits16(x, ldx) &&
                      fits16(out, ldout) && (!base || fits16(base, ldbase)) && fits16(l->a, 8) && fits16(l->b, 8);
    const Shape h = shape_of(*l, requests, rows);
    if (fits && h.rows) {
        const int rank_blocks = l->rank / kRanksPerBlock, col_blocks = (l->N + 255) / 256;
        const int64_t blocks = static_cast<int64_t>(rows) * std::max(rank_blocks, col_blocks);
        if (blocks > INT32_MAX) return SPMM_ERR_TOO_LARGE;
        SPMM_TRY(launch_dependent(bf16 ? lora_shrink_rows_kernel<SPMM_DTYPE_BF16> : lora_shrink_rows_kernel<SPMM_DTYPE_F16>,
                                  dim3(static_cast<unsigned>(rows) * rank_blocks), dim3(256), 0, s, a, rank_blocks));
        return launch_dependent(bf16 ? lora_expand_rows_kernel<SPMM_DTYPE_BF16> : lora_expand_rows_kernel<SPMM_DTYPE_F16>,
                                dim3(static_cast<unsigned>(rows) * col_blocks), dim3(256), 0, s, a, col_blocks);
    }
    if (fits) {
        PartialProducts p{offsets, adapter, requests, rows, l->adapters, l->rank, l->K, l->dtype, x, ldx, l->a, a.u, nullptr, h.most_splits};
        p.singles = reinterpret_cast<int*>(a.u + static_cast<size_t>(rows) * l->rank * h.most_splits);
        SPMM_TRY(partial_products(p, s, st));
        ExpandArgs e{};
        e.l = a;
        e.singles = p.singles;
        return bf16 ? expand<SPMM_DTYPE_BF16>(e, h.mtiles, s, st) : expand<SPMM_DTYPE_F16>(e, h.mtiles, s, st);
    }
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(rows, st->sm_count * 8)));
    if (adds)
        SPMM_TRY(launch_dependent(bf16 ? lora_shrink_any_kernel<SPMM_DTYPE_BF16> : lora_shrink_any_kernel<SPMM_DTYPE_F16>, grid, dim3(256), 0,
                                  s, a));
    return launch_dependent(bf16 ? lora_expand_any_kernel<SPMM_DTYPE_BF16> : lora_expand_any_kernel<SPMM_DTYPE_F16>, grid, dim3(256), 0, s,
                            a);
}

}  // extern "C"
