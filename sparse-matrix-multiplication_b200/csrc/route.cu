// Tokens routed to groups (experts) and back.
//
// The routing matrix R (tokens x sorted rows) has one 1 (or w[t, j]) at (t, pos[t, j]) for every pair that has a
// row. spmm_route_build sorts the pairs by group (a counting sort, stable), spmm_route_gather computes R1^T x,
// spmm_route_combine R_w ys, spmm_route_combine_grad the gradients R_w^T dy and (dy ys^T) at R's nonzeros.
// The three row kernels move rows and compute next to nothing: the rows' bytes through HBM bound them.
// All three walk tokens, not sorted rows, so that a token's own row crosses HBM once for its topk pairs.

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cstdint>

#include "rows.cuh"
#include "tcgen05.cuh"

namespace spmm_b200 {
namespace {

constexpr unsigned kFull = 0xffffffffu;

// ------------------------------------------------------------------ sort
//
// Counting sort over blocks of `per_block` pairs. With one block the histogram, its scan and the placement are one
// launch; with more, a first launch leaves each block's histogram in the workspace and every block of the second
// adds up what it needs (blocks x groups ints from L2), so there is no wait between blocks.

constexpr int kMaxSortThreads = 1024;
// Pairs that one block takes alone, without a workspace. 2048 of them: 3.8 / 5.3 / 9.6 us for 8 / 256 / 4096 groups, in two launches
// 5.7 / 6.8 / 11.4; 4096: 5.3 / 8.8 / 13.5, in two launches 5.9 / 7.6 / 13.5.
constexpr int kOneBlock = 4096;
// 131072 pairs, 8 / 256 / 4096 groups: 6.8 / 9.8 / 30.5 us; 1024 a block 7.2 / 26.2 / 48.3 (128 histograms for every block to add
// up); 4096 a block 7.8 / 12.6 / 27.9. The histograms and the order within a block bound it, not the 1.6 MB.
constexpr int kPairsPerBlock = 2048;
constexpr int kMaxSortBlocks = 128;   // blocks grow beyond kPairsPerBlock instead
constexpr int kMaxSortSmem = 4 * (10 * SPMM_MAX_GROUPS + 33);  // 8 histograms, totals and prefixes of the most groups: 160 KiB

struct SortShape {
    int warps;      // warps with a histogram of their own
    int blocks;
    int per_block;  // a multiple of 32 * warps
    size_t smem;
};

SortShape sort_shape(int pairs, int groups) {
    SortShape s{};
    // 128 pairs a warp (four steps) in blocks of the usual size; per-warp histograms (ints) within 128 KiB, totals and block
    // prefixes behind them.
    const int usual = pairs <= kOneBlock ? kOneBlock : kPairsPerBlock;
    s.warps = std::min(groups <= 1024 ? 32 : (groups <= 2048 ? 16 : 8), std::max(4, (std::min(pairs, usual) + 127) / 128));
    const int unit = 32 * s.warps;
    const long long want = std::max<long long>(std::max(1, std::min(pairs, usual)), (static_cast<long long>(pairs) + kMaxSortBlocks - 1) / kMaxSortBlocks);
    s.per_block = static_cast<int>((want + unit - 1) / unit * unit);
    s.blocks = std::max(1, static_cast<int>((static_cast<long long>(pairs) + s.per_block - 1) / s.per_block));
    s.smem = sizeof(int) * (static_cast<size_t>(s.warps) * groups + 2 * static_cast<size_t>(groups) + 1 + 32);
    return s;
}

// A pair's group, -1 for none.
__device__ __forceinline__ int group_of(const int* __restrict__ ids, int i, int groups, DeviceErrorRecord* err) {
    const int id = __ldg(ids + i);
    if (id >= groups) record_device_error(err, SPMM_ERR_BAD_INDEX, i);
    return id < 0 || id >= groups ? -1 : id;
}

__global__ void __launch_bounds__(kMaxSortThreads) route_count_kernel(const int* __restrict__ ids, int pairs, int groups,
                                                                   int per_block, int* __restrict__ counts,
                                                                   DeviceErrorRecord* err) {
    extern __shared__ int sm[];
    for (int g = threadIdx.x; g < groups; g += blockDim.x) sm[g] = 0;
    __syncthreads();
    grid_dependency_wait();
    allow_dependent_launch();
    const int begin = blockIdx.x * per_block, end = begin + min(per_block, pairs - begin);
    for (int i = begin + threadIdx.x; i < end; i += blockDim.x) {
        const int g = group_of(ids, i, groups, err);
        if (g >= 0) atomicAdd(sm + g, 1);
    }
    __syncthreads();
    for (int g = threadIdx.x; g < groups; g += blockDim.x) counts[static_cast<size_t>(blockIdx.x) * groups + g] = sm[g];
}

__global__ void __launch_bounds__(kMaxSortThreads)
    route_place_kernel(const int* __restrict__ ids, int pairs, int groups, int warps, int per_block,
                       const int* __restrict__ counts, int* __restrict__ offsets, int* __restrict__ order,
                       int* __restrict__ pos, DeviceErrorRecord* err) {
    extern __shared__ int sm[];
    int* hist = sm;                       // [warps][groups]: counts, then each warp's next row
    int* total = hist + warps * groups;   // [groups + 1]: counts over all blocks, then offsets
    int* before = total + groups + 1;     // [groups]: counts of the blocks before this one
    int* part = before + groups;          // [32]: scan of the warps' sums
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool alone = gridDim.x == 1;

    for (int i = threadIdx.x; i < warps * groups + 2 * groups + 1; i += blockDim.x) sm[i] = 0;
    __syncthreads();
    grid_dependency_wait();
    allow_dependent_launch();

    // Warp w owns the w-th run of per_block / warps pairs: pairs of one group keep their order.
    const int per_warp = per_block / warps;
    const int begin = static_cast<int>(min(static_cast<long long>(pairs),
                                           static_cast<long long>(blockIdx.x) * per_block + static_cast<long long>(warp) * per_warp));
    const int end = warp < warps ? begin + min(per_warp, pairs - begin) : begin;
    int* mine = hist + warp * groups;
#pragma unroll 4
    for (int i = begin + lane; i < end; i += 32) {
        const int g = group_of(ids, i, groups, alone ? err : nullptr);
        if (g >= 0) atomicAdd(mine + g, 1);
    }
    if (!alone) {
        const int parts = max(1, static_cast<int>(blockDim.x) / groups);
        for (int u = threadIdx.x; u < parts * groups; u += blockDim.x) {
            const int g = u % groups;
            int all = 0, prev = 0;
#pragma unroll 16
            for (int b = u / groups; b < static_cast<int>(gridDim.x); b += parts) {
                const int c = __ldg(counts + static_cast<size_t>(b) * groups + g);
                all += c;
                prev += b < static_cast<int>(blockIdx.x) ? c : 0;
            }
            atomicAdd(total + g, all);
            atomicAdd(before + g, prev);
        }
    }
    __syncthreads();
    if (alone) {
        for (int g = threadIdx.x; g < groups; g += blockDim.x) {
            int all = 0;
            for (int w = 0; w < warps; ++w) all += hist[w * groups + g];
            total[g] = all;
        }
        __syncthreads();
    }
    // Exclusive scan of the totals: each thread a run of them, warps by shuffles, then the warps' sums.
    const int run = (groups + blockDim.x - 1) / blockDim.x;
    const int g0 = min(groups, static_cast<int>(threadIdx.x) * run), g1 = min(groups, g0 + run);
    int sum = 0;
    for (int g = g0; g < g1; ++g) sum += total[g];
    int incl = sum;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int v = __shfl_up_sync(kFull, incl, d);
        if (lane >= d) incl += v;
    }
    if (lane == 31) part[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        int v = lane < static_cast<int>(blockDim.x >> 5) ? part[lane] : 0;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int u = __shfl_up_sync(kFull, v, d);
            if (lane >= d) v += u;
        }
        part[lane] = v;
    }
    __syncthreads();
    int at = incl - sum + (warp > 0 ? part[warp - 1] : 0);
    for (int g = g0; g < g1; ++g) {
        const int c = total[g];
        total[g] = at;
        at += c;
    }
    const int rows = part[31];
    __syncthreads();
    // Each warp's first row of each group.
    for (int g = threadIdx.x; g < groups; g += blockDim.x) {
        int next = total[g] + before[g];
        if (blockIdx.x == 0) offsets[g] = total[g];
        for (int w = 0; w < warps; ++w) {
            const int c = hist[w * groups + g];
            hist[w * groups + g] = next;
            next += c;
        }
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) offsets[groups] = rows;
    __syncthreads();
    int ahead = begin + lane < end ? group_of(ids, begin + lane, groups, nullptr) : -1;
    for (int base = begin; base < end; base += 32) {
        const int i = base + lane, g = ahead;
        ahead = base + 32 < end && i + 32 < end ? group_of(ids, i + 32, groups, nullptr) : -1;
        const unsigned peers = __match_any_sync(kFull, g);
        const int first = g >= 0 ? mine[g] : 0;
        __syncwarp();
        if (g >= 0 && lane == __ffs(peers) - 1) mine[g] = first + __popc(peers);
        __syncwarp();
        const int p = g >= 0 ? first + __popc(peers & ((1u << lane) - 1u)) : -1;
        if (i < end) {
            pos[i] = p;
            if (p >= 0 && order) order[p] = i;
        }
    }
    if (order)
        for (long long p = rows + static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; p < pairs;
             p += static_cast<long long>(gridDim.x) * blockDim.x)
            order[p] = -1;
}

// ------------------------------------------------------------------ rows

struct RouteArgs {
    int tokens, topk, rows;
    const int* __restrict__ pos;
    int nvec;         // vectors of a row
    int chunks;       // blocks along a row
    DeviceErrorRecord* err;
};

// The sorted row of a pair, -1 for none.
__device__ __forceinline__ int row_of(const RouteArgs& a, long long pair) {
    const int p = __ldg(a.pos + pair);
    if (p < -1 || p >= a.rows) record_device_error(a.err, SPMM_ERR_BAD_INDEX, pair);
    return p < 0 || p >= a.rows ? -1 : p;
}

// Threads (tx along a row, ty tokens): tx the power of two that covers a row, at most `most`.
dim3 row_block(int nvec, int most) {
    int tx = 1;
    while (tx < nvec && tx < most) tx *= 2;
    return dim3(tx, std::max(1, 128 / tx));
}

// xs[pos[t, j]] = x[t]: a thread holds U vectors of the token's row and writes them to its topk places.
template <int VB, int U>
__global__ void __launch_bounds__(128) route_gather_kernel(RouteArgs a, const char* __restrict__ x, long long ldx,
                                                           char* __restrict__ xs, long long ldxs) {
    using V = typename VecOf<VB>::type;
    grid_dependency_wait();
    allow_dependent_launch();
    const int chunk = blockIdx.x % a.chunks;
    const long long t = static_cast<long long>(blockIdx.x / a.chunks) * blockDim.y + threadIdx.y;
    if (t >= a.tokens) return;
    const int v0 = chunk * blockDim.x * U + threadIdx.x;
    V v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int c = v0 + u * blockDim.x;
        if (c < a.nvec) v[u] = __ldg(reinterpret_cast<const V*>(x + t * ldx) + c);
    }
    for (int j = 0; j < a.topk; ++j) {
        const int p = row_of(a, t * a.topk + j);
        if (p < 0) continue;
        V* dst = reinterpret_cast<V*>(xs + p * ldxs);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = v0 + u * blockDim.x;
            if (c < a.nvec) dst[c] = v[u];
        }
    }
}

// y[t] = sum_j w[t, j] ys[pos[t, j]]: a thread sums U vectors over the pairs, J x U = 8 loads in flight. FP32 FMA in the
// order of j, as spmm_csr_f32 sums a row's nonzeros; one rounding at the end.
template <int DT, int VB, int J, int U>
__global__ void __launch_bounds__(128) route_combine_kernel(RouteArgs a, const char* __restrict__ ys, long long ldys,
                                                            const float* __restrict__ w, char* __restrict__ y, long long ldy) {
    using R = RowVec<DT, VB>;
    using V = typename R::V;
    grid_dependency_wait();
    allow_dependent_launch();
    const int chunk = blockIdx.x % a.chunks;
    const long long t = static_cast<long long>(blockIdx.x / a.chunks) * blockDim.y + threadIdx.y;
    const int c0 = chunk * blockDim.x * U + threadIdx.x;
    if (t >= a.tokens || c0 >= a.nvec) return;
    float acc[U][R::N] = {};
    for (int j0 = 0; j0 < a.topk; j0 += J) {
        V v[J][U];
        float wj[J];
        int p[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            p[j] = -1;
            if (j0 + j >= a.topk) continue;
            const long long pair = t * a.topk + j0 + j;
            p[j] = row_of(a, pair);
            wj[j] = w ? __ldg(w + pair) : 1.f;
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if (p[j] < 0) continue;
            const V* row = reinterpret_cast<const V*>(ys + p[j] * ldys);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (U == 1 || c0 + u * static_cast<int>(blockDim.x) < a.nvec) v[j][u] = __ldg(row + c0 + u * blockDim.x);
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if (p[j] < 0) continue;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float f[R::N];
                R::unpack(v[j][u], f);
#pragma unroll
                for (int i = 0; i < R::N; ++i) acc[u][i] = fmaf(wj[j], f[i], acc[u][i]);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (U == 1 || c0 + u * static_cast<int>(blockDim.x) < a.nvec) reinterpret_cast<V*>(y + t * ldy)[c0 + u * blockDim.x] = R::pack(acc[u]);
}

// dys[pos[t, j]] = w[t, j] dy[t], dw[t, j] = <dy[t], ys[pos[t, j]]>: one block row (blockDim.x threads) takes a whole
// token, J pairs and U vectors at a time (their loads in flight together), so that a dot product is one tree in a fixed
// order and needs no second pass.
template <int DT, int VB, int J, int U>
__global__ void __launch_bounds__(256)
    route_combine_grad_kernel(RouteArgs a, const char* __restrict__ dy, long long lddy, const char* __restrict__ ys, long long ldys,
                              const float* __restrict__ w, char* __restrict__ dys, long long lddys, float* __restrict__ dw) {
    using R = RowVec<DT, VB>;
    using V = typename R::V;
    __shared__ float sums[8][J];  // [ty * warps along a row][J]; rows of one warp or less use shuffles only
    grid_dependency_wait();
    allow_dependent_launch();
    const long long t = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y;
    const bool real = t < a.tokens;
    const int tx = blockDim.x;
    for (int j0 = 0; j0 < a.topk; j0 += J) {
        int p[J];
        float wj[J], dot[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            p[j] = -1;
            dot[j] = 0.f;
            wj[j] = 1.f;
            if (!real || j0 + j >= a.topk) continue;
            const long long pair = t * a.topk + j0 + j;
            p[j] = row_of(a, pair);
            if (w) wj[j] = __ldg(w + pair);
        }
        if (real) {
            for (int c0 = threadIdx.x; c0 < a.nvec; c0 += tx * U) {
                V dv[U], v[U][J];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int c = c0 + u * tx;
                    if (c >= a.nvec) break;
                    dv[u] = __ldg(reinterpret_cast<const V*>(dy + t * lddy) + c);
                    if (!dw) continue;
#pragma unroll
                    for (int j = 0; j < J; ++j)
                        if (p[j] >= 0) v[u][j] = __ldg(reinterpret_cast<const V*>(ys + p[j] * ldys) + c);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int c = c0 + u * tx;
                    if (c >= a.nvec) break;
                    float g[R::N];
                    R::unpack(dv[u], g);
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        if (p[j] < 0) continue;
                        if (dys) {
                            float o[R::N];
#pragma unroll
                            for (int i = 0; i < R::N; ++i) o[i] = wj[j] * g[i];
                            reinterpret_cast<V*>(dys + p[j] * lddys)[c] = R::pack(o);
                        }
                        if (dw) {
                            float f[R::N];
                            R::unpack(v[u][j], f);
#pragma unroll
                            for (int i = 0; i < R::N; ++i) dot[j] = fmaf(g[i], f[i], dot[j]);
                        }
                    }
                }
            }
        }
        if (!dw) continue;
        for (int d = min(tx, 32) / 2; d > 0; d /= 2) {
#pragma unroll
            for (int j = 0; j < J; ++j) dot[j] += __shfl_xor_sync(kFull, dot[j], d);
        }
        if (tx <= 32) {
            if (real && threadIdx.x == 0) {
#pragma unroll
                for (int j = 0; j < J; ++j)
                    if (j0 + j < a.topk) dw[t * a.topk + j0 + j] = dot[j];
            }
        } else {
            const int warps = tx / 32;  // along a row
            const int slot = threadIdx.y * warps + threadIdx.x / 32;
            __syncthreads();
            if (threadIdx.x % 32 == 0) {
#pragma unroll
                for (int j = 0; j < J; ++j) sums[slot][j] = dot[j];
            }
            __syncthreads();
            if (real && threadIdx.x < J && j0 + static_cast<int>(threadIdx.x) < a.topk) {
                float s = 0.f;
                for (int k = 0; k < warps; ++k) s += sums[threadIdx.y * warps + k][threadIdx.x];
                dw[t * a.topk + j0 + threadIdx.x] = s;
            }
        }
    }
}

// ------------------------------------------------------------------ combine_grad, streamed
//
// For batches that fill the GPU for a while. A persistent block keeps a ring of row pieces in shared memory that bulk
// copies fill: 190 KB of reads are under way on every SM whatever the warps do, where the kernel above loads a token's rows,
// sums and writes before it looks up the next token's. Lane j of the producer warp issues pair j's copies, its position read
// a token ahead; the consumer warps share every stage (a warp that took only some of them could not tell one phase of a
// stage's barrier from the one two later). 16384 tokens x 8
// rows of 4 KB: 248 us by the kernel above (4.6 TB/s), 206 us streamed; the other two operators gain nothing by it
// (gather 198 -> 215 us, combine 212 -> 207 us at 8 KB rows).

constexpr int kRing = 196608;          // bytes of the ring
constexpr int kConsumers = 8;          // warps that take pieces out of it
constexpr int kMaxPairs = 8;           // pairs of a token that a stage holds
constexpr int kPiece = kConsumers * 512;  // bytes of a row that a stage holds at most: 16 to a thread
constexpr int kMaxStages = 32;

struct StreamArgs {
    RouteArgs r;
    const char* __restrict__ dy;
    long long lddy;
    const char* __restrict__ ys;
    long long ldys;
    const float* __restrict__ w;
    char* dys;
    long long lddys;
    float* dw;
    int row_bytes, piece, pieces;      // a row, a stage's piece of it, pieces of a row
    int stage_bytes, stages;
};

// Weights and positions of a stage's pairs, from the producer.
struct PairInfo {
    float w[kMaxPairs];
    int p[kMaxPairs];
};

struct RingState {
    unsigned long long full[kMaxStages], empty[kMaxStages];
    PairInfo pairs[kMaxStages];
    float sums[2][kConsumers][kMaxPairs];  // of alternate tokens
    int abort_flag;
};
constexpr int kRingSmem = kRing + static_cast<int>(sizeof(RingState)) + 128;

template <int DT, int J>  // J pairs at most
__global__ void __launch_bounds__(kConsumers * 32 + 32, 1) route_combine_grad_stream_kernel(StreamArgs a) {
    using R = RowVec<DT, 16>;
    extern __shared__ uint8_t raw[];
    uint8_t* ring = raw + ((128 - (smem_addr(raw) & 127)) & 127);
    RingState* b = reinterpret_cast<RingState*>(ring + kRing);
    volatile int* abort_flag = &b->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < a.stages; ++s) {
            mbar_init(smem_addr(&b->full[s]), 1);
            mbar_init(smem_addr(&b->empty[s]), kConsumers);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    grid_dependency_wait();
    allow_dependent_launch();

    if (warp == kConsumers) {
        // ---------------- producer
        int it = 0, next = -1;
        float next_w = 1.f;
        bool ok = true;
        const auto fetch = [&](long long t) {  // lane j's position and weight
            next = -1;
            if (t >= a.r.tokens || lane >= a.r.topk) return;
            const long long pair = t * a.r.topk + lane;
            next = __ldg(a.r.pos + pair);
            next_w = a.w ? __ldg(a.w + pair) : 1.f;
        };
        fetch(blockIdx.x);
        for (long long t = blockIdx.x; ok && t < a.r.tokens; t += gridDim.x) {
            int p = next;
            const float w = next_w;
            fetch(t + gridDim.x);
            if (p < -1 || p >= a.r.rows) {
                record_device_error(a.r.err, SPMM_ERR_BAD_INDEX, t * a.r.topk + lane);
                p = -1;
            }
            const int rows = 1 + (a.dw ? __popc(__ballot_sync(kFull, p >= 0)) : 0);  // dy's, and the pairs'
            for (int c = 0; c < a.pieces; ++c, ++it) {
                const int s = it % a.stages, at = c * a.piece, bytes = min(a.piece, a.row_bytes - at);
                const uint32_t full = smem_addr(&b->full[s]), dst = smem_addr(ring + s * a.stage_bytes);
                if (lane == 0) ok = mbar_wait(smem_addr(&b->empty[s]), ((it / a.stages) & 1u) ^ 1u, abort_flag);
                ok = __shfl_sync(kFull, ok ? 1 : 0, 0) != 0;
                if (!ok) break;
                if (lane < kMaxPairs) {
                    b->pairs[s].p[lane] = p;
                    b->pairs[s].w[lane] = w;
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive_expect_tx(full, bytes * rows);
                    bulk_load(dst, a.dy + t * a.lddy + at, bytes, full);
                }
                __syncwarp();
                if (a.dw && p >= 0) bulk_load(dst + (lane + 1) * a.piece, a.ys + p * a.ldys + at, bytes, full);
            }
        }
        if (!ok && lane == 0) {
            *abort_flag = 1;
            record_device_error(a.r.err, SPMM_ERR_TIMEOUT, 31);
        }
        // Every copy lands before the block ends.
        if (lane == 0)
            for (int i = max(0, it - a.stages); i < it; ++i) {
                const unsigned long long t0 = global_ns();
                while (!mbar_try_wait(smem_addr(&b->full[i % a.stages]), (i / a.stages) & 1u) && global_ns() - t0 < kWaitNs) {
                }
            }
        return;
    }
    // ---------------- consumers
    int it = 0, buf = 0;
    bool ok = true;
    for (long long t = blockIdx.x; t < a.r.tokens; t += gridDim.x, buf ^= 1) {
        float dot[J];
#pragma unroll
        for (int j = 0; j < J; ++j) dot[j] = 0.f;
        for (int c = 0; c < a.pieces; ++c, ++it) {
            const int s = it % a.stages, v = threadIdx.x * 16;
            // A timeout ends the waits and the work, not the warps' barriers below.
            ok = __all_sync(kFull, ok && mbar_wait(smem_addr(&b->full[s]), (it / a.stages) & 1u, abort_flag));
            if (!ok) continue;
            const uint8_t* stage = ring + s * a.stage_bytes;
            const PairInfo& info = b->pairs[s];
            if (v < min(a.piece, a.row_bytes - c * a.piece)) {
                float g[R::N];
                R::unpack(*reinterpret_cast<const uint4*>(stage + v), g);
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    if (j >= a.r.topk) continue;
                    const int p = info.p[j];
                    if (p < 0) continue;
                    if (a.dys) {
                        const float w = info.w[j];
                        float o[R::N];
#pragma unroll
                        for (int i = 0; i < R::N; ++i) o[i] = w * g[i];
                        *reinterpret_cast<uint4*>(a.dys + p * a.lddys + c * a.piece + v) = R::pack(o);
                    }
                    if (a.dw) {
                        float f[R::N];
                        R::unpack(*reinterpret_cast<const uint4*>(stage + (j + 1) * a.piece + v), f);
#pragma unroll
                        for (int i = 0; i < R::N; ++i) dot[j] = fmaf(g[i], f[i], dot[j]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive_count(smem_addr(&b->empty[s]), 1);
        }
        if (!a.dw) continue;
        // One tree of a fixed shape over the threads.
#pragma unroll
        for (int d = 16; d > 0; d /= 2) {
#pragma unroll
            for (int j = 0; j < J; ++j) dot[j] += __shfl_xor_sync(kFull, dot[j], d);
        }
        if (lane == 0) {
#pragma unroll
            for (int j = 0; j < J; ++j) b->sums[buf][warp][j] = dot[j];
        }
        asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32) : "memory");
        if (ok && static_cast<int>(threadIdx.x) < a.r.topk) {
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < kConsumers; ++k) sum += b->sums[buf][k][threadIdx.x];
            a.dw[t * a.r.topk + threadIdx.x] = sum;
        }
    }
    if (!ok && lane == 0) {
        *abort_flag = 1;
        record_device_error(a.r.err, SPMM_ERR_TIMEOUT, 32);
    }
}

int route_args(const spmm_route_view* r, int32_t H, int32_t dtype) {
    if (!r || r->tokens < 0 || r->topk < 1 || r->rows < 0 || H < 0) return SPMM_ERR_INVALID_ARG;
    if (dtype != SPMM_DTYPE_F16 && dtype != SPMM_DTYPE_BF16 && dtype != SPMM_DTYPE_F32) return SPMM_ERR_INVALID_ARG;
    if (r->tokens > 0 && !r->pos) return SPMM_ERR_INVALID_ARG;
    if (!words_fit(r->pos)) return SPMM_ERR_MISALIGNED;
    // Vectors and bytes of a row are counted in ints.
    if (static_cast<int64_t>(r->tokens) * r->topk > INT32_MAX - 4095 || H > (1 << 24)) return SPMM_ERR_TOO_LARGE;
    return SPMM_OK;
}

// An operand of `rows` rows: there when it has any, stride at least its length, elements on their own boundaries.
int check_rows(const void* p, int64_t ld, int32_t rows, int32_t H, int32_t dtype) {
    if (rows == 0 || H == 0) return SPMM_OK;
    if (!p || ld < H || ld > (INT64_C(1) << 40)) return SPMM_ERR_INVALID_ARG;
    return reinterpret_cast<uintptr_t>(p) % dtype_bytes(dtype) ? SPMM_ERR_MISALIGNED : SPMM_OK;
}

RouteArgs make_args(const spmm_route_view* r, int32_t H, int32_t dtype, int vb, DeviceState* st) {
    RouteArgs a{};
    a.tokens = r->tokens;
    a.topk = r->topk;
    a.rows = r->rows;
    a.pos = r->pos;
    a.nvec = static_cast<int>(static_cast<int64_t>(H) * dtype_bytes(dtype) / vb);
    a.err = st->err;
    return a;
}

// Blocks of a launch over tokens x chunks.
int row_grid(const RouteArgs& a, dim3 block, unsigned* grid) {
    const int64_t n = (static_cast<int64_t>(a.tokens) + block.y - 1) / block.y * a.chunks;
    if (n > INT32_MAX) return SPMM_ERR_TOO_LARGE;
    *grid = static_cast<unsigned>(n);
    return SPMM_OK;
}

template <int VB>
int gather_launch(RouteArgs a, const void* x, int64_t ldx, void* xs, int64_t ldxs, cudaStream_t s) {
    constexpr int U = 4;
    const dim3 block = row_block(a.nvec, 128);
    a.chunks = (a.nvec + block.x * U - 1) / (block.x * U);
    unsigned grid = 0;
    SPMM_TRY(row_grid(a, block, &grid));
    return launch_dependent(route_gather_kernel<VB, U>, dim3(grid), block, 0, s, a, static_cast<const char*>(x),
                            static_cast<long long>(ldx), static_cast<char*>(xs), static_cast<long long>(ldxs));
}

template <int DT, int VB, int J, int U>
int combine_launch_ju(RouteArgs a, const void* ys, int64_t ldys, const float* w, void* y, int64_t ldy, cudaStream_t s) {
    const dim3 block = row_block((a.nvec + U - 1) / U, 128);
    a.chunks = (a.nvec + block.x * U - 1) / (block.x * U);
    unsigned grid = 0;
    SPMM_TRY(row_grid(a, block, &grid));
    return launch_dependent(route_combine_kernel<DT, VB, J, U>, dim3(grid), block, 0, s, a, static_cast<const char*>(ys),
                            static_cast<long long>(ldys), w, static_cast<char*>(y), static_cast<long long>(ldy));
}

template <int DT, int VB>
int combine_launch(const RouteArgs& a, const void* ys, int64_t ldys, const float* w, void* y, int64_t ldy, cudaStream_t s) {
    // Few pairs leave loads for more vectors. Against 8 x 1, BF16: one token of 2 x 1001 1.8 -> 1.6 us, 2048 of 2 x 512 3.3 -> 2.5,
    // 4096 of 4 x 2048 18.6 -> 10.9, 16384 of 1 x 4096 132 -> 54; behind by 0.2 us at most (rows of 128 bytes).
    if (a.topk <= 2) return combine_launch_ju<DT, VB, 2, 4>(a, ys, ldys, w, y, ldy, s);
    if (a.topk <= 4) return combine_launch_ju<DT, VB, 4, 2>(a, ys, ldys, w, y, ldy, s);
    return combine_launch_ju<DT, VB, 8, 1>(a, ys, ldys, w, y, ldy, s);
}

template <int DT, int VB>
int combine_grad_launch(RouteArgs a, const void* dy, int64_t lddy, const void* ys, int64_t ldys, const float* w, void* dys,
                        int64_t lddys, float* dw, cudaStream_t s) {
    const dim3 block = row_block(a.nvec, 256);
    a.chunks = 1;
    unsigned grid = 0;
    SPMM_TRY(row_grid(a, block, &grid));
    // Eight 16-byte loads at a time, twice as many narrow ones (777 tokens x 4 rows of 4100 bytes: 13.1 us with 4 of them).
    constexpr int kWide = VB == 16 ? 1 : 2;
    auto* kernel = a.topk <= 2   ? route_combine_grad_kernel<DT, VB, 2, 4 * kWide>
                   : a.topk <= 4 ? route_combine_grad_kernel<DT, VB, 4, 2 * kWide>
                                 : route_combine_grad_kernel<DT, VB, 8, kWide>;
    return launch_dependent(kernel, dim3(grid), block, 0, s, a, static_cast<const char*>(dy), static_cast<long long>(lddy),
                            static_cast<const char*>(ys), static_cast<long long>(ldys), w, static_cast<char*>(dys),
                            static_cast<long long>(lddys), dw);
}

template <int DT>
int combine_grad_stream_launch(const RouteArgs& r, const void* dy, int64_t lddy, const void* ys, int64_t ldys, const float* w, void* dys,
                               int64_t lddys, float* dw, cudaStream_t s, DeviceState* st) {
    void (*kernel)(StreamArgs) = r.topk <= 2 ? route_combine_grad_stream_kernel<DT, 2>
                                 : r.topk <= 4 ? route_combine_grad_stream_kernel<DT, 4> : route_combine_grad_stream_kernel<DT, kMaxPairs>;
    static std::atomic<unsigned long long> attr_set[3];
    const int slot = r.topk <= 2 ? 0 : (r.topk <= 4 ? 1 : 2);
    const unsigned long long bit = st->device < 64 ? 1ull << st->device : 0ull;
    if (!bit || !(attr_set[slot].load(std::memory_order_acquire) & bit)) {
        SPMM_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingSmem));
        attr_set[slot].fetch_or(bit, std::memory_order_acq_rel);
    }
    StreamArgs a{r, static_cast<const char*>(dy), lddy, static_cast<const char*>(ys), ldys, w, static_cast<char*>(dys), lddys, dw, 0, 0, 0, 0, 0};
    a.row_bytes = r.nvec * 16;
    a.piece = std::min(a.row_bytes, kPiece);
    a.pieces = (a.row_bytes + a.piece - 1) / a.piece;
    a.stage_bytes = a.piece * (r.topk + 1);
    a.stages = std::min(kMaxStages, kRing / a.stage_bytes);
    const unsigned grid = static_cast<unsigned>(std::min(st->sm_count, r.tokens));
    return launch_dependent(kernel, dim3(grid), dim3(kConsumers * 32 + 32), kRingSmem, s, a);
}

#define SPMM_ROUTE_DISPATCH(fn, ...)                                                     \
    switch (dtype * 32 + vb) {                                                           \
        case SPMM_DTYPE_F16 * 32 + 16: return fn<SPMM_DTYPE_F16, 16>(__VA_ARGS__);       \
        case SPMM_DTYPE_F16 * 32 + 4: return fn<SPMM_DTYPE_F16, 4>(__VA_ARGS__);         \
        case SPMM_DTYPE_F16 * 32 + 2: return fn<SPMM_DTYPE_F16, 2>(__VA_ARGS__);         \
        case SPMM_DTYPE_BF16 * 32 + 16: return fn<SPMM_DTYPE_BF16, 16>(__VA_ARGS__);     \
        case SPMM_DTYPE_BF16 * 32 + 4: return fn<SPMM_DTYPE_BF16, 4>(__VA_ARGS__);       \
        case SPMM_DTYPE_BF16 * 32 + 2: return fn<SPMM_DTYPE_BF16, 2>(__VA_ARGS__);       \
        case SPMM_DTYPE_F32 * 32 + 16: return fn<SPMM_DTYPE_F32, 16>(__VA_ARGS__);       \
        default: return fn<SPMM_DTYPE_F32, 4>(__VA_ARGS__);                              \
    }

}  // namespace
}  // namespace spmm_b200

using namespace spmm_b200;

extern "C" {

int spmm_route_workspace_size(int32_t tokens, int32_t topk, int32_t groups, size_t* bytes) {
    if (!bytes || tokens < 0 || topk < 1 || groups < 1) return SPMM_ERR_INVALID_ARG;
    const int64_t pairs = static_cast<int64_t>(tokens) * topk;
    if (groups > SPMM_MAX_GROUPS || pairs > INT32_MAX - 4095) return SPMM_ERR_TOO_LARGE;
    const SortShape h = sort_shape(static_cast<int>(pairs), groups);
    *bytes = h.blocks == 1 ? 0 : sizeof(int) * static_cast<size_t>(h.blocks) * groups;
    return SPMM_OK;
}

int spmm_route_build(const int32_t* ids, int32_t tokens, int32_t topk, int32_t groups, int32_t* offsets, int32_t* order,
                     int32_t* pos, void* ws, size_t ws_bytes, void* stream) {
    size_t need = 0;
    SPMM_TRY(spmm_route_workspace_size(tokens, topk, groups, &need));
    if (!offsets || (tokens > 0 && (!ids || !pos)) || (need > 0 && (!ws || ws_bytes < need))) return SPMM_ERR_INVALID_ARG;
    if (!words_fit(ids, offsets, order, pos, static_cast<const int*>(ws))) return SPMM_ERR_MISALIGNED;
    DeviceState* st = nullptr;
    SPMM_TRY(current_device_state(&st));
    const cudaStream_t s = as_stream(stream);
    const int pairs = tokens * topk;
    const SortShape h = sort_shape(pairs, groups);
    if (h.smem > 48 * 1024) {
        // Once a device, for the largest of all calls: each call its own size would take it from a larger call's launch under
        // way in another thread.
        static std::atomic<unsigned long long> attr_set{0};
        const unsigned long long bit = st->device < 64 ? 1ull << st->device : 0ull;
        if (!bit || !(attr_set.load(std::memory_order_acquire) & bit)) {
            SPMM_CUDA_TRY(cudaFuncSetAttribute(route_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSortSmem));
            attr_set.fetch_or(bit, std::memory_order_acq_rel);
        }
    }
    int* counts = static_cast<int*>(ws);
    // More threads than the warps with histograms only where there are groups for them.
    const int threads = std::max(h.warps * 32, std::min(kMaxSortThreads, (groups + 31) / 32 * 32));
    if (h.blocks > 1)
        SPMM_TRY(launch_dependent(route_count_kernel, dim3(h.blocks), dim3(threads), sizeof(int) * groups, s, ids, pairs, groups,
                                  h.per_block, counts, st->err));
    return launch_dependent(route_place_kernel, dim3(h.blocks), dim3(threads), h.smem, s, ids, pairs, groups, h.warps, h.per_block,
                            counts, offsets, order, pos, st->err);
}

int spmm_route_gather(const spmm_route_view* r, const void* x, int64_t ldx, void* xs, int64_t ldxs, int32_t H, int32_t dtype,
                      void* stream) {
    SPMM_TRY(route_args(r, H, dtype));
    SPMM_TRY(check_rows(x, ldx, r->tokens, H, dtype));
    SPMM_TRY(check_rows(xs, ldxs, r->rows, H, dtype));
    DeviceState* st = nullptr;
    SPMM_TRY(current_device_state(&st));
    if (r->tokens == 0 || r->rows == 0 || H == 0) return SPMM_OK;
    const int e = dtype_bytes(dtype);
    RowAlign al;
    al.add(x, ldx * e);
    al.add(xs, ldxs * e);
    al.add(nullptr, static_cast<int64_t>(H) * e);
    const int vb = al.vector_bytes();
    const RouteArgs a = make_args(r, H, dtype, vb, st);
    if (vb == 16) return gather_launch<16>(a, x, ldx * e, xs, ldxs * e, as_stream(stream));
    if (vb == 4) return gather_launch<4>(a, x, ldx * e, xs, ldxs * e, as_stream(stream));
    return gather_launch<2>(a, x, ldx * e, xs, ldxs * e, as_stream(stream));
}

int spmm_route_combine(const spmm_route_view* r, const void* ys, int64_t ldys, const float* w, void* y, int64_t ldy, int32_t H,
                       int32_t dtype, void* stream) {
    SPMM_TRY(route_args(r, H, dtype));
    SPMM_TRY(check_rows(ys, ldys, r->rows, H, dtype));
    SPMM_TRY(check_rows(y, ldy, r->tokens, H, dtype));
    if (!words_fit(w)) return SPMM_ERR_MISALIGNED;
    DeviceState* st = nullptr;
    SPMM_TRY(current_device_state(&st));
    if (r->tokens == 0 || H == 0) return SPMM_OK;
    const int e = dtype_bytes(dtype);
    RowAlign al;
    if (r->rows > 0) al.add(ys, ldys * e);
    al.add(y, ldy * e);
    al.add(nullptr, static_cast<int64_t>(H) * e);
    const int vb = al.vector_bytes();
    const RouteArgs a = make_args(r, H, dtype, vb, st);
    SPMM_ROUTE_DISPATCH(combine_launch, a, ys, ldys * e, w, y, ldy * e, as_stream(stream))
}

int spmm_route_combine_grad(const spmm_route_view* r, const void* dy, int64_t lddy, const void* ys, int64_t ldys, const float* w,
                            void* dys, int64_t lddys, float* dw, int32_t H, int32_t dtype, void* stream) {
    SPMM_TRY(route_args(r, H, dtype));
    if (!dys && !dw) return SPMM_ERR_INVALID_ARG;
    SPMM_TRY(check_rows(dy, lddy, r->tokens, H, dtype));
    if (dw) SPMM_TRY(check_rows(ys, ldys, r->rows, H, dtype));
    if (dys) SPMM_TRY(check_rows(dys, lddys, r->rows, H, dtype));
    if (!words_fit(w, dw)) return SPMM_ERR_MISALIGNED;
    DeviceState* st = nullptr;
    SPMM_TRY(current_device_state(&st));
    if (r->tokens == 0 || (H == 0 && !dw)) return SPMM_OK;
    const int e = dtype_bytes(dtype);
    RowAlign al;
    if (H > 0) al.add(dy, lddy * e);
    if (H > 0 && r->rows > 0 && dw) al.add(ys, ldys * e);
    if (H > 0 && r->rows > 0 && dys) al.add(dys, lddys * e);
    al.add(nullptr, static_cast<int64_t>(H) * e);
    const int vb = al.vector_bytes();
    const RouteArgs a = make_args(r, H, dtype, vb, st);
    // Streamed: whole vectors, a stage's pairs, rows of a piece at least, and enough bytes that filling the ring pays.
    // (32 MB of 4 KB rows: 15.8 us above, 16.8 us streamed, of 8 KB rows 12.7 and 16.8; 128 MB: 66 and 57, two pairs 93 and 77.)
    constexpr int64_t kLeast = INT64_C(64) << 20;
    if (vb == 16 && r->topk <= kMaxPairs && static_cast<int64_t>(H) * e >= 1024 && static_cast<int64_t>(r->tokens) * r->topk * H * e >= kLeast) {
        if (dtype == SPMM_DTYPE_BF16) return combine_grad_stream_launch<SPMM_DTYPE_BF16>(a, dy, lddy * e, ys, ldys * e, w, dys, lddys * e, dw, as_stream(stream), st);
        if (dtype == SPMM_DTYPE_F16) return combine_grad_stream_launch<SPMM_DTYPE_F16>(a, dy, lddy * e, ys, ldys * e, w, dys, lddys * e, dw, as_stream(stream), st);
        return combine_grad_stream_launch<SPMM_DTYPE_F32>(a, dy, lddy * e, ys, ldys * e, w, dys, lddys * e, dw, as_stream(stream), st);
    }
    SPMM_ROUTE_DISPATCH(combine_grad_launch, a, dy, lddy * e, ys, ldys * e, w, dys, lddys * e, dw, as_stream(stream))
}

}  // extern "C"
