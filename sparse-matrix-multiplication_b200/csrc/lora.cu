// Low-rank adapters of many requests at once: out_p = base_p + s_i B_i (A_i x_p), i = the adapter of p's request.
//
// Two launches: shrink u_p = A_i x_p (rank values a row, FP32 in the workspace), expand out_p = base_p + s_i B_i u_p.
// Three forms of each: a few rows a request (CUDA cores, latency), many (tcgen05, the rows' bytes), any alignment.

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
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

// ------------------------------------------------------------------ any alignment: one block a row

template <int DT>
__global__ void __launch_bounds__(256) lora_shrink_any_kernel(LoraArgs a) {
    grid_dependency_wait();
    allow_dependent_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int p = blockIdx.x; p < a.rows; p += gridDim.x) {
        const int r = request_of(a, p);
        const int i = r < 0 ? -1 : adapter_of(a, r, threadIdx.x == 0 ? a.err : nullptr);
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
    if (blockIdx.x == 0 && a.offsets)
        for (int r = threadIdx.x; r < a.requests; r += 256) group_range(a.offsets, r, a.rows, a.err);  // records bad ones
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

// Dot product of eight 16-bit pairs, added to s.
template <int DT>
__device__ __forceinline__ float dot8(const uint4& a, const uint4& b, float s) {
    float x[8], y[8];
    RowVec<DT, 16>::unpack(a, x);
    RowVec<DT, 16>::unpack(b, y);
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fmaf(x[i], y[i], s);
    return s;
}

template <int DT>
__global__ void __launch_bounds__(256) lora_shrink_rows_kernel(LoraArgs a, int rank_blocks) {
    __shared__ float sums[8][kRanksPerBlock];
    grid_dependency_wait();
    allow_dependent_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int p = blockIdx.x / rank_blocks, q0 = (blockIdx.x - p * rank_blocks) * kRanksPerBlock;
    const int r = request_of(a, p);
    const int i = r < 0 ? -1 : adapter_of(a, r, threadIdx.x == 0 && q0 == 0 ? a.err : nullptr);
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
    if (blockIdx.x == 0 && a.offsets)
        for (int k = threadIdx.x; k < a.requests; k += 256) group_range(a.offsets, k, a.rows, a.err);  // records bad ones
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
//   warps 2..17   D * scale + base (from the stage) -> 32-byte stores; a warp has 32 rows x 32 columns, which is mostly
//                 latency: with 8 warps and twice the columns a tile took 2600 cycles, more than its bytes need (2800
//                 at 1.9 GHz less the start of every unit)
//   warps 18..21  the next tile's u: the parts' sum as two 16-bit terms, hi + lo, K-major under the 128-byte swizzle
// The MMA needs 16-bit u; one term would cost half a step of 16 bits in every product (2^-8 in bf16), two leave 2^-16
// for twice the MMAs, which still run under the copies.

constexpr int kTileM = 128;
constexpr int kEpilogueWarps = 16;
constexpr int kExpandThreads = (2 + kEpilogueWarps + 4) * 32;
constexpr int kSmallRows = 8;  // requests with no more rows load a base box of this many

template <int RB>  // rank in blocks of 64
struct ExpandLayout {
    static constexpr int kTn = RB == 4 ? 64 : 128;
    static constexpr int kU = 2 * RB * 16384;                 // hi blocks, lo blocks: 128 rows x 64 each
    static constexpr int kUs = RB == 1 ? 2 : 1;
    static constexpr int kB = RB * kTn * 128;
    static constexpr int kBase = kTn / 64 * 16384;            // 64-column blocks of 128 rows
    static constexpr int kStage = kB + kBase;
    static constexpr int kStages = RB == 1 ? 3 : (RB == 2 ? 2 : 1);
    static constexpr int kStage0 = kUs * kU;
    static constexpr int kBars = kStage0 + kStages * kStage;  // full[], empty[], u_full[2], u_empty[2], acc_full[2], acc_empty[2], drain
    static constexpr int kInfo = kBars + 8 * (2 * kStages + 9);  // StageInfo[kStages]
    static constexpr int kSlot = kInfo + 32 * kStages;
    static constexpr int kTable = kSlot + 8;
    static constexpr int kFixed = kTable + 1024;
};

struct ExpandArgs {
    LoraArgs l;
    int splits;
    int ntiles, per_unit, chunks;  // column tiles, of which a unit takes per_unit, units along a row
};

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
    int first, last;   // tile of its unit
    int pad;
};

__device__ __forceinline__ Unit unit_of(const ExpandArgs& e, const int* start, int u) {
    const int m = u / e.chunks, c = u - m * e.chunks;
    const int r = tile_group(start, e.l.requests, m);
    const GroupRange g = group_range(e.l.offsets, r, e.l.rows, nullptr);
    Unit x;
    x.row = g.begin + (m - start[r]) * kTileM;
    x.rows = min(kTileM, g.end - x.row);
    x.i = adapter_of(e.l, r, nullptr);
    x.nt0 = c * e.per_unit;
    x.nt1 = min(e.ntiles, x.nt0 + e.per_unit);
    return x;
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
                   acc_full0 = u_empty0 + 16, acc_empty0 = acc_full0 + 16, drain = acc_empty0 + 16;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base + L::kSlot);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    StageInfo* infos = reinterpret_cast<StageInfo*>(base + L::kInfo);
    int* start = reinterpret_cast<int*>(base + L::kTable);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, kEpilogueWarps);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(u_full0 + 8 * s, 4);
            mbar_init(u_empty0 + 8 * s, 1);
            mbar_init(acc_full0 + 8 * s, 1);
            mbar_init(acc_empty0 + 8 * s, kEpilogueWarps);
        }
        mbar_init(drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetch_tensormap(&map_b);
        if (a.base) prefetch_tensormap(&map_base);
    }
    if (warp == 1) tmem_alloc(smem_addr(tmem_slot), 2 * kTn);
    // Only the warps that read the shrink's parts wait for it (every block has them, so none ends before it): the shrink
    // itself waited for everything before it, and writes nothing else.
    allow_dependent_launch();
    build_tile_table(start, a.offsets, a.requests, a.rows, kTileM, blockIdx.x == 0 ? a.err : nullptr);
    const int units = start[a.requests] * e.chunks;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        // ---------------- producer
        if (elect_one()) {
            int it = 0;
            bool ok = true;
            for (int u = blockIdx.x;; u += gridDim.x) {
                Unit x{};
                StageInfo info{};
                const bool end = u >= units;
                if (!end) {
                    x = unit_of(e, start, u);
                    info.rows = x.rows;
                    info.row = x.row;
                    info.i = x.i;
                    info.scale = x.i >= 0 && a.scale ? __ldg(a.scale + x.i) : 1.f;
                }
                const bool small = x.rows <= kSmallRows;
                for (int nt = x.nt0; end ? nt == x.nt0 : nt < x.nt1; ++nt, ++it) {
                    const int s = it % kStages;
                    const uint32_t bar = full0 + 8 * s, sb = sbase + L::kStage0 + s * L::kStage, sbs = sb + L::kB;
                    if (!mbar_wait(empty0 + 8 * s, ((it / kStages) & 1u) ^ 1u, abort_flag)) {
                        ok = false;
                        break;
                    }
                    info.nt = nt;
                    info.first = nt == x.nt0;
                    info.last = nt == x.nt1 - 1;
                    infos[s] = info;
                    const int n0 = nt * kTn, blocks = min(kTn / 64, (a.N - n0 + 63) / 64);
                    if (end) {
                        mbar_arrive_count(bar, 1);
                        continue;
                    }
                    mbar_arrive_expect_tx(bar, (x.i >= 0 ? L::kB : 0) + (a.base ? blocks * (small ? kSmallRows * 128 : 16384) : 0));
                    if (x.i >= 0)
                        for (int k = 0; k < RB; ++k) tma_load_3d(sb + k * kTn * 128, &map_b, bar, 64 * k, n0, x.i);
                    if (a.base)
                        for (int k = 0; k < blocks; ++k)
                            tma_load_2d(sbs + k * 16384, small ? &map_base_small : &map_base, bar, n0 + 64 * k, x.row);
                }
                if (end || !ok) break;
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
            int nu = 0, n = 0;
            bool ok = true;
            for (int it = 0;; ++it) {
                const int s = it % kStages, buf = n & 1, ub = nu % kUs;
                ok = mbar_wait(full0 + 8 * s, (it / kStages) & 1u, abort_flag);
                if (!ok || infos[s].rows == 0) break;
                if (infos[s].i < 0) continue;
                ok = mbar_wait(acc_empty0 + 8 * buf, ((n >> 1) & 1u) ^ 1u, abort_flag) &&
                     (!infos[s].first || mbar_wait(u_full0 + 8 * ub, (nu / kUs) & 1u, abort_flag));
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
                umma_commit(acc_full0 + 8 * buf);
                ++n;
                if (infos[s].last) {
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
        // ---------------- epilogue: four warps a lane quarter, 32 columns each
        const int q = warp & 3, c0 = (warp - 2) / 4 * 32;
        const bool sectors = (reinterpret_cast<uintptr_t>(a.out) | static_cast<uintptr_t>(a.ldout * 2)) % 32 == 0;
        int n = 0;
        bool ok = true;
        for (int it = 0;; ++it) {
            const int s = it % kStages, buf = n & 1;
            ok = __all_sync(0xffffffffu, mbar_wait(full0 + 8 * s, (it / kStages) & 1u, abort_flag));
            if (!ok) break;
            const StageInfo x = infos[s];
            if (x.rows == 0) break;
            const int cols = min(kTn, a.N - x.nt * kTn);
            const bool some = q * 32 < x.rows && c0 < cols, has = x.i >= 0;
            // A block of 64 columns is 16 KB of the stage.
            uint8_t* block = base + L::kStage0 + s * L::kStage + L::kB + c0 / 64 * 16384 + q * 4096;
            uint4 b8[4];
            if (a.base && some) {
#pragma unroll
                for (int c = 0; c < 4; ++c) b8[c] = *swizzled_piece(block, lane, c0 % 64 / 8 + c);
            }
            uint32_t v[32];
            if (has) {
                ok = __all_sync(0xffffffffu, mbar_wait(acc_full0 + 8 * buf, (n >> 1) & 1u, abort_flag));
                if (!ok) break;
                tc_fence_after();
                if (some) tmem_ld32(tmem + buf * kTn + c0 + (static_cast<uint32_t>(q * 32) << 16), v);
                tc_fence_before();
            }
            // The stage and the accumulator are in registers: the next tile's copies and MMAs may begin.
            __syncwarp();
            if (lane == 0) {
                mbar_arrive_count(empty0 + 8 * s, 1);
                if (has) mbar_arrive_count(acc_empty0 + 8 * buf, 1);
            }
            if (has) ++n;
            if (some && q * 32 + lane < x.rows) {
                uint16_t* out = a.out + (x.row + q * 32 + lane) * a.ldout + x.nt * kTn + c0;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t w[8];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float f[8] = {};
                        if (a.base) RowVec<DT, 16>::unpack(b8[2 * h + c], f);
                        if (has) {
#pragma unroll
                            for (int k = 0; k < 8; ++k) f[k] = fmaf(__uint_as_float(v[16 * h + 8 * c + k]), x.scale, f[k]);
                        }
                        const uint4 o = RowVec<DT, 16>::pack(f);
                        w[4 * c] = o.x, w[4 * c + 1] = o.y, w[4 * c + 2] = o.z, w[4 * c + 3] = o.w;
                    }
                    const int col = c0 + 16 * h;
                    if (col + 16 <= cols) store_32(out + 16 * h, w, sectors);
                    else if (col < cols) *reinterpret_cast<uint4*>(out + 16 * h) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            __syncwarp();
        }
        if (!ok && lane == 0) {
            *abort_flag = 1;
            record_device_error(a.err, SPMM_ERR_TIMEOUT, 23);
        }
    } else {
        // ---------------- u: sum of the parts -> hi + lo
        grid_dependency_wait();
        const int pieces = (a.rank + 15) / 16 * 2;  // 8 ranks each; the last may lie past the rank and is zero
        int nu = 0;
        bool ok = true;
        for (int u = blockIdx.x; ok && u < units; u += gridDim.x) {
            const Unit x = unit_of(e, start, u);
            if (x.i < 0) continue;
            const int ub = nu % kUs;
            if (!__all_sync(0xffffffffu, mbar_wait(u_empty0 + 8 * ub, ((nu / kUs) & 1u) ^ 1u, abort_flag))) {
                ok = false;
                break;
            }
            // Pieces of 8 ranks, taken by consecutive threads; kAhead at a time so that their loads overlap.
            uint8_t* hi = base + ub * L::kU;
            const float* parts = a.u + static_cast<long long>(x.row) * a.rank;
            const long long stride = static_cast<long long>(a.rows) * a.rank;
            constexpr int kAhead = 2;
            for (int first = (warp - 2 - kEpilogueWarps) * 32 + lane; first < x.rows * pieces; first += kAhead * 128) {
                float f[kAhead][8] = {};
                int row[kAhead], piece[kAhead];
                bool real[kAhead];
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
                    row[j] = (first + 128 * j) / pieces;
                    piece[j] = first + 128 * j - row[j] * pieces;
                    real[j] = row[j] < x.rows && 8 * piece[j] < a.rank;
                }
                for (int k = 0; k < e.splits; ++k) {
                    float4 v[kAhead][2];
#pragma unroll
                    for (int j = 0; j < kAhead; ++j) {
                        const float4* src = reinterpret_cast<const float4*>(parts + k * stride + static_cast<long long>(row[j]) * a.rank + 8 * piece[j]);
                        if (real[j]) v[j][0] = src[0], v[j][1] = src[1];
                    }
#pragma unroll
                    for (int j = 0; j < kAhead; ++j) {
                        if (!real[j]) continue;
                        f[j][0] += v[j][0].x, f[j][1] += v[j][0].y, f[j][2] += v[j][0].z, f[j][3] += v[j][0].w;
                        f[j][4] += v[j][1].x, f[j][5] += v[j][1].y, f[j][6] += v[j][1].z, f[j][7] += v[j][1].w;
                    }
                }
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
                    if (row[j] >= x.rows) continue;
                    const uint4 top = RowVec<DT, 16>::pack(f[j]);
                    float g[8];
                    RowVec<DT, 16>::unpack(top, g);
#pragma unroll
                    for (int k = 0; k < 8; ++k) g[k] = f[j][k] - g[k];
                    const uint4 rest = RowVec<DT, 16>::pack(g);
                    const int at = row[j] * 128 + piece[j] / 8 * 16384 + (((piece[j] % 8) ^ (row[j] & 7)) << 4);
                    *reinterpret_cast<uint4*>(hi + at) = top;
                    *reinterpret_cast<uint4*>(hi + RB * 16384 + at) = rest;
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive_count(u_full0 + 8 * ub, 1);
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
        tmem_dealloc(tmem, 2 * kTn);
    }
}

template <int DT, int RB>
int expand_launch(const CUtensorMap& mb, const CUtensorMap& ms, const CUtensorMap& small, const ExpandArgs& e, long long units,
                  cudaStream_t s, DeviceState* st) {
    using L = ExpandLayout<RB>;
    static std::atomic<unsigned long long> attr_set{0};
    const unsigned long long bit = st->device < 64 ? 1ull << st->device : 0ull;
    if (!bit || !(attr_set.load(std::memory_order_acquire) & bit)) {
        SPMM_CUDA_TRY(cudaFuncSetAttribute(lora_expand_tc_kernel<DT, RB>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           L::kFixed + 4 * (SPMM_MAX_GROUPS + 1)));
        attr_set.fetch_or(bit, std::memory_order_acq_rel);
    }
    const size_t smem = L::kFixed + 4 * (static_cast<size_t>(e.l.requests) + 1);
    const unsigned grid = static_cast<unsigned>(std::min<long long>(units, st->sm_count));
    return launch_dependent(lora_expand_tc_kernel<DT, RB>, dim3(grid), dim3(kExpandThreads), smem, s, mb, ms, small, e);
}

template <int DT>
int expand(const ExpandArgs& e0, int64_t mtiles, cudaStream_t s, DeviceState* st) {
    ExpandArgs e = e0;
    const LoraArgs& a = e.l;
    const int rb = a.rank <= 64 ? 1 : (a.rank <= 128 ? 2 : 4);
    const int tn = rb == 4 ? 64 : 128;
    e.ntiles = (a.N + tn - 1) / tn;
    // Column tiles of a unit: u is made once for all of them, but units of one-row requests are cheap and the others
    // should spread evenly, so every SM gets six.
    e.per_unit = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(8, mtiles * e.ntiles / (6 * st->sm_count))));
    e.chunks = (e.ntiles + e.per_unit - 1) / e.per_unit;
    const int64_t units = mtiles * e.chunks;
    if (units > INT32_MAX) return SPMM_ERR_TOO_LARGE;
    CUtensorMap mb, ms{}, small{};
    const uint64_t N = a.N, rank = a.rank, rows = a.rows;
    SPMM_TRY(encode_3d(&mb, a.b, {rank, N, static_cast<uint64_t>(a.adapters)}, {rank * 2, N * rank * 2}, {64, static_cast<uint32_t>(tn), 1},
                       CU_TENSOR_MAP_SWIZZLE_128B));
    if (a.base) {
        SPMM_TRY(encode_2d(&ms, a.base, N, rows, a.ldbase * 2, 64, kTileM, CU_TENSOR_MAP_SWIZZLE_128B));
        SPMM_TRY(encode_2d(&small, a.base, N, rows, a.ldbase * 2, 64, kSmallRows, CU_TENSOR_MAP_SWIZZLE_128B));
    }
    if (rb == 1) return expand_launch<DT, 1>(mb, ms, small, e, units, s, st);
    if (rb == 2) return expand_launch<DT, 2>(mb, ms, small, e, units, s, st);
    return expand_launch<DT, 4>(mb, ms, small, e, units, s, st);
}

// ------------------------------------------------------------------ host

// How a call runs, by its sizes alone (the lengths are on the device). `fits`: 16-byte boundaries throughout.
struct Shape {
    bool rows;         // CUDA cores, a few rows a request
    int splits, steps_per_split;
    int64_t mtiles;
};

Shape shape_of(int32_t requests, int32_t rows, int32_t K) {
    Shape h{};
    h.rows = rows <= 4 * static_cast<int64_t>(requests);
    h.mtiles = rows / kTileM + std::min(requests, rows);
    // Ranges of the sum over K until about six tiles an SM (of 148) are there, each at least 8 steps of 64 long.
    const int steps = (K + 63) / 64;
    const int64_t want = h.rows ? 1 : std::max<int64_t>(1, std::min<int64_t>({8, 888 / std::max<int64_t>(1, h.mtiles), steps / 8}));
    h.steps_per_split = static_cast<int>((steps + want - 1) / want);
    h.splits = h.steps_per_split ? (steps + h.steps_per_split - 1) / h.steps_per_split : 1;
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
    *bytes = sizeof(float) * static_cast<size_t>(rows) * l->rank * shape_of(requests, rows, l->K).splits;
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
        if (reinterpret_cast<uintptr_t>(l->scale) % 4) return SPMM_ERR_MISALIGNED;
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
    const Shape h = shape_of(requests, rows, l->K);
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
        PartialProducts p{offsets, adapter, requests, rows, l->adapters, l->rank, l->K, l->dtype, x, ldx, l->a, a.u, h.splits, h.steps_per_split};
        SPMM_TRY(partial_products(p, s, st));
        ExpandArgs e{};
        e.l = a;
        e.splits = h.splits;
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
