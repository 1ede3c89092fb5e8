// Products of row groups with their own matrices: y_p = W_g x_p, dx_p = W_g^T dy_p, dW_g = sum_p dy_p x_p^T.
//
// All three are D[m, n] = sum_k A(m, k) B(n, k) for each group, with 16-bit A and B and FP32 sums:
//   forward   m = row of the group, n = feature out, k = feature in     (A = x,    B = w)
//   dx        m = row of the group, n = feature in,  k = feature out    (A = dy,   B = w^T)
//   dw        m = feature out,      n = feature in,  k = row of the group (A = dy^T, B = x^T)

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cstdint>

#include "groups.cuh"
#include "tcgen05.cuh"

namespace spmm_b200 {
namespace {

enum Form { kForward = 0, kDx = 1, kDw = 2 };

struct GroupedArgs {
    const int* __restrict__ offsets;
    int groups, rows, N, K;
    const uint16_t* __restrict__ a;  // x, dy, dy
    const uint16_t* __restrict__ b;  // w, w, x
    void* out;                       // y, dx, dw
    long long lda, ldb, ldo;         // strides of the row operands (ldb: dw only; ldo: not dw)
    int out_f32;
    DeviceErrorRecord* err;
};

// ------------------------------------------------------------------ tcgen05
//
// A persistent block takes 128 x TN tiles of D, 64 of k a step: one warp issues TMA copies into a ring of stages, one
// issues the MMAs (M = 128, N = TN, FP32 accumulators in TMEM, two of them so that the next tile's MMAs run under this
// one's epilogue), eight move TMEM -> registers -> memory: a lane holds a row's consecutive columns and
// stores whole 32-byte sectors.
// x, dy and w are read as they lie: K-major where k is the contiguous index (both operands of the forward product,
// dx's A), MN-major where it is not (dx's B, both of dw's), so nothing is transposed in memory.
// Ragged groups: a row tile may reach past its group. Rows of D past it are computed and not stored (rows do not mix
// in the MMA); in dw, where rows are summed, the last step issues only the MMAs that hold rows of the group (16 rows
// each) and the up to 15 rows past it are cleared in shared memory first, A's and B's, so NaN there cannot get in.

constexpr int kTileM = 128;
constexpr int kStepK = 64;
constexpr int kBand = 8;          // row tiles that run together down a band (their A and the band's B stay in L2)
// Warp 0 TMA, warp 1 MMA, then the epilogue's (sixteen were 2 to 5 % slower on large products), then, with SINGLES, eight
// for the groups of one row, or with ANY sixteen that load in TMA's place.
constexpr int kEpilogue = 8;
constexpr int kSingleThreads = 256;
constexpr int kLoaders = 16;
constexpr int tc_threads(bool singles, bool any) { return 64 + 32 * kEpilogue + (singles ? kSingleThreads : 0) + (any ? 32 * kLoaders : 0); }
constexpr int kSmallRows = 32;    // groups with no more rows left load a box of this many

constexpr int kTransposed = 32 * 33 * 4;  // ANY: an epilogue warp's 32 x 32 results, to be stored by columns of lanes
constexpr int kStoreBox = 32 * 128;       // dw: an epilogue warp's 32 rows of 128 bytes, for TMA to store

template <int FORM, int TN, bool ANY>
struct TcLayout {
    static constexpr int kA = kTileM * kStepK * 2;
    static constexpr int kB = TN * kStepK * 2;
    static constexpr int kStage = kA + kB;
    static constexpr int kStages = ANY ? 4 : (TN == 256 ? 4 : (TN == 128 ? 6 : 8));  // 192 KB, 128 with ANY
    static constexpr int kOut = kStages * kStage;
    // full[], empty[], acc_full[2], acc_empty[2], drain, tmem slot, abort
    static constexpr int kBars = kOut + (ANY ? kEpilogue * kTransposed : (FORM == kDw ? kEpilogue * kStoreBox : 0));
    static constexpr int kTable = kBars + 8 * (2 * kStages + 5) + 16;
    static constexpr int kFixed = kTable + 1024;     // room to align the base to 1 KB; then int[groups + 1]
};

struct TcArgs {
    const int* __restrict__ offsets;
    int groups, rows;
    int outs;          // columns of D
    int ms;            // dw: rows of D of each group
    int sum;           // not dw: length of the sum
    int mtiles;        // dw: row tiles of a group
    int ntiles;
    int blocks;        // that run at a time
    void* out;
    long long ldo;     // row stride of out
    int out_f32, dtype;
    // SINGLES only: at most this many ranges of the sum over k, each with a result of its own (split_stride elements apart),
    // and the groups' matrices by index (NULL: group g has matrix g).
    int most_splits;
    long long split_stride;
    const int* __restrict__ which;
    int matrices;
    int* singles;      // their number and the groups, for the caller
    // SINGLES and ANY: the operands themselves (A; B, with its stride in dw).
    const uint16_t* __restrict__ x;
    const uint16_t* __restrict__ b;
    long long ldx, ldb;
    DeviceErrorRecord* err;
};

struct Tile {
    int g, m0, n0;     // matrix, first row of D in the group, first column
    int cols;          // columns (a multiple of 8; 0: nothing to do)
    int begin, end;    // the group's rows
    int split;         // forward: the range of the sum,
    int first;         // its first step
    int steps;         // k steps
};

// The tiles in the order that blocks take them: block b those at b, b + blocks, ..., with a queue each the next that none has.
// The last round, if it does not give every block a tile, is cut into narrower ones (TN / parts columns) while that gives no
// block two: a block streams a tile no faster for the others' being idle.
struct Rounds {
    int tiles;         // all of them, full width
    int whole;         // those of the full rounds
    int parts;         // pieces of each of the rest
    int units;         // whole + (tiles - whole) * parts
    int splits;        // SINGLES: ranges of the sum, of split_steps steps; each tile comes once for each
    int split_steps;
};

// Into how many ranges the sum of `steps` steps is cut so that the rounds of tiles take the fewest steps, two more a round for
// its start. The same for every block, and for the reader of the parts.
__device__ __forceinline__ void choose_splits(Rounds& r, int tiles, int steps, int most) {
    r.splits = 1;
    r.split_steps = steps;
    long long best = LLONG_MAX;
    for (int s = 1; s <= most; ++s) {
        const int length = (steps + s - 1) / s, n = (steps + length - 1) / length;
        const long long cost = (static_cast<long long>(tiles) * n + gridDim.x - 1) / gridDim.x * (length + 2);
        if (cost < best) {
            best = cost;
            r.splits = n;
            r.split_steps = length;
        }
    }
}

template <int TN>
__host__ __device__ __forceinline__ Rounds rounds_of(int tiles, int grid) {
    Rounds r{};
    r.tiles = tiles;
    r.whole = tiles / grid * grid;
    const int rest = tiles - r.whole;
    r.parts = 1;
    while (r.parts < TN / 64 && rest * r.parts * 2 <= grid) r.parts *= 2;
    r.units = r.whole + rest * r.parts;
    return r;
}

// dw's tiles differ in length as the groups do, so they are taken one by one as blocks become free, those of the longest groups
// first (the other forms': tc_launch): the grid has a block for every tile, and the blocks that run take over those that have not started. Against equal
// numbers of tiles in the groups' order: 16384 rows over 8 groups that fall like 1 / i, 512 x 512: 33.6 -> 24.5 us; 3001 over 16,
// 520 x 776 in FP32: 19.2 -> 15.7; 8192 over 64 that fall like i^-1/2, 1024 x 1024: 39.7 -> 40.7 (short tiles, more of them at
// once at the stores). The pairs of blocks keep to equal numbers in the groups' order: they read less from L2 when they run in
// step (65536 rows over 128 groups, 1024 x 2048: 324 us, sorted 343; 16384 over 8, 4096 x 2048: 200 us, as they become free 228).
constexpr int kMostSorted = 128;  // groups; with more they come as they lie

// The groups by falling length, equal ones as they lie. Called by every thread of the block; ends with a barrier.
__device__ __forceinline__ void sort_groups(const TcArgs& a, int* length, uint8_t* order) {
    const int g = threadIdx.x;
    if (g < a.groups) {
        const GroupRange r = group_range(a.offsets, g, a.rows, a.err);  // records bad ones
        length[g] = r.end - r.begin;
    }
    __syncthreads();
    if (g < a.groups) {
        int before = 0;
        for (int h = 0; h < a.groups; ++h) before += length[h] > length[g] || (length[h] == length[g] && h < g);
        order[before] = static_cast<uint8_t>(g);
    }
    __syncthreads();
}

// Answers to the block's requests for tiles, four of them: from the producer, which asks, to the other warps.
struct TileQueue {
    static constexpr int kAnswers = 4;
    uint32_t answers, full, empty;  // 16 bytes each, barriers

    // Request n, once answer n - kAnswers has been read by all.
    __device__ __forceinline__ bool ask(int n, volatile int* abort_flag) const {
        const uint32_t s = n % kAnswers;
        if (!mbar_wait(empty + 8 * s, ((n / kAnswers) & 1u) ^ 1u, abort_flag)) return false;
        mbar_arrive_expect_tx(full + 8 * s, 16);
        take_block(answers + 16 * s, full + 8 * s);
        return true;
    }
    // Its answer. The reader then arrives on its `empty`, unless it is the one that asks.
    __device__ __forceinline__ bool answer(int n, volatile int* abort_flag, int* t) const {
        const uint32_t s = n % kAnswers;
        if (!mbar_wait(full + 8 * s, (n / kAnswers) & 1u, abort_flag)) return false;
        *t = taken_block(answers + 16 * s);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the next answer comes by the asynchronous proxy
        return true;
    }
    // By a whole warp.
    __device__ __forceinline__ bool next(int n, volatile int* abort_flag, int* t) const {
        const bool ok = __all_sync(0xffffffffu, answer(n, abort_flag, t));
        if (ok && (threadIdx.x & 31) == 0) mbar_arrive_count(empty + 8 * (n % kAnswers), 1);
        return ok;
    }
};

template <int FORM, int TN, bool SINGLES>
__device__ __forceinline__ Tile tile_of(const TcArgs& a, const int* start, const uint8_t* order, const Rounds& rounds, int t) {
    Tile r;
    int g, local, mtiles, width = TN, part = 0;
    if (t >= rounds.whole && rounds.parts > 1) {
        const int k = t - rounds.whole;
        t = rounds.whole + k / rounds.parts;
        part = k % rounds.parts;
        width = TN / rounds.parts;
    }
    r.split = 0;
    if constexpr (SINGLES) {
        r.split = t % rounds.splits;
        t /= rounds.splits;
    }
    if constexpr (FORM == kDw) {
        const int per = a.mtiles * a.ntiles;
        g = t / per;
        local = t - g * per;
        mtiles = a.mtiles;
        if (order) g = order[g];
    } else {
        g = tile_group(start, a.groups, t / a.ntiles);
        local = t - start[g] * a.ntiles;
        mtiles = start[g + 1] - start[g];
    }
    const int band = local / (kBand * a.ntiles);
    const int high = min(kBand, mtiles - band * kBand);
    local -= band * kBand * a.ntiles;
    r.m0 = (band * kBand + local % high) * kTileM;
    r.n0 = local / high * TN + part * width;
    r.cols = max(0, min(width, a.outs - r.n0));
    const GroupRange range = group_range(a.offsets, g, a.rows, nullptr);
    r.begin = range.begin;
    r.end = range.end;
    r.g = FORM == kForward ? max(0, group_matrix(a.which, g, a.matrices, nullptr)) : g;
    const int sum = FORM == kDw ? r.end - r.begin : a.sum;
    r.steps = (sum + kStepK - 1) / kStepK;
    r.first = 0;
    if constexpr (SINGLES) {
        r.first = r.split * rounds.split_steps;
        r.steps = min(rounds.split_steps, r.steps - r.first);
    }
    return r;
}

// The MMAs of one stage, 16 of k each; the first overwrites the accumulator unless `add`.
template <int FORM>
__device__ __forceinline__ void mma_step(uint32_t acc, uint32_t stage, uint32_t idesc, int slices, bool add) {
    // From one slice to the next: 32 bytes along a K-major row, two 8-row atoms down an MN-major column (units of 16).
    constexpr uint64_t kNextA = FORM == kDw ? 128 : 2, kNextB = FORM == kForward ? 2 : 128;
    const uint64_t da = FORM == kDw ? smem_desc(stage, 8192, 1024, kSwizzle128) : smem_desc(stage, 16, 1024, kSwizzle128);
    const uint32_t sb = stage + kTileM * kStepK * 2;
    const uint64_t db = FORM == kForward ? smem_desc(sb, 16, 1024, kSwizzle128) : smem_desc(sb, 8192, 1024, kSwizzle128);
    if (slices == 4) {
        umma_f16(acc, da, db, idesc, add ? 1u : 0u);
#pragma unroll
        for (int j = 1; j < 4; ++j) umma_f16(acc, da + j * kNextA, db + j * kNextB, idesc, 1u);
    } else {
        for (int j = 0; j < slices; ++j) umma_f16(acc, da + j * kNextA, db + j * kNextB, idesc, add || j > 0 ? 1u : 0u);
    }
}

// Four results (b's rows q .. q + 3) for the row of a group of one, by one warp.
template <int DT>
__device__ __forceinline__ void single_products(const TcArgs& a, int g, int q) {
    const int lane = threadIdx.x & 31;
    const long long row = group_range(a.offsets, g, a.rows, nullptr).begin;
    const int i = group_matrix(a.which, g, a.matrices, nullptr);
    if (i < 0) return;
    const int nvec = a.sum / 8;
    const uint4* x = reinterpret_cast<const uint4*>(a.x + row * a.ldx);
    const uint4* b = reinterpret_cast<const uint4*>(a.b + (static_cast<long long>(i) * a.outs + q) * a.sum);  // outs is a multiple of 8
    float s[4] = {};
#pragma unroll 4
    for (int c = lane; c < nvec; c += 32) {
        const uint4 v = __ldg(x + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] = dot8<DT>(v, __ldg(b + static_cast<long long>(j) * nvec + c), s[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int d = 16; d > 0; d /= 2) s[j] += __shfl_xor_sync(0xffffffffu, s[j], d);
    }
    if (lane == 0) *reinterpret_cast<float4*>(static_cast<float*>(a.out) + row * a.ldo + q) = make_float4(s[0], s[1], s[2], s[3]);
}

// ANY: operands off 16-byte boundaries, which TMA cannot address. Sixteen warps fill the stages instead, in the layout that
// TMA would have written: a lane reads the two aligned 16-byte vectors that hold its eight elements and shifts them into
// place, so the reads are as wide as TMA's; elements past the operand are zero. 5003 rows over 60 groups, N = 999,
// K = 1957: 226 us (a CUDA-core kernel: 1.7 ms); 16384 rows over 8, N = 2047, K = 2049: 200 TFLOP/s, bound by these loads.

// The eight elements from `at` on, of which `count` belong to the row (at most 0: none).
struct Unaligned {
    uint4 lo, hi;
    int shift, count;
};

__device__ __forceinline__ Unaligned load_unaligned(const uint16_t* at, int count) {
    Unaligned v;
    const uintptr_t p = reinterpret_cast<uintptr_t>(at);
    const uint4* base = reinterpret_cast<const uint4*>(p & ~static_cast<uintptr_t>(15));
    v.shift = static_cast<int>(p & 15);
    v.count = min(count, 8);
    v.lo = v.hi = make_uint4(0, 0, 0, 0);
    // Whole vectors: behind an operand that does not end on 16 bytes up to 14 bytes more are read, of the same 16 and so of the
    // same page, and shifted out or cleared.
    if (v.count > 0) v.lo = __ldg(base);
    if (v.shift + 2 * v.count > 16) v.hi = __ldg(base + 1);
    return v;
}

__device__ __forceinline__ uint4 shift_unaligned(const Unaligned& v) {
    const uint32_t w[8] = {v.lo.x, v.lo.y, v.lo.z, v.lo.w, v.hi.x, v.hi.y, v.hi.z, v.hi.w};
    uint32_t t[6], u[5], o[4];
#pragma unroll
    for (int i = 0; i < 6; ++i) t[i] = v.shift & 8 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) u[i] = v.shift & 4 ? t[i + 1] : t[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        o[i] = __funnelshift_r(u[i], u[i + 1], (v.shift & 2) * 8);
        o[i] = 2 * i >= v.count ? 0u : (2 * i + 1 >= v.count ? o[i] & 0xffffu : o[i]);
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}

// Row `line` of a stage's 128-byte rows (A's 128, then B's TN) at step k0: where its 64 elements begin and how many are real.
template <int FORM>
__device__ __forceinline__ const uint16_t* stage_line(const TcArgs& a, const Tile& r, int k0, int line, int* count) {
    const bool in_a = line < kTileM;
    const int l = in_a ? line : line - kTileM, box = l & ~63, k = k0 + (l & 63);  // MN-major: boxes of 64 columns, rows of k
    bool real;
    int col, cols;
    const uint16_t* row;
    if (FORM == kDw) {
        const long long p = r.begin + k;
        real = p < r.end;
        col = (in_a ? r.m0 : r.n0) + box;
        cols = in_a ? a.ms : r.n0 + r.cols;
        row = in_a ? a.x + p * a.ldx : a.b + p * a.ldb;
    } else if (in_a) {
        const long long p = r.begin + r.m0 + l;
        real = p < r.end;
        col = k0;
        cols = a.sum;
        row = a.x + p * a.ldx;
    } else if (FORM == kForward) {
        const int n = r.n0 + l;
        real = l < r.cols;
        col = k0;
        cols = a.sum;
        row = a.b + (static_cast<long long>(r.g) * a.outs + n) * a.sum;
    } else {
        real = k < a.sum;
        col = r.n0 + box;
        cols = r.n0 + r.cols;
        row = a.b + (static_cast<long long>(r.g) * a.sum + k) * a.outs;
    }
    *count = real ? cols - col : 0;
    return row + col;
}

// 32 consecutive results of a row, of which `cols` (a multiple of 8) exist, rounded once where the output has 16 bits.
__device__ __forceinline__ void store_piece(const TcArgs& a, const uint32_t (&v)[32], char* out, int cols, bool sectors) {
    if (a.out_f32) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = v[8 * c + i];
            if (8 * c < cols) store_32(out + 32 * c, w, sectors);
        }
    } else {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float lo = __uint_as_float(v[16 * c + 2 * i]), hi = __uint_as_float(v[16 * c + 2 * i + 1]);
                w[i] = a.dtype == SPMM_DTYPE_BF16 ? pack_half2<SPMM_DTYPE_BF16>(lo, hi) : pack_half2<SPMM_DTYPE_F16>(lo, hi);
            }
            if (16 * c + 16 <= cols) store_32(out + 32 * c, w, sectors);
            else if (16 * c < cols) *reinterpret_cast<uint4*>(out + 32 * c) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// dw's tiles end where the operand does, which TMA knows: a warp's 32 rows in boxes of 128 bytes a row through shared memory,
// for which nothing waits. (Each lane its row's sectors, as above, is one line a lane: 64 groups of 8 rows, 1024 x 1024 in
// FP32, took 95 us where this takes 58.)
__device__ __forceinline__ void store_boxes(const TcArgs& a, uint32_t acc, uint8_t* box, const CUtensorMap* map, bool zero, int part, int cols, int n0,
                                            int row, int g) {
    const int lane = threadIdx.x & 31, per = a.out_f32 ? 32 : 64;  // columns of a box
    for (int c0 = part * per; c0 < cols; c0 += 2 * per) {
        if (lane == 0) bulk_store_read_wait();
        __syncwarp();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (h && a.out_f32) break;
            uint32_t v[32];
            tmem_ld32(acc + c0 + 32 * h, v);
            if (zero) {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = 0u;
            }
            if (a.out_f32) {
#pragma unroll
                for (int c = 0; c < 8; ++c) *swizzled_piece(box, lane, c) = make_uint4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float lo = __uint_as_float(v[8 * c + 2 * i]), hi = __uint_as_float(v[8 * c + 2 * i + 1]);
                        w[i] = a.dtype == SPMM_DTYPE_BF16 ? pack_half2<SPMM_DTYPE_BF16>(lo, hi) : pack_half2<SPMM_DTYPE_F16>(lo, hi);
                    }
                    *swizzled_piece(box, lane, 4 * h + c) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) tma_store_3d(map, smem_addr(box), n0 + c0, row, g);
    }
}

// SINGLES (forward, FP32 out): groups of one row are left to eight warps more.
template <int FORM, int TN, bool SINGLES, bool ANY>
__global__ void __launch_bounds__(tc_threads(SINGLES, ANY), 1)
    grouped_tc_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_a_small,
                      const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_b_wide /* dw: the output */, TcArgs a) {
    using L = TcLayout<FORM, TN, ANY>;
    constexpr int kStages = L::kStages;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_addr(smem_raw);
    uint8_t* base = smem_raw + (((raw + 1023u) & ~1023u) - raw);  // 1 KB: the 128-byte swizzle's atoms
    const uint32_t sbase = smem_addr(base);
    const uint32_t full0 = sbase + L::kBars, empty0 = full0 + 8 * kStages, acc_full0 = empty0 + 8 * kStages, acc_empty0 = acc_full0 + 16,
                   drain = acc_empty0 + 16;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base + L::kBars + 8 * (2 * kStages + 5));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* start = reinterpret_cast<int*>(base + L::kTable);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __shared__ int singles;
    __shared__ uint16_t single[SINGLES ? SPMM_MAX_GROUPS : 1];
    constexpr bool kQueue = !ANY && !SINGLES;
    __shared__ alignas(16) uint4 answers[kQueue ? TileQueue::kAnswers : 1];
    __shared__ unsigned long long answer_bars[kQueue ? 2 * TileQueue::kAnswers : 1];  // full[], empty[]
    __shared__ int lengths[FORM == kDw ? kMostSorted : 1];
    __shared__ uint8_t sorted[FORM == kDw ? kMostSorted : 1];
    const TileQueue queue{smem_addr(answers), smem_addr(answer_bars), smem_addr(answer_bars) + 8 * TileQueue::kAnswers};
    const bool queued = kQueue && gridDim.x > static_cast<unsigned>(a.blocks);  // else a tile a block
    const uint8_t* order = FORM == kDw && queued && a.groups <= kMostSorted ? sorted : nullptr;

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        if constexpr (kQueue) {
            for (int s = 0; s < TileQueue::kAnswers; ++s) {
                mbar_init(queue.full + 8 * s, 1);
                mbar_init(queue.empty + 8 * s, 1 + kEpilogue);
            }
        }
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full0 + 8 * s, ANY ? kLoaders : 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(acc_full0 + 8 * s, 1);
            mbar_init(acc_empty0 + 8 * s, kEpilogue);
        }
        mbar_init(drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if constexpr (!ANY) {
            prefetch_tensormap(&map_a);
            prefetch_tensormap(&map_b);
        }
    }
    if (warp == 1) tmem_alloc(smem_addr(tmem_slot), 2 * TN);
    grid_dependency_wait();
    allow_dependent_launch();
    int tiles;
    if constexpr (FORM == kDw) {
        if (order) sort_groups(a, lengths, sorted);
        else if (queued || blockIdx.x == 0)  // any block may be the one that others take over
            for (int g = threadIdx.x; g < a.groups; g += blockDim.x) group_range(a.offsets, g, a.rows, a.err);  // records bad ones
        tiles = a.groups * a.mtiles * a.ntiles;
    } else {
        DeviceErrorRecord* err = queued || blockIdx.x == 0 ? a.err : nullptr;  // likewise
        if constexpr (SINGLES) {
            build_table(start, a.groups, [&](int g) {
                const GroupRange r = group_range(a.offsets, g, a.rows, err);
                const int rows = r.end - r.begin;
                single[g] = is_single(r) ? 1 : 0;
                if (group_matrix(a.which, g, a.matrices, err) < 0 || is_single(r)) return 0;
                return (rows + kTileM - 1) / kTileM;
            });
            if (warp == 2) {
                // The flags in place to a list in the order of the groups, so that every block has the same.
                int n = 0;
                for (int g0 = 0; g0 < a.groups; g0 += 32) {
                    const unsigned mask = __ballot_sync(0xffffffffu, g0 + lane < a.groups && single[min(g0 + lane, a.groups - 1)]);
                    if ((mask >> lane) & 1u) single[n + __popc(mask & ((1u << lane) - 1u))] = static_cast<uint16_t>(g0 + lane);
                    n += __popc(mask);
                    __syncwarp();
                }
                if (lane == 0) singles = n;
            }
        } else {
            build_tile_table(start, a.offsets, a.groups, a.rows, kTileM, err);
        }
        tiles = min(start[a.groups], most_tiles(a.groups, a.rows, kTileM)) * a.ntiles;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    Rounds rounds = rounds_of<TN>(tiles, a.blocks);
    if constexpr (SINGLES) {
        choose_splits(rounds, tiles, (a.sum + kStepK - 1) / kStepK, a.most_splits);
        rounds.units = rounds.whole = tiles * rounds.splits;  // cut along the sum, not the columns
    }

    // The grid may have more blocks than there are tiles, which only the device knows: queued, they are all taken over.
    const int end = queued ? INT_MAX : rounds.units;
    if (warp == 0) {
        // ---------------- producer
        if (!ANY && elect_one()) {
            int it = 0, s = 0;
            uint32_t phase = 1;
            bool ok = true;
            int asked = 0;
            const auto next = [&](int t, int n) {  // the tile behind the block's n-th, t
                if (!queued) return t + static_cast<int>(gridDim.x);
                if (ok && asked == n) ok = queue.ask(asked, abort_flag), asked += ok;
                if (ok) ok = queue.answer(n, abort_flag, &t);
                return t;
            };
            for (int t = blockIdx.x, n = 0; ok && t < end; t = next(t, n++)) {
                if (t >= rounds.units) continue;
                const Tile r = tile_of<FORM, TN, SINGLES>(a, start, order, rounds, t);
                const bool small = FORM != kDw && r.end - r.begin - r.m0 <= kSmallRows;
                // Boxes of 64 columns that lie wholly past the operand are not loaded; their part of D is not stored.
                if (r.cols == 0) continue;
                const int nb = (r.cols + 63) / 64;
                const bool wide = nb == TN / 64;  // forward: one copy of TN rows of w (four of 64 rows took 5 % longer on large products)
                const int na = min(2, (a.ms - r.m0 + 63) / 64);  // dw
                const uint32_t bytes = (FORM == kDw ? na * 8192 : (small ? kSmallRows * 128 : L::kA)) + nb * 8192;
                for (int ks = 0; ks < r.steps; ++ks, ++it) {
                    const uint32_t bar = full0 + 8 * s, sa = sbase + s * L::kStage, sb = sa + L::kA;
                    if (!mbar_wait(empty0 + 8 * s, phase, abort_flag)) {
                        ok = false;
                        break;
                    }
                    mbar_arrive_expect_tx(bar, bytes);
                    if (++s == kStages) s = 0, phase ^= 1u;
                    const int k0 = (r.first + ks) * kStepK;
                    if constexpr (FORM == kDw) {
                        for (int j = 0; j < na; ++j) tma_load_2d(sa + j * 8192, &map_a, bar, r.m0 + 64 * j, r.begin + k0);
                        for (int j = 0; j < nb; ++j) tma_load_2d(sb + j * 8192, &map_b, bar, r.n0 + 64 * j, r.begin + k0);
                    } else {
                        tma_load_2d(sa, small ? &map_a_small : &map_a, bar, k0, r.begin + r.m0);
                        if (FORM == kForward && wide) {
                            tma_load_3d(sb, &map_b_wide, bar, k0, r.n0, r.g);
                        } else {
                            for (int j = 0; j < nb; ++j)
                                tma_load_3d(sb + j * 8192, &map_b, bar, FORM == kForward ? k0 : r.n0 + 64 * j, FORM == kForward ? r.n0 + 64 * j : k0, r.g);
                        }
                    }
                    // Not before the tile's last loads: a tile taken earlier would wait here while other blocks are free.
                    if (queued && ks == r.steps - 1) ok = queue.ask(asked, abort_flag), asked += ok;
                }
            }
            if (!ok) {
                *abort_flag = 1;
                record_device_error(a.err, SPMM_ERR_TIMEOUT, 11);
            }
            // The block's shared memory outlives every copy into it and every arrival on its barriers.
            if (!ok && asked > 0) {
                const unsigned long long t0 = global_ns();
                while (!mbar_try_wait(queue.full + 8 * ((asked - 1) % TileQueue::kAnswers), ((asked - 1) / TileQueue::kAnswers) & 1u) &&
                       global_ns() - t0 < kWaitNs) {
                }
            }
            for (int i = max(0, it - kStages); i < it; ++i) {
                const unsigned long long t0 = global_ns();
                while (!mbar_try_wait(full0 + 8 * (i % kStages), (i / kStages) & 1u) && global_ns() - t0 < kWaitNs) {
                }
                if (ok) mbar_wait(empty0 + 8 * (i % kStages), (i / kStages) & 1u, abort_flag);
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer: one lane; in dw the whole warp clears the rows past a group's end
        int it = 0, n = 0, taken = 0;
        bool ok = true;
        const auto next = [&](int t) {
            if (!queued) return t + static_cast<int>(gridDim.x);
            ok = ok && queue.next(taken++, abort_flag, &t);
            return t;
        };
        for (int t = blockIdx.x; ok && t < end; t = next(t)) {
            if (t >= rounds.units) continue;
            const Tile r = tile_of<FORM, TN, SINGLES>(a, start, order, rounds, t);
            if (r.cols == 0) continue;
            const int buf = n & 1;
            const uint32_t acc = tmem + buf * TN;
            const uint32_t idesc = instr_desc_f16(a.dtype, (r.cols + 15) / 16 * 16, FORM == kDw, FORM != kForward);
            const int sum = FORM == kDw ? r.end - r.begin : a.sum;
            const int left = min(kStepK, sum - (r.first + r.steps - 1) * kStepK);  // of the last step
            const int clear = FORM == kDw && !ANY && left % 16 != 0;
            if (elect_one()) {
                ok = mbar_wait(acc_empty0 + 8 * buf, ((n >> 1) & 1u) ^ 1u, abort_flag);
                tc_fence_after();
                int s = it % kStages;
                uint32_t phase = (it / kStages) & 1u;
                for (int ks = 0; ok && ks < r.steps - clear; ++ks) {
                    ok = mbar_wait(full0 + 8 * s, phase, abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                    mma_step<FORM>(acc, sbase + s * L::kStage, idesc, ks == r.steps - 1 ? (left + 15) / 16 : 4, ks > 0);
                    umma_commit(empty0 + 8 * s);
                    if (++s == kStages) s = 0, phase ^= 1u;
                }
            }
            ok = __all_sync(0xffffffffu, ok);
            it += r.steps;
            if (FORM == kDw && !ANY && clear && ok) {
                const int s = (it - 1) % kStages, slices = (left + 15) / 16;
                ok = __all_sync(0xffffffffu, mbar_wait(full0 + 8 * s, ((it - 1) / kStages) & 1u, abort_flag));
                if (ok) {
                    const int nb = (r.cols + 63) / 64, na = min(2, (a.ms - r.m0 + 63) / 64);
                    const int pieces = (slices * 16 - left) * 8;  // 16-byte pieces of a box's rows to clear
                    uint8_t* st = base + s * L::kStage;
                    for (int b = 0; b < na + nb; ++b) {
                        uint4* rows = reinterpret_cast<uint4*>(st + (b < na ? b * 8192 : L::kA + (b - na) * 8192) + left * 128);
                        for (int i = lane; i < pieces; i += 32) rows[i] = make_uint4(0, 0, 0, 0);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    tc_fence_after();
                    if (elect_one()) {
                        mma_step<FORM>(acc, sbase + s * L::kStage, idesc, slices, r.steps > 1);
                        umma_commit(empty0 + 8 * s);
                    }
                    __syncwarp();
                }
            }
            if (elect_one()) umma_commit(acc_full0 + 8 * buf);
            __syncwarp();
            ++n;
        }
        if (!ok && lane == 0) {
            *abort_flag = 1;
            record_device_error(a.err, SPMM_ERR_TIMEOUT, 12);
        }
    } else if (SINGLES && warp >= 2 + kEpilogue) {
        // ---------------- groups of one row, while the tiles stream
        const int n = singles, quads = a.outs / 4, warps = kSingleThreads / 32;
        if (blockIdx.x == 0) {
            const int first = threadIdx.x - 32 * (2 + kEpilogue);
            if (first == 0) a.singles[0] = n, a.singles[1] = rounds.splits;
            for (int k = first; k < n; k += kSingleThreads) a.singles[2 + k] = single[k];
        }
        const long long items = static_cast<long long>(n) * quads;
        for (long long k = static_cast<long long>(blockIdx.x) * warps + warp - 2 - kEpilogue; k < items; k += static_cast<long long>(gridDim.x) * warps) {
            const int m = static_cast<int>(k / quads), q = 4 * static_cast<int>(k - static_cast<long long>(m) * quads), g = single[m];
            if (a.dtype == SPMM_DTYPE_BF16) single_products<SPMM_DTYPE_BF16>(a, g, q);
            else single_products<SPMM_DTYPE_F16>(a, g, q);
        }
    } else if (ANY && warp >= 2 + kEpilogue) {
        // ---------------- loads in TMA's place: eight lanes to a row of 128 bytes, 64 rows a pass, two passes' reads together
        const int group = (warp - 2 - kEpilogue) * 4 + lane / 8, piece = lane & 7;
        int s = 0;
        uint32_t phase = 1;
        bool ok = true;
        for (int t = blockIdx.x; ok && t < rounds.units; t += gridDim.x) {
            const Tile r = tile_of<FORM, TN, SINGLES>(a, start, order, rounds, t);
            if (r.cols == 0) continue;
            for (int ks = 0; ks < r.steps; ++ks) {
                ok = __all_sync(0xffffffffu, mbar_wait(empty0 + 8 * s, phase, abort_flag));
                if (!ok) break;
                uint8_t* stage = base + s * L::kStage;
                for (int line = group; line < kTileM + TN; line += 128) {
                    Unaligned v[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        int count;
                        const uint16_t* at = stage_line<FORM>(a, r, ks * kStepK, line + 64 * j, &count);
                        v[j] = load_unaligned(at + 8 * piece, count - 8 * piece);
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) *swizzled_piece(stage, line + 64 * j, piece) = shift_unaligned(v[j]);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive_count(full0 + 8 * s, 1);
                if (++s == kStages) s = 0, phase ^= 1u;
            }
        }
        for (int k = 0; ok && k < kStages; ++k) {  // the MMAs' last arrivals come before the block ends
            ok = __all_sync(0xffffffffu, mbar_wait(empty0 + 8 * s, phase, abort_flag));
            if (++s == kStages) s = 0, phase ^= 1u;
        }
        if (!ok && lane == 0) {
            *abort_flag = 1;
            record_device_error(a.err, SPMM_ERR_TIMEOUT, 14);
        }
    } else {
        // ---------------- epilogue: two warps a lane quarter, alternate 32-column pieces
        const int q = warp & 3, part = (warp - 2) >> 2;  // warps q and q + 4 may access TMEM lanes 32 q ..
        const int size = a.out_f32 ? 4 : 2;
        const bool sectors = (reinterpret_cast<uintptr_t>(a.out) | static_cast<uintptr_t>(a.ldo * size)) % 32 == 0;
        int n = 0, taken = 0;
        bool ok = true;
        const auto next = [&](int t) {
            if (!queued) return t + static_cast<int>(gridDim.x);
            ok = queue.next(taken++, abort_flag, &t);
            return t;
        };
        for (int t = blockIdx.x; ok && t < end; t = next(t)) {
            if (t >= rounds.units) continue;
            const Tile r = tile_of<FORM, TN, SINGLES>(a, start, order, rounds, t);
            if (r.cols == 0) continue;
            const int buf = n & 1;
            if (!__all_sync(0xffffffffu, mbar_wait_sum(acc_full0 + 8 * buf, (n >> 1) & 1u, abort_flag, r.steps))) {
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t acc = tmem + buf * TN + (static_cast<uint32_t>(q * 32) << 16);
            const int row = r.m0 + q * 32 + lane, rows = FORM == kDw ? a.ms : r.end - r.begin;
            const long long at = FORM == kDw ? static_cast<long long>(r.g) * a.ms + row : r.begin + row;
            char* out = static_cast<char*>(a.out) + (at * a.ldo + r.n0 + r.split * a.split_stride) * size;
            const int cols = r.cols;
            if (FORM == kDw && !ANY && r.m0 + q * 32 < rows) {
                store_boxes(a, acc, base + L::kOut + (warp - 2) * kStoreBox, &map_b_wide, r.steps == 0, part, cols, r.n0, r.m0 + q * 32, r.g);
            } else if (r.m0 + q * 32 < rows) {
                for (int c0 = part * 32; c0 < cols; c0 += 8 * kEpilogue) {
                    uint32_t v[32];
                    tmem_ld32(acc + c0, v);
                    if (ANY && r.steps == 0) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = 0u;
                    }
                    if constexpr (ANY) {
                        // Elements one by one, a row's 32 by the warp's lanes.
                        float* tile = reinterpret_cast<float*>(base + L::kOut + (warp - 2) * kTransposed);
#pragma unroll
                        for (int i = 0; i < 32; ++i) tile[lane * 33 + i] = __uint_as_float(v[i]);
                        __syncwarp();
                        char* corner = static_cast<char*>(a.out) + ((at - lane) * a.ldo + r.n0 + c0 + lane) * size;
                        const int high = c0 + lane < cols ? min(32, rows - (row - lane)) : 0;
#pragma unroll 8
                        for (int i = 0; i < high; ++i) {
                            const float f = tile[i * 33 + lane];
                            char* o = corner + i * a.ldo * size;
                            if (a.out_f32) *reinterpret_cast<float*>(o) = f;
                            else if (a.dtype == SPMM_DTYPE_BF16) *reinterpret_cast<uint16_t*>(o) = float_to_half_bits<SPMM_DTYPE_BF16>(f);
                            else *reinterpret_cast<uint16_t*>(o) = float_to_half_bits<SPMM_DTYPE_F16>(f);
                        }
                    } else if (row < rows) {
                        store_piece(a, v, out + c0 * size, cols - c0, sectors);
                    }
                    __syncwarp();
                }
            }
            __syncwarp();
            tc_fence_before();
            if (lane == 0) mbar_arrive_count(acc_empty0 + 8 * buf, 1);
            ++n;
        }
        if (FORM == kDw && !ANY && lane == 0) bulk_store_wait();
        if (!ok && lane == 0) {
            *abort_flag = 1;
            record_device_error(a.err, SPMM_ERR_TIMEOUT, 13);
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        if (*abort_flag) {
            // MMAs still in flight end before their accumulators are given back.
            if (elect_one()) {
                umma_commit(drain);
                const unsigned long long t0 = global_ns();
                while (!mbar_try_wait(drain, 0) && global_ns() - t0 < kWaitNs) {
                }
            }
            __syncwarp();
        }
        tmem_dealloc(tmem, 2 * TN);
    }
}

template <int FORM, int TN, bool SINGLES = false, bool ANY = false>
int tc_launch(const CUtensorMap& ma, const CUtensorMap& small, const CUtensorMap& mb, const CUtensorMap& wide, const TcArgs& a, long long tiles, cudaStream_t s,
              DeviceState* st) {
    using L = TcLayout<FORM, TN, ANY>;
    // The attribute belongs to the device's context: set once a device, for the largest table.
    static std::atomic<unsigned long long> attr_set{0};
    const unsigned long long bit = st->device < 64 ? 1ull << st->device : 0ull;
    if (!bit || !(attr_set.load(std::memory_order_acquire) & bit)) {
        SPMM_CUDA_TRY(cudaFuncSetAttribute(grouped_tc_kernel<FORM, TN, SINGLES, ANY>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           L::kFixed + (FORM == kDw ? 0 : 4 * (SPMM_MAX_GROUPS + 1))));
        attr_set.fetch_or(bit, std::memory_order_acq_rel);
    }
    const size_t smem = L::kFixed + (FORM == kDw ? 0 : 4 * (static_cast<size_t>(a.groups) + 1));
    // With a queue a block for every unit, those that run take the others'. dw's are known here; of the other two there are as
    // many as there can be, and a queue where rows of w lie across 128-byte lines: there blocks stream at unequal rates
    // (20000 rows over 128 groups, 1400 x 2040: 234 -> 209 us; 5003 over 60, 1000 x 1960: 79 -> 72; 6000 over 40, dx of
    // 1288 x 2568: 84 -> 80). Elsewhere they keep step, and the same read of each other's operands in L2 (20000 over 128,
    // 1408 x 2048: 189 us, 193 queued).
    const bool queue = !ANY && !SINGLES && (FORM == kDw || (tiles > 2 * st->sm_count && (FORM == kForward ? a.sum : a.outs) % 64 != 0));
    long long units = std::min<long long>(tiles * (TN / 64), st->sm_count);
    if (queue) units = FORM == kDw ? rounds_of<TN>(static_cast<int>(tiles), st->sm_count).units : std::min<long long>(tiles * (TN / 64), tiles + st->sm_count);
    const unsigned grid = static_cast<unsigned>(SINGLES ? st->sm_count : units);
    TcArgs args = a;
    args.blocks = queue ? st->sm_count : static_cast<int>(grid);
    return launch_dependent(grouped_tc_kernel<FORM, TN, SINGLES, ANY>, dim3(grid), dim3(tc_threads(SINGLES, ANY)), smem, s, ma, small, mb, wide, args);
}

// ------------------------------------------------------------------ tcgen05, pairs of blocks
//
// Long groups: two blocks of a cluster take a 256 x 256 tile with cta_group::2. Each loads its 128 rows of A and half of B's
// 256 columns, and the MMA reads both halves, so a block fills 32 KB a step for the work that takes a block of its own 48. That
// fill bounds the single blocks' kernel (70 bytes a clock and SM from L2 at 80 % of the tensor rate) and costs it clock under
// the power cap: 32768 rows x 4096 x 4096 over 8 groups, 921 -> 756 us back to back. In dw each block clears its own rows past
// a group's end: such a last step completes on a barrier of the block itself, and both blocks tell block 0 when they are done.

constexpr int kPairM = 256, kPairN = 256;

template <int FORM>
struct PairLayout {
    static constexpr int kA = 128 * kStepK * 2;
    static constexpr int kStage = kA + 128 * kStepK * 2;
    static constexpr int kStages = 6;
    static constexpr int kOut = kStages * kStage;
    // full[] (block 0's count), empty[], acc_full[2], acc_empty[2] (block 0's), drain, tail_full, tail_empty,
    // tail_ready (block 0's)
    static constexpr int kBars = kOut + (FORM == kDw ? kEpilogue * kStoreBox : 0);
    static constexpr int kSlot = kBars + 8 * (2 * kStages + 8);
    static constexpr int kTable = kSlot + 16;
    static constexpr int kFixed = kTable + 1024;
};

// Tile t: group, first row and column of D, the group's rows, steps of its sum.
struct PairTile {
    int g, m0, n0, begin, end, steps;
};

template <int FORM>
__device__ __forceinline__ PairTile pair_tile(const TcArgs& a, const int* start, int t) {
    constexpr int kPairBand = kBand / 2;
    PairTile r;
    int local, mtiles;
    if constexpr (FORM == kDw) {
        const int per = a.mtiles * a.ntiles;
        r.g = t / per;
        local = t - r.g * per;
        mtiles = a.mtiles;
    } else {
        r.g = tile_group(start, a.groups, t / a.ntiles);
        local = t - start[r.g] * a.ntiles;
        mtiles = start[r.g + 1] - start[r.g];
    }
    const int band = local / (kPairBand * a.ntiles), high = min(kPairBand, mtiles - band * kPairBand);
    local -= band * kPairBand * a.ntiles;
    r.m0 = (band * kPairBand + local % high) * kPairM;
    r.n0 = local / high * kPairN;
    const GroupRange range = group_range(a.offsets, r.g, a.rows, nullptr);
    r.begin = range.begin;
    r.end = range.end;
    r.steps = ((FORM == kDw ? r.end - r.begin : a.sum) + kStepK - 1) / kStepK;
    return r;
}

template <int FORM>
__device__ __forceinline__ void pair_step(uint32_t acc, uint32_t stage, uint32_t idesc, int slices, bool add) {
    constexpr uint64_t kNextA = FORM == kDw ? 128 : 2, kNextB = FORM == kForward ? 2 : 128;
    const uint64_t da = FORM == kDw ? smem_desc(stage, 8192, 1024, kSwizzle128) : smem_desc(stage, 16, 1024, kSwizzle128);
    const uint32_t sb = stage + PairLayout<FORM>::kA;
    const uint64_t db = FORM == kForward ? smem_desc(sb, 16, 1024, kSwizzle128) : smem_desc(sb, 8192, 1024, kSwizzle128);
    umma_f16_pair(acc, da, db, idesc, add ? 1u : 0u);
#pragma unroll
    for (int j = 1; j < 4; ++j)
        if (j < slices) umma_f16_pair(acc, da + j * kNextA, db + j * kNextB, idesc, 1u);
}

template <int FORM>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(64 + 32 * kEpilogue, 1)
    grouped_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                        const __grid_constant__ CUtensorMap map_out /* dw */, TcArgs a) {
    using L = PairLayout<FORM>;
    constexpr int kStages = L::kStages;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_addr(smem_raw);
    uint8_t* base = smem_raw + (((raw + 1023u) & ~1023u) - raw);  // the same offset in both blocks
    const uint32_t sbase = smem_addr(base);
    const uint32_t full0 = sbase + L::kBars, empty0 = full0 + 8 * kStages, acc_full0 = empty0 + 8 * kStages, acc_empty0 = acc_full0 + 16,
                   drain = acc_empty0 + 16, tail_full = drain + 8, tail_empty = tail_full + 8, tail_ready = tail_empty + 8;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base + L::kSlot);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* start = reinterpret_cast<int*>(base + L::kTable);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = static_cast<int>(cluster_rank()), pair = blockIdx.x / 2, pairs = gridDim.x / 2;

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(acc_full0 + 8 * s, 1);
            mbar_init(acc_empty0 + 8 * s, 2 * kEpilogue);
        }
        mbar_init(drain, 1);
        mbar_init(tail_full, 1);
        mbar_init(tail_empty, 1);
        mbar_init(tail_ready, 2);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetch_tensormap(&map_a);
        prefetch_tensormap(&map_b);
    }
    if (warp == 1) tmem_alloc_pair(smem_addr(tmem_slot), 2 * kPairN);
    grid_dependency_wait();
    allow_dependent_launch();
    int tiles;
    if constexpr (FORM == kDw) {
        if (blockIdx.x == 0)
            for (int g = threadIdx.x; g < a.groups; g += blockDim.x) group_range(a.offsets, g, a.rows, a.err);  // records bad ones
        tiles = a.groups * a.mtiles * a.ntiles;
    } else {
        build_tile_table(start, a.offsets, a.groups, a.rows, kPairM, blockIdx.x == 0 ? a.err : nullptr);
        tiles = min(start[a.groups], most_tiles(a.groups, a.rows, kPairM)) * a.ntiles;
    }
    tc_fence_before();
    cluster_sync();  // the barriers of both blocks are set up, both have their TMEM
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        // ---------------- producer: this block's rows of A and half of B; block 0's barrier counts the bytes of both
        if (elect_one()) {
            int it = 0, s = 0, tails = 0;
            uint32_t phase = 1;
            bool ok = true;
            for (int t = pair; ok && t < tiles; t += pairs) {
                const PairTile r = pair_tile<FORM>(a, start, t);
                const int m = r.m0 + 128 * rank, col = r.n0 + 128 * rank;
                for (int ks = 0; ks < r.steps; ++ks, ++it) {
                    const bool tail = FORM == kDw && ks == r.steps - 1 && (r.end - r.begin) % 16 != 0;
                    const uint32_t sa = sbase + s * L::kStage, sb = sa + L::kA;
                    const uint32_t bar = tail ? cluster_addr(tail_full, rank) : cluster_addr(full0 + 8 * s, 0);
                    ok = mbar_wait(empty0 + 8 * s, phase, abort_flag);
                    // One step that completes on tail_full at a time: its MMAs are done before the next begins.
                    if (tail && tails > 0) ok = ok && mbar_wait(tail_empty, (tails - 1) & 1u, abort_flag);
                    if (!ok) break;
                    if (tail) {
                        mbar_arrive_expect_tx(tail_full, L::kStage);
                        ++tails;
                    }
                    if (rank == 0) mbar_arrive_expect_tx(full0 + 8 * s, tail ? 0 : 2 * L::kStage);
                    if (++s == kStages) s = 0, phase ^= 1u;
                    if constexpr (FORM == kDw) {
                        for (int j = 0; j < 2; ++j) {
                            tma_load_2d_pair(sa + 8192 * j, &map_a, bar, m + 64 * j, r.begin + ks * kStepK);
                            tma_load_2d_pair(sb + 8192 * j, &map_b, bar, col + 64 * j, r.begin + ks * kStepK);
                        }
                        continue;
                    }
                    tma_load_2d_pair(sa, &map_a, bar, ks * kStepK, r.begin + m);
                    if constexpr (FORM == kForward) {
                        tma_load_3d_pair(sb, &map_b, bar, ks * kStepK, col, r.g);
                    } else {
                        tma_load_3d_pair(sb, &map_b, bar, col, ks * kStepK, r.g);
                        tma_load_3d_pair(sb + 8192, &map_b, bar, col + 64, ks * kStepK, r.g);
                    }
                }
            }
            if (!ok) {
                *abort_flag = 1;
                record_device_error(a.err, SPMM_ERR_TIMEOUT, 41);
                // Block 0's barrier, which may be what did not move, is the only one that sees this block's copies land: a
                // while, far longer than a copy takes.
                const unsigned long long t0 = global_ns();
                while (global_ns() - t0 < 10ull * 1000 * 1000) {
                }
            }
            // The stages' last MMAs are done, and so the copies into them.
            for (int i = max(0, it - kStages); ok && i < it; ++i) mbar_wait(empty0 + 8 * (i % kStages), (i / kStages) & 1u, abort_flag);
            if (ok && tails > 0) mbar_wait(tail_empty, (tails - 1) & 1u, abort_flag);
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer, one lane in block 0; in dw the warp of either block clears rows past a group's end
        const uint32_t idesc = instr_desc_f16(a.dtype, kPairN, FORM == kDw, FORM != kForward, kPairM);
        int it = 0, n = 0, tails = 0;
        int since = 0;  // steps since the last that ended in a cleared one
        bool ok = true;
        for (int t = pair; ok && t < tiles; t += pairs, ++n) {
            const PairTile r = pair_tile<FORM>(a, start, t);
            since = min(since, 1 << 30) + min(r.steps, 1 << 30);
            const int buf = n & 1, left = (r.end - r.begin) - (r.steps - 1) * kStepK;  // dw: rows of the last step
            const int clear = FORM == kDw && left % 16 != 0;  // 0 of an empty group too
            const uint32_t acc = tmem + buf * kPairN;
            if (rank == 0 && elect_one()) {
                ok = mbar_wait(acc_empty0 + 8 * buf, ((n >> 1) & 1u) ^ 1u, abort_flag);
                tc_fence_after();
                int s = it % kStages;
                uint32_t phase = (it / kStages) & 1u;
                for (int ks = 0; ok && ks < r.steps - clear; ++ks) {
                    ok = mbar_wait(full0 + 8 * s, phase, abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                    // Forward, dx: past the sum there are zeros; dw: whole slices of 16 rows.
                    pair_step<FORM>(acc, sbase + s * L::kStage, idesc, FORM == kDw && ks == r.steps - 1 ? left / 16 : 4, ks > 0);
                    umma_commit_pair(empty0 + 8 * s);
                    if (++s == kStages) s = 0, phase ^= 1u;
                }
            }
            ok = __all_sync(0xffffffffu, ok);
            it += r.steps;
            if (FORM == kDw && clear && ok) {
                const int s = (it - 1) % kStages, slices = (left + 15) / 16;
                // The other block's warp has nothing to do before this: it waits for all of the tiles since the last.
                ok = __all_sync(0xffffffffu, mbar_wait_sum(tail_full, tails & 1u, abort_flag, since));
                since = 0;
                if (ok) {
                    const int pieces = (slices * 16 - left) * 8;  // 16-byte pieces of a box's rows to clear
                    for (int b = 0; b < 4; ++b) {
                        uint4* rows = reinterpret_cast<uint4*>(base + s * L::kStage + b * 8192 + left * 128);
                        for (int i = lane; i < pieces; i += 32) rows[i] = make_uint4(0, 0, 0, 0);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(cluster_addr(tail_ready, 0));
                    if (rank == 0 && elect_one()) {
                        ok = mbar_wait_cluster(tail_ready, tails & 1u, abort_flag) && mbar_wait(full0 + 8 * s, ((it - 1) / kStages) & 1u, abort_flag);
                        if (ok) {
                            tc_fence_after();
                            pair_step<FORM>(acc, sbase + s * L::kStage, idesc, slices, r.steps > 1);
                            umma_commit_pair(tail_empty);
                            umma_commit_pair(empty0 + 8 * s);
                        }
                    }
                    ok = __all_sync(0xffffffffu, ok);
                }
                ++tails;
            }
            if (rank == 0 && ok && elect_one()) umma_commit_pair(acc_full0 + 8 * buf);
            __syncwarp();
        }
        if (!ok && lane == 0) {
            *abort_flag = 1;
            record_device_error(a.err, SPMM_ERR_TIMEOUT, 42);
        }
    } else {
        // ---------------- epilogue: this block's 128 rows
        const int q = warp & 3, part = (warp - 2) >> 2;
        const int size = a.out_f32 ? 4 : 2;
        const bool sectors = (reinterpret_cast<uintptr_t>(a.out) | static_cast<uintptr_t>(a.ldo * size)) % 32 == 0;
        int n = 0;
        bool ok = true;
        for (int t = pair; t < tiles; t += pairs, ++n) {
            const PairTile r = pair_tile<FORM>(a, start, t);
            const int buf = n & 1;
            if (!__all_sync(0xffffffffu, mbar_wait_sum(acc_full0 + 8 * buf, (n >> 1) & 1u, abort_flag, r.steps))) {
                ok = false;
                break;
            }
            tc_fence_after();
            const int first = r.m0 + 128 * rank + q * 32, rows = FORM == kDw ? a.ms : r.end - r.begin, cols = min(kPairN, a.outs - r.n0);
            if constexpr (FORM == kDw) {
                if (first < rows)
                    store_boxes(a, tmem + buf * kPairN + (static_cast<uint32_t>(q * 32) << 16), base + L::kOut + (warp - 2) * kStoreBox, &map_out, r.steps == 0,
                                part, cols, r.n0, first, r.g);
                __syncwarp();
                tc_fence_before();
                if (lane == 0) mbar_arrive_cluster(cluster_addr(acc_empty0 + 8 * buf, 0));
                continue;
            }
            char* out = static_cast<char*>(a.out) + (static_cast<long long>(r.begin + first + lane) * a.ldo + r.n0) * size;
            for (int c0 = part * 32; first < rows && c0 < cols; c0 += 8 * kEpilogue) {
                uint32_t v[32];
                tmem_ld32(tmem + buf * kPairN + c0 + (static_cast<uint32_t>(q * 32) << 16), v);
                if (first + lane < rows) store_piece(a, v, out + c0 * size, cols - c0, sectors);
                __syncwarp();
            }
            __syncwarp();
            tc_fence_before();
            if (lane == 0) mbar_arrive_cluster(cluster_addr(acc_empty0 + 8 * buf, 0));
        }
        if (FORM == kDw && lane == 0) bulk_store_wait();
        if (!ok && lane == 0) {
            *abort_flag = 1;
            record_device_error(a.err, SPMM_ERR_TIMEOUT, 43);
        }
    }

    tc_fence_before();
    __syncwarp();
    cluster_sync();  // neither block's shared memory or TMEM goes while the other may use it
    if (warp == 1) {
        tc_fence_after();
        if (rank == 0 && *abort_flag) {
            // MMAs still in flight end before their accumulators are given back.
            if (elect_one()) {
                umma_commit_pair(drain);
                const unsigned long long t0 = global_ns();
                while (!mbar_try_wait(drain, 0) && global_ns() - t0 < kWaitNs) {
                }
            }
            __syncwarp();
        }
        tmem_dealloc_pair(tmem, 2 * kPairN);
    }
    cluster_sync();
}

template <int FORM>
int pair_launch(const GroupedArgs& g, TcArgs a, cudaStream_t s, DeviceState* st) {
    static std::atomic<unsigned long long> attr_set{0};
    const unsigned long long bit = st->device < 64 ? 1ull << st->device : 0ull;
    if (!bit || !(attr_set.load(std::memory_order_acquire) & bit)) {
        SPMM_CUDA_TRY(cudaFuncSetAttribute(grouped_pair_kernel<FORM>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           PairLayout<FORM>::kFixed + (FORM == kDw ? 0 : 4 * (SPMM_MAX_GROUPS + 1))));
        attr_set.fetch_or(bit, std::memory_order_acq_rel);
    }
    a.ntiles = (a.outs + kPairN - 1) / kPairN;
    a.mtiles = (g.N + kPairM - 1) / kPairM;
    CUtensorMap ma, mb, out{};
    const uint64_t rows = g.rows, N = g.N, K = g.K, groups = g.groups, size = g.out_f32 ? 4 : 2;
    SPMM_TRY(encode_2d(&ma, g.a, FORM == kForward ? K : N, rows, g.lda * 2, 64, FORM == kDw ? 64 : 128, CU_TENSOR_MAP_SWIZZLE_128B));
    if constexpr (FORM == kDw) {
        SPMM_TRY(encode_2d(&mb, g.b, K, rows, g.ldb * 2, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B));
        SPMM_TRY(encode_3d(&out, g.out, {K, N, groups}, {K * size, N * K * size}, {static_cast<uint32_t>(128 / size), 32, 1},
                           CU_TENSOR_MAP_SWIZZLE_128B, g.out_f32));
    } else {
        SPMM_TRY(encode_3d(&mb, g.b, {K, N, groups}, {K * 2, N * K * 2}, {64, FORM == kForward ? 128u : 64u, 1}, CU_TENSOR_MAP_SWIZZLE_128B));
    }
    const size_t smem = PairLayout<FORM>::kFixed + (FORM == kDw ? 0 : 4 * (static_cast<size_t>(a.groups) + 1));
    return launch_dependent(grouped_pair_kernel<FORM>, dim3(static_cast<unsigned>(st->sm_count / 2 * 2)), dim3(64 + 32 * kEpilogue), smem, s, ma, mb, out, a);
}

bool fits16(const void* p, int64_t ld, int size) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * size % 16 == 0; }

// Whether TMA and stores of 16 bytes can address the operands.
template <int FORM>
bool tma_fits(const GroupedArgs& a) {
    if (a.N % 8 || a.K % 8 || a.rows == 0 || a.N == 0 || a.K == 0) return false;
    const int size = a.out_f32 ? 4 : 2;
    if (!fits16(a.a, a.lda, 2) || !fits16(a.b, FORM == kDw ? a.ldb : 8, 2)) return false;
    return fits16(a.out, FORM == kDw ? 8 : a.ldo, size);
}

template <int FORM>
int grouped_launch(const GroupedArgs& a, int dtype, cudaStream_t s, DeviceState* st) {
    if (st->cc_major != 10) return SPMM_ERR_UNSUPPORTED;
    const bool any = !tma_fits<FORM>(a);  // also empty sums, for which there is nothing to map
    TcArgs t{};
    t.offsets = a.offsets;
    t.groups = a.groups;
    t.rows = a.rows;
    t.outs = FORM == kForward ? a.N : a.K;
    t.ms = a.N;
    t.sum = FORM == kForward ? a.K : a.N;
    t.mtiles = (a.N + kTileM - 1) / kTileM;
    t.out = a.out;
    t.ldo = FORM == kDw ? a.K : a.ldo;
    t.out_f32 = a.out_f32;
    t.dtype = dtype;
    t.x = a.a;
    t.b = a.b;
    t.ldx = a.lda;
    t.ldb = a.ldb;
    t.err = a.err;
    // Row tiles: exact for dw, else as many as the groups can have (how many they do have is on the device).
    const int64_t mtiles = FORM == kDw ? static_cast<int64_t>(a.groups) * t.mtiles : most_tiles(a.groups, a.rows, kTileM);
    if (mtiles * ((t.outs + 63) / 64) > INT32_MAX) return SPMM_ERR_TOO_LARGE;  // of the narrowest kind
    // Pairs of blocks where every pair has about four tiles (with three their coarser rounds cost what they gain: 0.92 to 1.13
    // of the single blocks' rate) and the groups are long: a row tile of 256 wastes 128 rows of a group on average, in dw a tile
    // has that much more to store. Measured at 16384 rows, 2048 x 2048, pairs against single blocks: 192 rows a group 1.07
    // (forward), 1.05 (dx), 0.76 (dw); 384: 1.10, 1.13, 1.06; 1024: 1.20, 1.16, 1.12.
    const int64_t pair_rows = FORM == kDw ? static_cast<int64_t>(a.groups) * ((a.N + kPairM - 1) / kPairM) : a.rows / kPairM;
    const int64_t pair_tiles = pair_rows * ((t.outs + kPairN - 1) / kPairN);
    if (!any && t.outs >= kPairN && (FORM != kDw || a.N >= kPairM) && a.rows / a.groups >= (FORM == kDw ? 384 : 192) && pair_tiles >= 2 * st->sm_count)
        return pair_launch<FORM>(a, t, s, st);
    // The widest tile that still gives every SM one: a wide tile reads A less often, narrow ones spread few rows.
    int tn = 256;
    if (any) tn = 128;
    while (!any && tn > 64 && (mtiles * ((t.outs + tn - 1) / tn) < st->sm_count || t.outs <= tn / 2)) tn /= 2;
    t.ntiles = (t.outs + tn - 1) / tn;
    const int64_t tiles = mtiles * t.ntiles;

    CUtensorMap ma{}, small{}, mb{}, wide{};
    if (any) return tc_launch<FORM, 128, false, true>(ma, small, mb, wide, t, tiles, s, st);
    const uint64_t rows = a.rows, N = a.N, K = a.K;
    const uint64_t inner = FORM == kForward ? K : N;  // columns of A's operand
    SPMM_TRY(encode_2d(&ma, a.a, inner, rows, a.lda * 2, 64, FORM == kDw ? 64 : kTileM, CU_TENSOR_MAP_SWIZZLE_128B));
    SPMM_TRY(encode_2d(&small, a.a, inner, rows, a.lda * 2, 64, kSmallRows, CU_TENSOR_MAP_SWIZZLE_128B));
    if constexpr (FORM == kDw) {
        SPMM_TRY(encode_2d(&mb, a.b, K, rows, a.ldb * 2, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B));
        const uint64_t size = a.out_f32 ? 4 : 2;  // the output's map
        SPMM_TRY(encode_3d(&wide, a.out, {K, N, static_cast<uint64_t>(a.groups)}, {K * size, N * K * size}, {static_cast<uint32_t>(128 / size), 32, 1},
                           CU_TENSOR_MAP_SWIZZLE_128B, a.out_f32));
    } else {
        const auto encode_w = [&](CUtensorMap* map, int box_rows) {
            return encode_3d(map, a.b, {K, N, static_cast<uint64_t>(a.groups)}, {K * 2, N * K * 2}, {64, static_cast<uint32_t>(box_rows), 1},
                             CU_TENSOR_MAP_SWIZZLE_128B);
        };
        SPMM_TRY(encode_w(&mb, 64));
        if (FORM == kForward) SPMM_TRY(encode_w(&wide, tn));
    }
    if (tn == 256) return tc_launch<FORM, 256>(ma, small, mb, wide, t, tiles, s, st);
    if (tn == 128) return tc_launch<FORM, 128>(ma, small, mb, wide, t, tiles, s, st);
    return tc_launch<FORM, 64>(ma, small, mb, wide, t, tiles, s, st);
}

int check_common(const int32_t* offsets, int32_t groups, int32_t rows, int32_t N, int32_t K, int32_t dtype, int32_t out_dtype) {
    if (groups < 1 || rows < 0 || N < 0 || K < 0 || !offsets) return SPMM_ERR_INVALID_ARG;
    if (dtype != SPMM_DTYPE_F16 && dtype != SPMM_DTYPE_BF16) return SPMM_ERR_INVALID_ARG;
    if (out_dtype != dtype && out_dtype != SPMM_DTYPE_F32) return SPMM_ERR_INVALID_ARG;
    if (!words_fit(offsets)) return SPMM_ERR_MISALIGNED;
    // Tile and row numbers are ints; the sizes of any operand that fits a GPU are far below this.
    if (groups > SPMM_MAX_GROUPS || rows > INT32_MAX - 256 || N > (1 << 24) || K > (1 << 24)) return SPMM_ERR_TOO_LARGE;
    return SPMM_OK;
}

int check_operand(const void* p, int64_t ld, int64_t cols, int bytes) {
    if (!p || ld < cols || ld > (INT64_C(1) << 32)) return SPMM_ERR_INVALID_ARG;
    return reinterpret_cast<uintptr_t>(p) % bytes ? SPMM_ERR_MISALIGNED : SPMM_OK;
}

}  // namespace

int partial_products(const PartialProducts& p, cudaStream_t s, DeviceState* st) {
    TcArgs t{};
    t.offsets = p.offsets;
    t.groups = p.groups;
    t.rows = p.rows;
    t.outs = p.rank;
    t.sum = p.K;
    t.ntiles = 1;
    t.out = p.parts;
    t.ldo = p.rank;
    t.out_f32 = 1;
    t.dtype = p.dtype;
    t.most_splits = p.most_splits;
    t.split_stride = static_cast<long long>(p.rows) * p.rank;
    t.which = p.which;
    t.matrices = p.matrices;
    t.x = static_cast<const uint16_t*>(p.x);
    t.b = static_cast<const uint16_t*>(p.a);
    t.ldx = p.ldx;
    t.singles = p.singles;
    t.err = st->err;
    const int tn = p.rank <= 64 ? 64 : (p.rank <= 128 ? 128 : 256);
    const int64_t tiles = static_cast<int64_t>(most_tiles(p.groups, p.rows, kTileM)) * p.most_splits;
    if (tiles > INT32_MAX) return SPMM_ERR_TOO_LARGE;
    CUtensorMap ma, small, mb, wide;
    const uint64_t rows = p.rows, K = p.K, rank = p.rank;
    SPMM_TRY(encode_2d(&ma, p.x, K, rows, p.ldx * 2, 64, kTileM, CU_TENSOR_MAP_SWIZZLE_128B));
    SPMM_TRY(encode_2d(&small, p.x, K, rows, p.ldx * 2, 64, kSmallRows, CU_TENSOR_MAP_SWIZZLE_128B));
    SPMM_TRY(encode_3d(&mb, p.a, {K, rank, static_cast<uint64_t>(p.matrices)}, {K * 2, rank * K * 2}, {64, 64, 1}, CU_TENSOR_MAP_SWIZZLE_128B));
    SPMM_TRY(encode_3d(&wide, p.a, {K, rank, static_cast<uint64_t>(p.matrices)}, {K * 2, rank * K * 2}, {64, static_cast<uint32_t>(tn), 1},
                       CU_TENSOR_MAP_SWIZZLE_128B));
    if (tn == 256) return tc_launch<kForward, 256, true>(ma, small, mb, wide, t, tiles, s, st);
    if (tn == 128) return tc_launch<kForward, 128, true>(ma, small, mb, wide, t, tiles, s, st);
    return tc_launch<kForward, 64, true>(ma, small, mb, wide, t, tiles, s, st);
}

}  // namespace spmm_b200

using namespace spmm_b200;

extern "C" {

int spmm_grouped_mm(const int32_t* offsets, int32_t groups, int32_t rows, const void* x, int64_t ldx, const void* w, void* y,
                    int64_t ldy, int32_t N, int32_t K, int32_t dtype, int32_t out_dtype, void* stream) {
    SPMM_TRY(check_common(offsets, groups, rows, N, K, dtype, out_dtype));
    if (rows > 0 && N > 0) {
        if (K > 0) {
            SPMM_TRY(check_operand(x, ldx, K, 2));
            SPMM_TRY(check_operand(w, K, K, 2));
        }
        SPMM_TRY(check_operand(y, ldy, N, dtype_bytes(out_dtype)));
    }
    DeviceState* st = nullptr;
    SPMM_TRY(current_device_state(&st));
    if (rows == 0 || N == 0) return SPMM_OK;
    GroupedArgs a{};
    a.offsets = offsets;
    a.groups = groups;
    a.rows = rows;
    a.N = N;
    a.K = K;
    a.a = static_cast<const uint16_t*>(x);
    a.b = static_cast<const uint16_t*>(w);
    a.out = y;
    a.lda = ldx;
    a.ldo = ldy;
    a.out_f32 = out_dtype == SPMM_DTYPE_F32;
    a.err = st->err;
    return grouped_launch<kForward>(a, dtype, as_stream(stream), st);
}

int spmm_grouped_mm_dx(const int32_t* offsets, int32_t groups, int32_t rows, const void* dy, int64_t lddy, const void* w, void* dx,
                       int64_t lddx, int32_t N, int32_t K, int32_t dtype, int32_t out_dtype, void* stream) {
    SPMM_TRY(check_common(offsets, groups, rows, N, K, dtype, out_dtype));
    if (rows > 0 && K > 0) {
        if (N > 0) {
            SPMM_TRY(check_operand(dy, lddy, N, 2));
            SPMM_TRY(check_operand(w, K, K, 2));
        }
        SPMM_TRY(check_operand(dx, lddx, K, dtype_bytes(out_dtype)));
    }
    DeviceState* st = nullptr;
    SPMM_TRY(current_device_state(&st));
    if (rows == 0 || K == 0) return SPMM_OK;
    GroupedArgs a{};
    a.offsets = offsets;
    a.groups = groups;
    a.rows = rows;
    a.N = N;
    a.K = K;
    a.a = static_cast<const uint16_t*>(dy);
    a.b = static_cast<const uint16_t*>(w);
    a.out = dx;
    a.lda = lddy;
    a.ldo = lddx;
    a.out_f32 = out_dtype == SPMM_DTYPE_F32;
    a.err = st->err;
    return grouped_launch<kDx>(a, dtype, as_stream(stream), st);
}

int spmm_grouped_mm_dw(const int32_t* offsets, int32_t groups, int32_t rows, const void* dy, int64_t lddy, const void* x, int64_t ldx,
                       void* dw, int32_t N, int32_t K, int32_t dtype, int32_t out_dtype, void* stream) {
    SPMM_TRY(check_common(offsets, groups, rows, N, K, dtype, out_dtype));
    if (N > 0 && K > 0) {
        if (rows > 0) {
            SPMM_TRY(check_operand(dy, lddy, N, 2));
            SPMM_TRY(check_operand(x, ldx, K, 2));
        }
        SPMM_TRY(check_operand(dw, K, K, dtype_bytes(out_dtype)));
    }
    DeviceState* st = nullptr;
    SPMM_TRY(current_device_state(&st));
    if (N == 0 || K == 0) return SPMM_OK;
    GroupedArgs a{};
    a.offsets = offsets;
    a.groups = groups;
    a.rows = rows;
    a.N = N;
    a.K = K;
    a.a = static_cast<const uint16_t*>(dy);
    a.b = static_cast<const uint16_t*>(x);
    a.out = dw;
    a.lda = lddy;
    a.ldb = ldx;
    a.out_f32 = out_dtype == SPMM_DTYPE_F32;
    a.err = st->err;
    return grouped_launch<kDw>(a, dtype, as_stream(stream), st);
}

}  // extern "C"
