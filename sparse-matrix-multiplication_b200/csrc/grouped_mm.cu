// Products of row groups with their own matrices: y_p = W_g x_p, dx_p = W_g^T dy_p, dW_g = sum_p dy_p x_p^T.
//
// All three are D[m, n] = sum_k A(m, k) B(n, k) for each group, with 16-bit A and B and FP32 sums:
//   forward   m = row of the group, n = feature out, k = feature in     (A = x,    B = w)
//   dx        m = row of the group, n = feature in,  k = feature out    (A = dy,   B = w^T)
//   dw        m = feature out,      n = feature in,  k = row of the group (A = dy^T, B = x^T)

#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "groups.cuh"

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

// ------------------------------------------------------------------ any strides and alignment
//
// 64 x 64 tiles, 16 of k at a time through shared memory as FP32, 4 x 4 results a thread. For operands that TMA
// cannot address (rows off 16-byte boundaries) and for empty sums.

constexpr int kTile = 64;
constexpr int kStep = 16;

template <int FORM, int DT>
__global__ void __launch_bounds__(256) grouped_any_kernel(GroupedArgs a) {
    extern __shared__ int start[];
    __shared__ float As[kStep][kTile + 1], Bs[kStep][kTile + 1];
    grid_dependency_wait();
    allow_dependent_launch();
    const int outs = FORM == kDx ? a.K : (FORM == kForward ? a.N : a.K);  // columns of D
    const int ntiles = (outs + kTile - 1) / kTile;
    long long tiles;
    if constexpr (FORM == kDw) {
        tiles = static_cast<long long>(a.groups) * ((a.N + kTile - 1) / kTile) * ntiles;
    } else {
        build_tile_table(start, a.offsets, a.groups, a.rows, kTile, blockIdx.x == 0 ? a.err : nullptr);
        tiles = static_cast<long long>(start[a.groups]) * ntiles;
    }
    const int tm = (threadIdx.x / 16) * 4, tn = (threadIdx.x % 16) * 4;
    for (long long t = blockIdx.x; t < tiles; t += gridDim.x) {
        const int nt = static_cast<int>(t % ntiles) * kTile;
        int g, m0, ms, ks;  // group, first row of D in the group, rows of D, length of the sum
        GroupRange r;
        if constexpr (FORM == kDw) {
            const int mtiles = (a.N + kTile - 1) / kTile;
            const int mt = static_cast<int>((t / ntiles) % mtiles);
            g = static_cast<int>(t / ntiles / mtiles);
            r = group_range(a.offsets, g, a.rows, nt == 0 && mt == 0 ? a.err : nullptr);
            m0 = mt * kTile;
            ms = a.N;
            ks = r.end - r.begin;
        } else {
            const int mt = static_cast<int>(t / ntiles);
            g = tile_group(start, a.groups, mt);
            r = group_range(a.offsets, g, a.rows, nullptr);
            m0 = (mt - start[g]) * kTile;
            ms = r.end - r.begin;
            ks = FORM == kForward ? a.K : a.N;
        }
        float acc[4][4] = {};
        for (int k0 = 0; k0 < ks; k0 += kStep) {
            __syncthreads();
            for (int i = threadIdx.x; i < kTile * kStep; i += 256) {
                // Consecutive threads take the index that is contiguous in memory.
                const int mk_k = FORM == kDw ? i / kTile : i % kStep, mk_m = FORM == kDw ? i % kTile : i / kStep;
                float v = 0.f;
                if (m0 + mk_m < ms && k0 + mk_k < ks) {
                    const long long row = FORM == kDw ? r.begin + k0 + mk_k : r.begin + m0 + mk_m;
                    const int col = FORM == kDw ? m0 + mk_m : k0 + mk_k;
                    v = half_bits_to_float<DT>(__ldg(a.a + row * a.lda + col));
                }
                As[mk_k][mk_m] = v;
                const int nk_k = FORM == kForward ? i % kStep : i / kTile, nk_n = FORM == kForward ? i / kStep : i % kTile;
                v = 0.f;
                if (nt + nk_n < outs && k0 + nk_k < ks) {
                    long long at;
                    if constexpr (FORM == kForward) at = (static_cast<long long>(g) * a.N + nt + nk_n) * a.K + k0 + nk_k;
                    else if constexpr (FORM == kDx) at = (static_cast<long long>(g) * a.N + k0 + nk_k) * a.K + nt + nk_n;
                    else at = static_cast<long long>(r.begin + k0 + nk_k) * a.ldb + nt + nk_n;
                    v = half_bits_to_float<DT>(__ldg(a.b + at));
                }
                Bs[nk_k][nk_n] = v;
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kStep; ++k) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(As[k][tm + i], Bs[k][tn + j], acc[i][j]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = m0 + tm + i;
            if (m >= ms) continue;
            const long long row = FORM == kDw ? (static_cast<long long>(g) * a.N + m) * a.K : (r.begin + m) * a.ldo;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int n = nt + tn + j;
                if (n >= outs) continue;
                if (a.out_f32) static_cast<float*>(a.out)[row + n] = acc[i][j];
                else static_cast<uint16_t*>(a.out)[row + n] = float_to_half_bits<DT>(acc[i][j]);
            }
        }
    }
}

template <int FORM>
int any_launch(const GroupedArgs& a, int dtype, cudaStream_t s, DeviceState* st) {
    const size_t smem = FORM == kDw ? 0 : sizeof(int) * (static_cast<size_t>(a.groups) + 1);
    const int outs = FORM == kForward ? a.N : a.K;
    const int64_t ntiles = (outs + kTile - 1) / kTile;
    const int64_t mtiles = FORM == kDw ? static_cast<int64_t>(a.groups) * ((a.N + kTile - 1) / kTile)
                                       : a.rows / kTile + std::min<int64_t>(a.groups, a.rows);
    const unsigned grid = static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(mtiles * ntiles, st->sm_count * 6)));
    if (dtype == SPMM_DTYPE_BF16)
        return launch_dependent(grouped_any_kernel<FORM, SPMM_DTYPE_BF16>, dim3(grid), dim3(256), smem, s, a);
    return launch_dependent(grouped_any_kernel<FORM, SPMM_DTYPE_F16>, dim3(grid), dim3(256), smem, s, a);
}

int check_common(const int32_t* offsets, int32_t groups, int32_t rows, int32_t N, int32_t K, int32_t dtype, int32_t out_dtype) {
    if (groups < 1 || rows < 0 || N < 0 || K < 0 || !offsets) return SPMM_ERR_INVALID_ARG;
    if (dtype != SPMM_DTYPE_F16 && dtype != SPMM_DTYPE_BF16) return SPMM_ERR_INVALID_ARG;
    if (out_dtype != dtype && out_dtype != SPMM_DTYPE_F32) return SPMM_ERR_INVALID_ARG;
    // Tile and row numbers are ints; the sizes of any operand that fits a GPU are far below this.
    if (groups > SPMM_MAX_GROUPS || rows > INT32_MAX - 256 || N > (1 << 24) || K > (1 << 24)) return SPMM_ERR_TOO_LARGE;
    return SPMM_OK;
}

int check_operand(const void* p, int64_t ld, int64_t cols, int bytes) {
    if (!p || ld < cols || ld > (INT64_C(1) << 32)) return SPMM_ERR_INVALID_ARG;
    return reinterpret_cast<uintptr_t>(p) % bytes ? SPMM_ERR_MISALIGNED : SPMM_OK;
}

}  // namespace
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
    return any_launch<kForward>(a, dtype, as_stream(stream), st);
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
    return any_launch<kDx>(a, dtype, as_stream(stream), st);
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
    return any_launch<kDw>(a, dtype, as_stream(stream), st);
}

}  // extern "C"
