// Low-rank adapters of many requests at once: out_p = base_p + s_i B_i (A_i x_p), i = the adapter of p's request.
//
// Two launches: shrink u_p = A_i x_p (rank values a row, FP32 in the workspace), expand out_p = base_p + s_i B_i u_p.

#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "groups.cuh"

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
    *bytes = sizeof(float) * static_cast<size_t>(rows) * l->rank;
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
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(rows, st->sm_count * 8)));
    const bool bf16 = l->dtype == SPMM_DTYPE_BF16;
    if (adds)
        SPMM_TRY(launch_dependent(bf16 ? lora_shrink_any_kernel<SPMM_DTYPE_BF16> : lora_shrink_any_kernel<SPMM_DTYPE_F16>, grid, dim3(256), 0,
                                  s, a));
    return launch_dependent(bf16 ? lora_expand_any_kernel<SPMM_DTYPE_BF16> : lora_expand_any_kernel<SPMM_DTYPE_F16>, grid, dim3(256), 0, s,
                            a);
}

}  // extern "C"
