// Helpers of the operators over dense rows (route.cu, grouped_mm.cu, lora.cu): vectors of 16-bit or FP32
// elements as floats, launches as programmatic dependents, alignment of row operands.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstdint>

#include "common.cuh"

namespace spmm_b200 {

// Index arrays, weights and scales: 4-byte elements on their own boundaries.
template <typename... P>
inline bool words_fit(const P*... p) {
    return ((reinterpret_cast<uintptr_t>(p) | ...)) % 4 == 0;
}

inline int dtype_bytes(int dtype) { return dtype == SPMM_DTYPE_F32 ? 4 : 2; }

// The widest vector (16, 4 or 2 bytes) that row r + column c of every operand fits: base pointers and row
// strides (in bytes) as given.
struct RowAlign {
    uintptr_t bits = 0;
    void add(const void* p, int64_t row_bytes) { bits |= reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(row_bytes); }
    int vector_bytes() const { return bits % 16 == 0 ? 16 : (bits % 4 == 0 ? 4 : 2); }
};

template <int BYTES>
struct VecOf;
template <>
struct VecOf<16> { using type = uint4; };
template <>
struct VecOf<4> { using type = uint32_t; };
template <>
struct VecOf<2> { using type = uint16_t; };

template <int DT>
__device__ __forceinline__ float half_bits_to_float(uint16_t h) {
    if constexpr (DT == SPMM_DTYPE_BF16) return __uint_as_float(static_cast<uint32_t>(h) << 16);
    else return __half2float(__ushort_as_half(h));
}

template <int DT>
__device__ __forceinline__ uint16_t float_to_half_bits(float f) {
    if constexpr (DT == SPMM_DTYPE_BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(f));
    else return __half_as_ushort(__float2half_rn(f));
}

// Two 16-bit elements of one word, rounded to nearest even.
template <int DT>
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    if constexpr (DT == SPMM_DTYPE_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

// A vector of VB bytes of dtype DT: N elements as floats.
template <int DT, int VB>
struct RowVec {
    using V = typename VecOf<VB>::type;
    static constexpr int kElem = DT == SPMM_DTYPE_F32 ? 4 : 2;
    static constexpr int N = VB / kElem;
    static_assert(N >= 1, "a vector holds at least one element");

    static __device__ __forceinline__ void unpack(const V& v, float (&f)[N]) {
        if constexpr (VB == 2) {
            f[0] = half_bits_to_float<DT>(v);
        } else {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
            for (int i = 0; i < VB / 4; ++i) {
                if constexpr (DT == SPMM_DTYPE_F32) {
                    f[i] = __uint_as_float(w[i]);
                } else {
                    f[2 * i] = half_bits_to_float<DT>(static_cast<uint16_t>(w[i] & 0xffffu));
                    f[2 * i + 1] = half_bits_to_float<DT>(static_cast<uint16_t>(w[i] >> 16));
                }
            }
        }
    }

    static __device__ __forceinline__ V pack(const float (&f)[N]) {
        V v;
        if constexpr (VB == 2) {
            v = float_to_half_bits<DT>(f[0]);
        } else {
            uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int i = 0; i < VB / 4; ++i) {
                if constexpr (DT == SPMM_DTYPE_F32) w[i] = __float_as_uint(f[i]);
                else w[i] = pack_half2<DT>(f[2 * i], f[2 * i + 1]);
            }
        }
        return v;
    }
};

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

// Launch as a programmatic dependent of the previous kernel in the stream: the kernel calls
// grid_dependency_wait() before it touches global memory.
template <typename... P, typename... A>
int launch_dependent(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, A&&... args) {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    SPMM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...));
    return SPMM_OK;
}

}  // namespace spmm_b200
