// Element types and index types of the label operators (splat_labels.h).
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

#include "../../include/splat_labels.h"

namespace splat {

using bf16 = __nv_bfloat16;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ bf16 from_float<bf16>(float v) {
    return __float2bfloat16_rn(v);
}

// Token or label i, -1 when it is outside [0, entries).
__device__ __forceinline__ int64_t index_at(const void* indices, int wide, uint64_t i, uint64_t entries) {
    const int64_t v = wide ? static_cast<const long long*>(indices)[i] : (int64_t)static_cast<const int*>(indices)[i];
    return v >= 0 && (uint64_t)v < entries ? v : -1;
}

// N elements moved together.
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

inline size_t element_size(sp_element e) { return e == SP_F32 ? 4 : 2; }

// The largest power-of-two element count, at most 16 bytes, in which rows of `dim` elements at
// `stride` from `base` can be moved.
inline int pack_width(const void* base, int64_t stride, uint32_t dim, size_t size) {
    int n = (int)(16 / size);
    const uintptr_t at = reinterpret_cast<uintptr_t>(base);
    while (n > 1 && (at % (n * size) != 0 || stride % n != 0 || dim % (uint32_t)n != 0)) n /= 2;
    return n;
}

}  // namespace splat
