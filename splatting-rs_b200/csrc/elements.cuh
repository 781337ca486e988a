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

// N elements moved together, as one word: copying the elements by their own type becomes N loads
// (bf16 rows of 256 columns: a lookup of 500,000 took 67 us instead of 57, their gradient 242
// instead of 125).
template <int BYTES>
struct Word;
template <>
struct Word<2> {
    using type = uint16_t;
};
template <>
struct Word<4> {
    using type = uint32_t;
};
template <>
struct Word<8> {
    using type = uint2;
};
template <>
struct Word<16> {
    using type = uint4;
};

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    using W = typename Word<sizeof(T) * N>::type;
    W word;
    // Element j as f32: bf16 is the upper half of one.
    __device__ __forceinline__ float get(int j) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(reinterpret_cast<const uint32_t*>(&word)[j]);
        else if constexpr (N == 1) return __uint_as_float((uint32_t)word << 16);
        else {
            const uint32_t two = reinterpret_cast<const uint32_t*>(&word)[j / 2];
            return __uint_as_float(j % 2 ? two & 0xffff0000u : two << 16);
        }
    }
    // Rounded to nearest even.
    __device__ __forceinline__ void set(const float (&v)[N]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < N; ++j) reinterpret_cast<uint32_t*>(&word)[j] = __float_as_uint(v[j]);
        } else if constexpr (N == 1) {
            word = __bfloat16_as_ushort(__float2bfloat16_rn(v[0]));
        } else {
#pragma unroll
            for (int j = 0; j < N / 2; ++j) {
                const __nv_bfloat162 two = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                reinterpret_cast<uint32_t*>(&word)[j] = reinterpret_cast<const uint32_t&>(two);
            }
        }
    }
};

template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* from) {
    Pack<T, N> p;
    p.word = *reinterpret_cast<const typename Pack<T, N>::W*>(from);
    return p;
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T* to, const Pack<T, N>& p) {
    *reinterpret_cast<typename Pack<T, N>::W*>(to) = p.word;
}
// A store that leaves the caches to others (evict first).
template <typename T, int N>
__device__ __forceinline__ void store_streaming(T* to, const Pack<T, N>& p) {
    __stcs(reinterpret_cast<typename Pack<T, N>::W*>(to), p.word);
}

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
