// What the operators of a training step share (ds_embed.hip, ds_clip.hip, ds_vocab*.hip): element types, and vectors of
// them on their way to and from 32-bit floats.
#pragma once
#include "ds_common.h"
#include <math.h>

namespace ds {

struct bf16_t { uint16_t bits; };
struct f16_t { uint16_t bits; };

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16_t v) { return __uint_as_float((uint32_t)v.bits << 16); }
__device__ __forceinline__ float to_float(f16_t v) { return (float)__builtin_bit_cast(_Float16, v.bits); }

// Round to nearest even, once, from 32 bits: the only rounding between the sums and a 16-bit output.
template <typename E> __device__ __forceinline__ E from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16_t from_float<bf16_t>(float v)
{
    return bf16_t{__builtin_bit_cast(uint16_t, (__bf16)v)};
}
template <> __device__ __forceinline__ f16_t from_float<f16_t>(float v)
{
    return f16_t{__builtin_bit_cast(uint16_t, (_Float16)v)};
}

// N elements that travel as one access.
template <typename E, int N> struct alignas(sizeof(E) * N) Vec { E v[N]; };

// A result that nobody reads soon.
template <typename E, int N>
__device__ __forceinline__ void store_streaming(Vec<E, N> *to, const Vec<E, N> &v)
{
    constexpr int kBytes = sizeof(E) * N;
    if constexpr (kBytes == 16) {
        typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
        __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), (u32x4 *)to);
    } else if constexpr (kBytes == 8) {
        __builtin_nontemporal_store(__builtin_bit_cast(uint64_t, v), (uint64_t *)to);
    } else if constexpr (kBytes == 4) {
        __builtin_nontemporal_store(__builtin_bit_cast(uint32_t, v), (uint32_t *)to);
    } else {
        __builtin_nontemporal_store(__builtin_bit_cast(uint16_t, v), (uint16_t *)to);
    }
}

// N elements wherever they lie; those from `left` on are not touched (and zeros).
template <typename E, int N>
__device__ __forceinline__ Vec<E, N> load_any(const E *p, int64_t left)
{
    Vec<E, N> v{};
    if (left >= N) {
        __builtin_memcpy(&v, p, sizeof(v));
    } else {
#pragma unroll
        for (int e = 0; e < N - 1; ++e)
            if (e < left) v.v[e] = p[e];
    }
    return v;
}
template <typename E, int N>
__device__ __forceinline__ void store_any(E *p, const Vec<E, N> &v, int64_t left)
{
    static_assert(sizeof(v) == 16, "");
    if (left >= N) {
        // (the compiler is kept from seeing the same values stored on both paths, for which it finds common pieces)
        typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
        u32x4 w = __builtin_bit_cast(u32x4, v);
        asm("" : "+v"(w));
        __builtin_memcpy(p, &w, 16);
    } else {
#pragma unroll
        for (int e = 0; e < N - 1; ++e)
            if (e < left) p[e] = v.v[e];
    }
}

inline int element_bytes(int type) { return type == DS_F32 ? 4 : type == DS_BF16 || type == DS_F16 ? 2 : 0; }

// The widest access, in elements of `bytes`, that every one of the sizes (in elements) and addresses allows.
inline int vector_elements(int bytes, std::initializer_list<int64_t> sizes, std::initializer_list<const void *> at)
{
    int n = 16 / bytes;
    for (int64_t s : sizes)
        while (n > 1 && s % n) n >>= 1;
    for (const void *p : at)
        while (n > 1 && (uintptr_t)p % (size_t)(n * bytes)) n >>= 1;
    return n;
}

// Token numbers come as 32- or 64-bit integers; whatever is not in [0, V) is returned as -1.
__device__ __forceinline__ int token_at(const void *ids, int wide, int64_t i, int64_t V)
{
    const int64_t id = wide ? ((const int64_t *)ids)[i] : (int64_t)((const int32_t *)ids)[i];
    return id >= 0 && id < V ? (int)id : -1;
}

}  // namespace ds
