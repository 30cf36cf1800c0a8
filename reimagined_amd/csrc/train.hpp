// Shared pieces of the operators a block is trained with (layer norm, gated recurrence, balance
// loss): vectors at any alignment, checks of buffers.
#pragma once

#include "common.hpp"

namespace nsosx {

// Eight consecutive elements in one load or store at the elements' own alignment: the memory
// unit takes a 16-byte access at any address, so rows of an odd length need no path of their own.
struct __attribute__((packed, aligned(2))) bf16x8_any { uint32_t w[4]; };
struct __attribute__((packed, aligned(4))) f32x8_any { float v[8]; };

template <int DT>
__device__ __forceinline__ void load8_any(const void* p, int64_t i, float (&v)[8]) {
    if constexpr (DT == NSOSX_F32) {
        const f32x8_any a = *reinterpret_cast<const f32x8_any*>(static_cast<const float*>(p) + i);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = a.v[j];
    } else {
        const bf16x8_any a = *reinterpret_cast<const bf16x8_any*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[2 * j] = __uint_as_float(a.w[j] << 16);
            v[2 * j + 1] = __uint_as_float(a.w[j] & 0xffff0000u);
        }
    }
}

template <int DT>
__device__ __forceinline__ void store8_any(void* p, int64_t i, const float (&v)[8]) {
    if constexpr (DT == NSOSX_F32) {
        f32x8_any a;
#pragma unroll
        for (int j = 0; j < 8; ++j) a.v[j] = v[j];
        *reinterpret_cast<f32x8_any*>(static_cast<float*>(p) + i) = a;
    } else {
        bf16x8_any a;
#pragma unroll
        for (int j = 0; j < 4; ++j) a.w[j] = pack_bf16x2(v[2 * j], v[2 * j + 1]);
        *reinterpret_cast<bf16x8_any*>(static_cast<uint16_t*>(p) + i) = a;
    }
}

// Eight elements as loaded: what is asked for early is kept in this form, half the registers for bf16,
// and costs no wait before it is used.
template <int DT> struct Raw8;
template <> struct Raw8<NSOSX_BF16> {
    bf16x8_any w;
    __device__ __forceinline__ void load(const void* p, int64_t i) {
        w = *reinterpret_cast<const bf16x8_any*>(static_cast<const uint16_t*>(p) + i);
    }
    __device__ __forceinline__ float get(int j) const {
        return __uint_as_float(j & 1 ? w.w[j / 2] & 0xffff0000u : w.w[j / 2] << 16);
    }
    __device__ __forceinline__ void wait() {  // (a use: the load is back behind it)
        asm volatile("" : "+v"(w.w[0]), "+v"(w.w[1]), "+v"(w.w[2]), "+v"(w.w[3])::"memory");
    }
};
template <> struct Raw8<NSOSX_F32> {
    f32x8_any v;
    __device__ __forceinline__ void load(const void* p, int64_t i) {
        v = *reinterpret_cast<const f32x8_any*>(static_cast<const float*>(p) + i);
    }
    __device__ __forceinline__ float get(int j) const { return v.v[j]; }
    __device__ __forceinline__ void wait() {
#pragma unroll
        for (int j = 0; j < 8; ++j) asm volatile("" : "+v"(v.v[j])::"memory");
    }
};

// whether [a, a + a_bytes) and [b, b + b_bytes) share a byte but are not the same buffer
inline bool crosses(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
    return overlaps(a, a_bytes, b, b_bytes) && !(a == b && a_bytes == b_bytes);
}

inline int64_t dtype_bytes(int dtype) { return dtype == NSOSX_F32 ? 4 : 2; }

}  // namespace nsosx
