// Shared pieces of the operators a block is trained with (layer norm, gated recurrence, balance
// loss): vectors at any alignment, sums over partial columns.
#pragma once

#include "common.hpp"

namespace nsosx {

// Eight (two) consecutive elements in one load or store at the elements' own alignment: the memory
// unit takes a 16-byte access at any address, so rows of an odd length need no path of their own.
struct __attribute__((packed, aligned(2))) bf16x8_any { uint32_t w[4]; };
struct __attribute__((packed, aligned(4))) f32x8_any { float v[8]; };
struct __attribute__((packed, aligned(2))) bf16x2_any { uint32_t w; };
struct __attribute__((packed, aligned(4))) f32x2_any { float v[2]; };

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

// The first n (0 .. 8) of eight elements; the rest read as zeros and are not written.
template <int DT>
__device__ __forceinline__ void load8_part(const void* p, int64_t i, int n, float (&v)[8]) {
    if (n >= 8) {
        load8_any<DT>(p, i, v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < n ? load_act<DT>(p, i + j) : 0.0f;
    }
}

template <int DT>
__device__ __forceinline__ void store8_part(void* p, int64_t i, int n, const float (&v)[8]) {
    if (n >= 8) {
        store8_any<DT>(p, i, v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < n) store_act<DT>(p, i + j, v[j]);
    }
}

// out[a][c] = scale[c] * sum_n part[a][n][c] for a < arrays (out NULL entries are skipped), in a
// fixed order; scale NULL: 1.
void launch_column_sums(const float* part, int arrays, int n, int cols, float* out0, float* out1,
                        hipStream_t st);

// whether [a, a + a_bytes) and [b, b + b_bytes) share a byte but are not the same buffer
inline bool crosses(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
    return overlaps(a, a_bytes, b, b_bytes) && !(a == b && a_bytes == b_bytes);
}

inline int64_t dtype_bytes(int dtype) { return dtype == NSOSX_F32 ? 4 : 2; }

}  // namespace nsosx
