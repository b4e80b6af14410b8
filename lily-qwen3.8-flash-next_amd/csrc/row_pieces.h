// row_pieces.h - rows of any alignment in pieces of eight elements a lane: f32, bf16 or 8-bit floats in memory, f32 in
// registers.
#pragma once

#include <hip/hip_runtime.h>

#include "device_common.h"

namespace lily {

constexpr float E4M3_TOP = 448.0f;
constexpr float E4M3_TINY = 0x1p-116f;   // a row below it is zeros: 448 / max|y| stays finite down to here

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

// Eight elements as they lie in memory: two pieces of 16 bytes of f32, one of bf16.  (Rows may start at any
// element: the hardware takes wide accesses there.)
struct Raw {
    u32x4 a, b;
};
typedef u32x4 u32x4_at2 __attribute__((aligned(2)));
typedef u32x4 u32x4_at4 __attribute__((aligned(4)));
typedef f32x4 f32x4_at4 __attribute__((aligned(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_at1 __attribute__((aligned(1)));
__device__ __forceinline__ Raw load8(const void* row, uint32_t i, bool bf16) {
    Raw r;
    if (bf16) {
        r.a = *(const LILY_GLOBAL u32x4_at2*)(static_cast<const uint16_t*>(row) + i);
        r.b = r.a;
    } else {
        r.a = *(const LILY_GLOBAL u32x4_at4*)(static_cast<const uint32_t*>(row) + i);
        r.b = *(const LILY_GLOBAL u32x4_at4*)(static_cast<const uint32_t*>(row) + i + 4);
    }
    return r;
}
__device__ __forceinline__ void widen(const Raw& r, bool bf16, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (bf16) {
            v[2 * j] = lilym_bits_f32(r.a[j] << 16);
            v[2 * j + 1] = lilym_bits_f32(r.a[j] & 0xffff0000u);
        } else {
            v[j] = lilym_bits_f32(r.a[j]);
            v[4 + j] = lilym_bits_f32(r.b[j]);
        }
    }
}
// The same of one type.
template <bool BF16>
struct Eight;
template <>
struct Eight<true> {
    u32x4 a;
    __device__ __forceinline__ void load(const void* row, uint32_t i) { a = *(const LILY_GLOBAL u32x4_at2*)(static_cast<const uint16_t*>(row) + i); }
    __device__ __forceinline__ void widened(float (&v)[8]) const { widen({a, a}, true, v); }
};
template <>
struct Eight<false> {
    u32x4 a, b;
    __device__ __forceinline__ void load(const void* row, uint32_t i) {
        a = *(const LILY_GLOBAL u32x4_at4*)(static_cast<const uint32_t*>(row) + i);
        b = *(const LILY_GLOBAL u32x4_at4*)(static_cast<const uint32_t*>(row) + i + 4);
    }
    __device__ __forceinline__ void widened(float (&v)[8]) const { widen({a, b}, false, v); }
};
__device__ __forceinline__ float load1(const void* row, uint32_t i, bool bf16) {
    return bf16 ? load_logit<LILY_BF16>(row, i) : load_logit<LILY_F32>(row, i);
}
__device__ __forceinline__ float rounded(float v, bool bf16) {
    return bf16 ? lilym_bits_f32(bf16_pair(v, 0.0f) << 16) : v;
}
__device__ __forceinline__ void store1(void* row, uint32_t i, float v, uint32_t dtype) {
    if (dtype == LILY_F32) {
        static_cast<float*>(row)[i] = v;
    } else if (dtype == LILY_BF16) {
        static_cast<uint16_t*>(row)[i] = (uint16_t)bf16_pair(v, 0.0f);
    } else {
        static_cast<uint8_t*>(row)[i] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(v, 0.0f, 0, false);
    }
}
__device__ __forceinline__ void store8(void* row, uint32_t i, const float (&v)[8], uint32_t dtype) {
    if (dtype == LILY_F32) {
        LILY_GLOBAL f32x4_at4* p = (LILY_GLOBAL f32x4_at4*)(static_cast<float*>(row) + i);
        p[0] = f32x4{v[0], v[1], v[2], v[3]};
        p[1] = f32x4{v[4], v[5], v[6], v[7]};
    } else if (dtype == LILY_BF16) {
        *(LILY_GLOBAL u32x4_at2*)(static_cast<uint16_t*>(row) + i) =
            u32x4{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7])};
    } else {
        // (nearest even by the conversion; |v| <= 448 (1 + 2^-22), which rounds to 448)
        int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
        int hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], 0, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], hi, true);
        *(LILY_GLOBAL u32x2_at1*)(static_cast<uint8_t*>(row) + i) = u32x2{(uint32_t)lo, (uint32_t)hi};
    }
}

// The wave's sum in every lane: within each row of 16 lanes by DPP shifts, then the four rows' totals.
__device__ __forceinline__ float wave_sum_f(float v) {
#define LILY_ROW_SHR_ADD(n) \
    v += lilym_bits_f32((uint32_t)__builtin_amdgcn_update_dpp(0, (int)lilym_f32_bits(v), 0x110 + (n), 0xf, 0xf, false));
    LILY_ROW_SHR_ADD(1)
    LILY_ROW_SHR_ADD(2)
    LILY_ROW_SHR_ADD(4)
    LILY_ROW_SHR_ADD(8)
#undef LILY_ROW_SHR_ADD
    const int b = (int)lilym_f32_bits(v);
    float t = 0.0f;
#pragma unroll
    for (int l = 15; l < 64; l += 16) {
        t += lilym_bits_f32((uint32_t)__builtin_amdgcn_readlane(b, l));
    }
    return t;
}

// The largest of a row of 16 lanes (64 lanes hold four), in all of them.
__device__ __forceinline__ uint32_t sixteen_max_u32(uint32_t v) {
#define LILY_ROW_ROR_MAX(n) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x120 + (n), 0xf, 0xf, false));
    LILY_ROW_ROR_MAX(1)
    LILY_ROW_ROR_MAX(2)
    LILY_ROW_ROR_MAX(4)
    LILY_ROW_ROR_MAX(8)
#undef LILY_ROW_ROR_MAX
    return v;
}

// What eight-bit values of largest magnitude `top` (its bits: a NaN lies above every number) are stored with: the scale,
// and what they are multiplied by.  (A NaN passes through both; one multiplication by 448 / m is within 1.5 ulp of a
// division by the scale.)
struct Scale8 {
    float scale, inverse;
};
__device__ __forceinline__ Scale8 scale_of(uint32_t top) {
    const float m = lilym_bits_f32(top);
    const bool zeros = m < E4M3_TINY;
    return {zeros ? 0.0f : m / E4M3_TOP, zeros ? 0.0f : E4M3_TOP / m};
}

}  // namespace lily
