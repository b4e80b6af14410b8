// project.h - what the kernels of the matrix product with an epilogue share: operands, products, the
// epilogue.
//
//     out[r][v] = residual[r][v] + act(xs[r] * ws[v] * sum_i x[r][i] * w[v][i] + bias[v])
//
// Both operands are contiguous along d, in bf16 or in 8-bit floats (E4M3), and are taken 128 bytes of a row
// at a time: eight pieces of 16 bytes.  A lane of a 16 x 16 product holds row lane % 16 and, of the
// 128 bytes, pieces g and g + 4, g = lane / 16.  (Which element of d meets which is free as
// long as both operands agree.)  The weights are the products' first operand, so that a lane's four sums
// are four neighbouring outputs of one row.
#pragma once

#include <hip/hip_runtime.h>

#include "device_common.h"
#include "operators.h"

namespace lily {

constexpr uint32_t LINE = 128;   // bytes of a row that are taken at a time

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct ProjectArgs {
    const char* x;
    const char* w;
    const float* x_scales;      // or null
    const float* w_scales;      // or null
    const void* bias;           // or null
    const void* residual;       // or null
    void* out;
    uint64_t x_stride, w_stride;               // bytes
    uint64_t residual_stride, out_stride;      // elements
    uint32_t rows, n, d_bytes;
    uint32_t bias_bf16, residual_bf16, out_bf16, act;
    uint32_t wide;              // four neighbouring outputs (and residuals) start at multiples of their size
    uint32_t splits;            // parts of d, each a workgroup's
    uint32_t relaxed;           // the form of their hand-over
    Handed<uint64_t> part;      // their sums
    uint32_t* ticket;           // [tiles], zero between launches
};

// The operand of a lane: two pieces.
struct Frag {
    u32x4 lo, hi;
};

// How 128 bytes of two rows are multiplied.
//
// PRODUCT_E4M3 is the matrix cores' own 8-bit product: twice bf16's rate, but the eight products of eight
// neighbouring elements are aligned to the largest exponent E among them and cut off at 2^(E - 13) before they
// are added (measured: 2^10 + 0.2197 comes out as 2^10 + 0.125, 2^10 in one such group and 0.2197 in the next
// exactly).  That leaves up to 7 * 2^-13 of each group's largest product, 6e-5 of the result for normal
// data: a seventieth of the rounding of a bf16 output, and only such outputs take it.
// PRODUCT_E4M3_WIDE turns both operands into bf16 (exact) on their way: products and sums as bf16 has them.
enum Products { PRODUCT_BF16, PRODUCT_E4M3, PRODUCT_E4M3_WIDE };

typedef __bf16 pj_bf16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ bf16x8 widened(uint32_t a, uint32_t b) {
    const pj_bf16x2 p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)a, 1.0f, false);
    const pj_bf16x2 q = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)a, 1.0f, true);
    const pj_bf16x2 r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)b, 1.0f, false);
    const pj_bf16x2 t = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)b, 1.0f, true);
    return bf16x8{p[0], p[1], q[0], q[1], r[0], r[1], t[0], t[1]};
}

template <Products P>
__device__ __forceinline__ f32x4 product(const Frag& w, const Frag& x, f32x4 c) {
    if constexpr (P == PRODUCT_E4M3) {
        const u32x8 a = __builtin_shufflevector(w.lo, w.hi, 0, 1, 2, 3, 4, 5, 6, 7);
        const u32x8 b = __builtin_shufflevector(x.lo, x.hi, 0, 1, 2, 3, 4, 5, 6, 7);
        // (both operands E4M3, block scales of one)
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_bit_cast(i32x8, a), __builtin_bit_cast(i32x8, b),
                                                                c, 0, 0, 0, 0, 0, 0);
    } else if constexpr (P == PRODUCT_E4M3_WIDE) {
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widened(w.lo[0], w.lo[1]), widened(x.lo[0], x.lo[1]), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widened(w.lo[2], w.lo[3]), widened(x.lo[2], x.lo[3]), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widened(w.hi[0], w.hi[1]), widened(x.hi[0], x.hi[1]), c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(widened(w.hi[2], w.hi[3]), widened(x.hi[2], x.hi[3]), c, 0, 0, 0);
    } else {
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w.lo), __builtin_bit_cast(bf16x8, x.lo), c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w.hi), __builtin_bit_cast(bf16x8, x.hi), c, 0, 0, 0);
    }
}

// The activations, f32.  The reciprocal is the hardware's (1 ulp); none of the forms cancels: GELU's
// tail comes from erfc, the other two are v times a logistic function.
__device__ __forceinline__ float logistic(float v) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * v));
}
__device__ __forceinline__ float activated(float v, uint32_t act) {
    switch (act) {
    case LILY_ACT_SILU:
        return v * logistic(v);
    case LILY_ACT_GELU:
        return 0.5f * v * erfcf(-0.70710678118654752f * v);
    case LILY_ACT_GELU_TANH: {
        const float u = 1.5957691216057308f * (v + 0.044715f * v * v * v);   // 2 sqrt(2 / pi) (v + ...)
        return v * logistic(u);
    }
    case LILY_ACT_RELU:
        return v > 0.0f || v != v ? v : 0.0f;
    default:
        return v;
    }
}

typedef float pj_f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t pj_u32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pj_bf16_pair(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((pj_f32x2{a, b}), pj_bf16x2));
}

// What the epilogue knows of four neighbouring columns before it sees a row.
struct Columns {
    float scale[4], bias[4];
};
__device__ __forceinline__ Columns columns_at(const ProjectArgs& a, uint32_t v0) {
    Columns c;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t v = min(v0 + (uint32_t)j, a.n - 1u);
        c.scale[j] = a.w_scales != nullptr ? gload(a.w_scales + v) : 1.0f;
        c.bias[j] = a.bias == nullptr ? 0.0f
                    : a.bias_bf16     ? lilym_bits_f32((uint32_t)gload(static_cast<const uint16_t*>(a.bias) + v) << 16)
                                      : gload(static_cast<const float*>(a.bias) + v);
    }
    return c;
}

// Sums of row r (< rows), columns v0 .. v0 + 3, finished and stored.
__device__ __forceinline__ void finish(const ProjectArgs& a, uint32_t r, uint32_t v0, const Columns& c, float x_scale, f32x4 sum) {
    if (v0 >= a.n) {
        return;
    }
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[j] = sum[j] * x_scale * c.scale[j] + c.bias[j];
    }
    if (a.act != LILY_ACT_NONE) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = activated(v[j], a.act);
        }
    }
    const uint64_t at = (uint64_t)r * a.out_stride + v0, from = (uint64_t)r * a.residual_stride + v0;
    if (a.wide && v0 + 4u <= a.n) {
        if (a.residual != nullptr) {
            if (a.residual_bf16) {
                const pj_u32x2 q = gload(reinterpret_cast<const pj_u32x2*>(static_cast<const uint16_t*>(a.residual) + from));
                v[0] += lilym_bits_f32(q.x << 16);
                v[1] += lilym_bits_f32(q.x & 0xffff0000u);
                v[2] += lilym_bits_f32(q.y << 16);
                v[3] += lilym_bits_f32(q.y & 0xffff0000u);
            } else {
                const f32x4 q = gload(reinterpret_cast<const f32x4*>(static_cast<const float*>(a.residual) + from));
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[j] += q[j];
                }
            }
        }
        if (a.out_bf16) {
            *(LILY_GLOBAL pj_u32x2*)(static_cast<uint16_t*>(a.out) + at) =
                pj_u32x2{pj_bf16_pair(v[0], v[1]), pj_bf16_pair(v[2], v[3])};
        } else {
            *(LILY_GLOBAL f32x4*)(static_cast<float*>(a.out) + at) = f32x4{v[0], v[1], v[2], v[3]};
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (v0 + (uint32_t)j < a.n) {
            if (a.residual != nullptr) {
                v[j] += a.residual_bf16 ? load_logit<LILY_BF16>(static_cast<const uint16_t*>(a.residual) + from, (uint32_t)j)
                                        : load_logit<LILY_F32>(static_cast<const float*>(a.residual) + from, (uint32_t)j);
            }
            if (a.out_bf16) {
                *(LILY_GLOBAL uint16_t*)(static_cast<uint16_t*>(a.out) + at + j) = (uint16_t)pj_bf16_pair(v[j], 0.0f);
            } else {
                *(LILY_GLOBAL float*)(static_cast<float*>(a.out) + at + j) = v[j];
            }
        }
    }
}

hipError_t launch_project_few(hipStream_t stream, const ProjectArgs& a, bool e4m3);
hipError_t launch_project_tiles(hipStream_t stream, ProjectArgs& a, bool e4m3, uint64_t part_words, uint32_t tickets,
                                uint32_t handover);

}  // namespace lily
