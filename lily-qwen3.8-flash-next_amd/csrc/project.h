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
#include "project_plan.h"

namespace lily {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

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
// PRODUCT_BLOCKS and PRODUCT_BLOCKS_WIDE are the same two for operands with a scale for each 128 elements, which are 128 bytes:
// a line's products are summed by themselves, and their sum times both scales is added in f32.
enum Products { PRODUCT_BF16, PRODUCT_E4M3, PRODUCT_E4M3_WIDE, PRODUCT_BLOCKS, PRODUCT_BLOCKS_WIDE };
constexpr bool in_blocks(Products p) { return p == PRODUCT_BLOCKS || p == PRODUCT_BLOCKS_WIDE; }

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
    static_assert(P != PRODUCT_E4M3 && P != PRODUCT_BLOCKS, "few rows are read at the speed of memory: they take the exact products");
    if constexpr (P == PRODUCT_E4M3_WIDE || P == PRODUCT_BLOCKS_WIDE) {
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
// tail is formed by itself, the other two are v times a logistic function.
__device__ __forceinline__ float logistic(float v) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * v));
}
// The normal distribution's tail beyond |v|, exp(-v^2 / 2) t Q(t) with t = 1 / (1 + 0.36 |v|): Q is the polynomial of degree 9
// that is nearest to exp(v^2 / 2) Phi(-|v|) / t relatively, over |v| <= 14.5, where the tail leaves the numbers (a least-squares fit on
// Chebyshev points, its weights raised where it is worst: 2e-8).  With its roundings within (8 + v^2) 2^-24 of the tail.
// 26 operations a value where erfc takes some eighty: 8192 x 4096 x 4096 bf16 266 us with that, a row at a time.
__device__ __forceinline__ float tail_beyond(float v) {
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.36f, fabsf(v), 1.0f));
    float q = 0.010566466f;
    q = __builtin_fmaf(q, t, -0.084390737f);
    q = __builtin_fmaf(q, t, 0.25836042f);
    q = __builtin_fmaf(q, t, -0.36961335f);
    q = __builtin_fmaf(q, t, 0.21752089f);
    q = __builtin_fmaf(q, t, -0.053044252f);
    q = __builtin_fmaf(q, t, 0.11190969f);
    q = __builtin_fmaf(q, t, 0.12111426f);
    q = __builtin_fmaf(q, t, 0.14397095f);
    q = __builtin_fmaf(q, t, 0.14360565f);
    return __builtin_amdgcn_exp2f(v * v * -0.72134752f) * (t * q);
}
template <int N>
__device__ __forceinline__ void activate(float (&v)[N], uint32_t act) {   // (one branch for all of them)
    if (act == LILY_ACT_SILU) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            v[j] *= logistic(v[j]);
        }
    } else if (act == LILY_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float tail = tail_beyond(v[j]);
            v[j] *= v[j] > 0.0f ? 1.0f - tail : tail;
        }
    } else if (act == LILY_ACT_GELU_TANH) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            v[j] *= logistic(1.5957691216057308f * (v[j] + 0.044715f * v[j] * v[j] * v[j]));   // 2 sqrt(2 / pi) (v + ...)
        }
    } else if (act == LILY_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            v[j] = v[j] > 0.0f || v[j] != v[j] ? v[j] : 0.0f;
        }
    }
}

typedef float pj_f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t pj_u32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pj_bf16_pair(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((pj_f32x2{a, b}), pj_bf16x2));
}

// What the epilogue knows of four neighbouring columns before it sees a row.  (As it lies in memory: values are
// widened where they are used, so that nobody waits for them before.)
struct Columns {
    float scale[4];
    uint32_t raw[4];
    __device__ __forceinline__ void load(const ProjectArgs& a, uint32_t v0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t v = min(v0 + (uint32_t)j, a.n - 1u);
            scale[j] = 1.0f;
            raw[j] = 0u;
            if (a.w_scales != nullptr) {
                scale[j] = gload(a.w_scales + v);
            }
            if (a.bias != nullptr) {
                raw[j] = a.bias_bf16 ? (uint32_t)gload(static_cast<const uint16_t*>(a.bias) + v)
                                     : gload(static_cast<const uint32_t*>(a.bias) + v);
            }
        }
    }
    __device__ __forceinline__ float bias(const ProjectArgs& a, int j) const {
        return lilym_bits_f32(a.bias_bf16 ? raw[j] << 16 : raw[j]);
    }
};

// (rows of any alignment: the hardware takes wide accesses at any element)
typedef pj_u32x2 pj_u32x2_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef u32x4 pj_u32x4_any __attribute__((aligned(4)));

// Row r (r < rows) of columns v0 .. v0 + 3 (v0 < n): load() asks for what the epilogue reads of it, store() finishes
// its sums.
struct Finish {
    float scale;
    u32x4 res;   // two bf16 a word, or f32
    __device__ __forceinline__ void load(const ProjectArgs& a, uint32_t r, uint32_t v0) {
        if (a.x_scales != nullptr) {
            scale = gload(a.x_scales + r);
        }
        if (a.residual == nullptr) {
            return;
        }
        const uint64_t from = (uint64_t)r * a.residual_stride + v0;
        if (v0 + 4u <= a.n && a.residual_bf16) {
            const pj_u32x2 t = *(const LILY_GLOBAL pj_u32x2_any*)(static_cast<const uint16_t*>(a.residual) + from);
            res = u32x4{t.x, t.y, 0u, 0u};
        } else if (v0 + 4u <= a.n) {
            res = *(const LILY_GLOBAL pj_u32x4_any*)(static_cast<const uint32_t*>(a.residual) + from);
        } else {
            uint32_t t[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint64_t at = from + min((uint32_t)j, a.n - 1u - v0);
                t[j] = a.residual_bf16 ? (uint32_t)gload(static_cast<const uint16_t*>(a.residual) + at)
                                       : gload(static_cast<const uint32_t*>(a.residual) + at);
            }
            res = a.residual_bf16 ? u32x4{t[0] | t[1] << 16, t[2] | t[3] << 16, 0u, 0u} : u32x4{t[0], t[1], t[2], t[3]};
        }
    }
    __device__ __forceinline__ void store(const ProjectArgs& a, uint32_t r, uint32_t v0, const Columns& c, f32x4 sum) const {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float t = a.x_scales != nullptr ? sum[j] * scale : sum[j];
            v[j] = t * c.scale[j] + c.bias(a, j);
        }
        activate(v, a.act);
        if (a.residual != nullptr) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t half = (j & 1) ? res[j / 2] & 0xffff0000u : res[j / 2] << 16;
                v[j] += lilym_bits_f32(a.residual_bf16 ? half : res[j]);
            }
        }
        const uint64_t at = (uint64_t)r * a.out_stride + v0;
        if (v0 + 4u > a.n) {
#pragma unroll
            for (int j = 0; j < 3; ++j) {
                if (v0 + (uint32_t)j < a.n) {
                    if (a.out_bf16) {
                        *(LILY_GLOBAL uint16_t*)(static_cast<uint16_t*>(a.out) + at + j) = (uint16_t)pj_bf16_pair(v[j], 0.0f);
                    } else {
                        *(LILY_GLOBAL float*)(static_cast<float*>(a.out) + at + j) = v[j];
                    }
                }
            }
        } else if (a.out_bf16) {
            *(LILY_GLOBAL pj_u32x2_any*)(static_cast<uint16_t*>(a.out) + at) = pj_u32x2{pj_bf16_pair(v[0], v[1]), pj_bf16_pair(v[2], v[3])};
        } else {
            *(LILY_GLOBAL f32x4_any*)(static_cast<float*>(a.out) + at) = f32x4{v[0], v[1], v[2], v[3]};
        }
    }
};

// What a lane knows of the weights' scales: those of 64 lines of d, one a lane, handed out by line.  (A register that is filled in a
// loop and read in it would be waited for, and with it everything asked for since, at every reading: it is waited for where it
// is filled.)
struct WeightScales {
    const float* from;   // of the first line
    uint32_t count;      // lines
    float run;
    __device__ __forceinline__ void ask(uint32_t line) {   // line: a multiple of 64 below count
        run = gload(from + min(line + (threadIdx.x & 63u), count - 1u));
    }
    __device__ __forceinline__ void settle() { asm volatile("" : "+v"(run)); }
    __device__ __forceinline__ float of(uint32_t line) const {
        return lilym_bits_f32((uint32_t)__builtin_amdgcn_readlane((int)lilym_f32_bits(run), (int)(line & 63u)));
    }
};

hipError_t launch_project_few(hipStream_t stream, const ProjectArgs& a, Products products);
// `tile`: 64, 128 or 256 rows and outputs; a.splits parts of d.
hipError_t launch_project_tiles(hipStream_t stream, const ProjectArgs& a, bool e4m3, uint32_t tile);
hipError_t launch_project_join(hipStream_t stream, const ProjectArgs& a);

}  // namespace lily
