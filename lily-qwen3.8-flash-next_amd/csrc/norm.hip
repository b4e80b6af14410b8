// norm.hip - the residual's addition and the root-mean-square norm in front of the head.
//
//     h = x + residual (rounded to the stream's type),  y = h / sqrt(mean(h^2) + eps) * (w + offset)
//
// One workgroup per row: a thread keeps its part of the row in registers between the sum of squares
// and the outputs, so a row is read once and written once, whatever the number of outputs, and an
// output may lie where an input lay.  Eight-bit rows need the largest |y| as well, which is a second
// reduction over the same registers.  Bound by memory, 3 to 5 operations a byte: 8192 x 4096 bf16 with a bf16 residual
// and sum to E4M3 45.6 us (235 MB, 5.2 TB/s; a copy reaches 5.8), 61 x 2560 4.2 and 4 x 4096 3.0 us on the device, where a
// launch, one trip to memory and two reductions are all there is.
#include <hip/hip_runtime.h>

#include "device_common.h"
#include "operators.h"

namespace lily {

namespace {

struct NormArgs {
    const void* x;
    const void* residual;
    void* sum;
    const void* weight;
    void* out;
    float* scales;
    uint64_t x_stride, residual_stride, sum_stride, out_stride;   // elements
    uint32_t d;
    uint32_t x_bf16, stream_bf16, weight_bf16, out_dtype;
    float eps, offset;
};

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

// CH: pieces of eight elements a thread holds (CH * 8 * blockDim.x >= d).  RAGGED: d is no multiple of 8, and the
// last piece goes element by element.
template <int CH, bool RAGGED>
__global__ void __launch_bounds__(1024) k_rms_norm(const NormArgs a) {
    __shared__ float part[16];
    __shared__ uint32_t top_of[16];
    const uint32_t tid = threadIdx.x, nt = blockDim.x, lane = tid & 63u, wave = tid >> 6, waves = nt >> 6;
    const uint64_t row = blockIdx.x;
    const char* x = static_cast<const char*>(a.x) + row * a.x_stride * (a.x_bf16 ? 2u : 4u);
    const char* res = static_cast<const char*>(a.residual) + row * a.residual_stride * (a.stream_bf16 ? 2u : 4u);
    char* sum = static_cast<char*>(a.sum) + row * a.sum_stride * (a.stream_bf16 ? 2u : 4u);
    char* out = static_cast<char*>(a.out) + row * a.out_stride * (a.out_dtype == LILY_F32 ? 4u : a.out_dtype == LILY_BF16 ? 2u : 1u);
    const bool with_residual = a.residual != nullptr;
    float h[CH][8], w[CH][8];
    auto at = [&](int c) { return ((uint32_t)c * nt + tid) * 8u; };
    auto whole = [&](int c) { return RAGGED ? at(c) + 8u <= a.d : at(c) < a.d; };

    // Everything the row needs is asked for before any of it is looked at (the weights too: they are the same for all
    // rows and come from the L2).  What is not there is worth zeros.
    Raw rx[CH], rr[CH], rw[CH];
    auto from = [&](int c) { return RAGGED ? at(c) : min(at(c), a.d - 8u); };   // (no branch around a load where none is needed)
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        if (!RAGGED || whole(c)) {
            rx[c] = load8(x, from(c), a.x_bf16);
        }
    }
    if (with_residual) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if (!RAGGED || whole(c)) {
                rr[c] = load8(res, from(c), a.stream_bf16);
            }
        }
    }
    if (a.weight != nullptr) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if (!RAGGED || whole(c)) {
                rw[c] = load8(a.weight, from(c), a.weight_bf16);
            }
        }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const uint32_t i = at(c);
        float r[8];
        if (!RAGGED || whole(c)) {
            widen(rx[c], a.x_bf16, h[c]);
            if (with_residual) {
                widen(rr[c], a.stream_bf16, r);
            }
            if (a.weight != nullptr) {
                widen(rw[c], a.weight_bf16, w[c]);
            }
            if (!RAGGED && i >= a.d) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    h[c][j] = r[j] = w[c][j] = 0.0f;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool there = i + (uint32_t)j < a.d;
                h[c][j] = there ? load1(x, i + (uint32_t)j, a.x_bf16) : 0.0f;
                r[j] = there && with_residual ? load1(res, i + (uint32_t)j, a.stream_bf16) : 0.0f;
                w[c][j] = there && a.weight != nullptr ? load1(a.weight, i + (uint32_t)j, a.weight_bf16) : 0.0f;
            }
        }
        if (with_residual) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                h[c][j] = rounded(h[c][j] + r[j], a.stream_bf16);
            }
            if (a.sum != nullptr) {   // (it may lie where x or the residual lies: the thread has read its own elements)
                if (whole(c)) {
                    store8(sum, i, h[c], a.stream_bf16 ? LILY_BF16 : LILY_F32);
                } else if (RAGGED) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if (i + (uint32_t)j < a.d) {
                            store1(sum, i + (uint32_t)j, h[c][j], a.stream_bf16 ? LILY_BF16 : LILY_F32);
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            w[c][j] = a.weight != nullptr ? w[c][j] + a.offset : 1.0f;
        }
    }

    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            ss += h[c][j] * h[c][j];
        }
    }
    ss = wave_sum_f(ss);
    if (lane == 0u) {
        part[wave] = ss;
    }
    __syncthreads();
    ss = 0.0f;
    for (uint32_t q = 0; q < waves; ++q) {
        ss += part[q];
    }
    const float r = 1.0f / sqrtf(ss / (float)a.d + a.eps);
    uint32_t top = 0;   // the largest |y| as its bits: a NaN is above every number
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            h[c][j] = h[c][j] * r * w[c][j];
            top = max(top, lilym_f32_bits(h[c][j]) & 0x7fffffffu);
        }
    }
    if (a.out_dtype == LILY_E4M3) {
        top = wave_max_u32(top);
        if (lane == 0u) {
            top_of[wave] = top;
        }
        __syncthreads();
        for (uint32_t q = 0; q < waves; ++q) {
            top = max(top, top_of[q]);
        }
        const float m = lilym_bits_f32(top);
        const bool zeros = m < E4M3_TINY;
        // (a NaN passes through both; one multiplication by 448 / m is within 1.5 ulp of a division by the scale)
        const float inv = zeros ? 0.0f : E4M3_TOP / m;
        if (tid == 0u) {
            a.scales[row] = zeros ? 0.0f : m / E4M3_TOP;
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                h[c][j] *= inv;
            }
        }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const uint32_t i = at(c);
        if (whole(c)) {
            store8(out, i, h[c], a.out_dtype);
        } else if (RAGGED) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (i + (uint32_t)j < a.d) {
                    store1(out, i + (uint32_t)j, h[c][j], a.out_dtype);
                }
            }
        }
    }
}

}  // namespace

hipError_t launch_rms_norm(hipStream_t stream, const lily_norm& n) {
    NormArgs a = {};
    a.x = n.x_dev;
    a.residual = n.residual_dev;
    a.sum = n.sum_dev;
    a.weight = n.weight_dev;
    a.out = n.out_dev;
    a.scales = n.scales_dev;
    a.x_stride = n.x_stride;
    a.residual_stride = n.residual_stride;
    a.sum_stride = n.sum_stride;
    a.out_stride = n.out_stride;
    a.d = n.d;
    a.x_bf16 = n.x_dtype == LILY_BF16;
    a.stream_bf16 = n.stream_dtype == LILY_BF16;
    a.weight_bf16 = n.weight_dtype == LILY_BF16;
    a.out_dtype = n.out_dtype;
    a.eps = n.eps;
    a.offset = n.weight_offset;
    const NormShape shape = norm_shape(n.d);
    const uint32_t ch = shape.pieces;
    const dim3 grid(n.rows), block(shape.threads);
#define LILY_NORM(CH)                                                              \
    if (n.d % 8u != 0u) {                                                          \
        hipLaunchKernelGGL((k_rms_norm<CH, true>), grid, block, 0, stream, a);     \
    } else {                                                                       \
        hipLaunchKernelGGL((k_rms_norm<CH, false>), grid, block, 0, stream, a);    \
    }
    if (ch == 1u) {
        LILY_NORM(1)
    } else if (ch == 2u) {
        LILY_NORM(2)
    } else {
        LILY_NORM(4)
    }
#undef LILY_NORM
    return hipGetLastError();
}

}  // namespace lily
