// layer_norm.hip - the residual's addition with the layer norm, and its backward pass.
//
//     h = x + residual (rounded to the stream's type),  y = (h - mean) / sqrt(var + eps) * w + b
//
// One workgroup per row: a thread keeps its part of the row in registers through both sums (the values', then that of the
// squared distances from their mean, which does not cancel) and the outputs, so a row is read once and written once.  A
// block of 128 elements with a scale of its own is a row of 16 lanes: its largest value takes no memory and no barrier.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "operators.h"
#include "row_pieces.h"

namespace lily {

namespace {

struct LayerArgs {
    const void* x;
    const void* residual;
    void* sum;
    const void* weight;
    const void* bias;
    void* out;
    float* scales;
    float* mean;
    float* rstd;
    uint64_t x_stride, residual_stride, sum_stride, out_stride, scales_stride;   // elements
    uint32_t d;
    uint32_t x_bf16, stream_bf16, weight_bf16, out_dtype, blocks;
    float eps;
};

__device__ __forceinline__ const char* row_at(const void* p, uint64_t row, uint64_t stride, bool bf16) {
    return static_cast<const char*>(p) + row * stride * (bf16 ? 2u : 4u);
}

// The workgroup's sum in every thread; `part` is a place of its own for each sum.
__device__ __forceinline__ float group_sum(float v, float* part, uint32_t waves) {
    v = wave_sum_f(v);
    if ((threadIdx.x & 63u) == 0u) {
        part[threadIdx.x >> 6] = v;
    }
    __syncthreads();
    v = 0.0f;
    for (uint32_t q = 0; q < waves; ++q) {
        v += part[q];
    }
    return v;
}

// CH: pieces of eight elements a thread holds (CH * 8 * blockDim.x >= d).  RAGGED: d is no multiple of 8, and the
// last piece goes element by element.
template <int CH, bool RAGGED>
__global__ void __launch_bounds__(1024) k_layer_norm(const LayerArgs a) {
    __shared__ float part[2][16];
    __shared__ uint32_t top_of[16];
    const uint32_t tid = threadIdx.x, nt = blockDim.x, lane = tid & 63u, wave = tid >> 6, waves = nt >> 6;
    const uint64_t row = blockIdx.x;
    const char* x = row_at(a.x, row, a.x_stride, a.x_bf16);
    const char* res = row_at(a.residual, row, a.residual_stride, a.stream_bf16);
    char* sum = const_cast<char*>(row_at(a.sum, row, a.sum_stride, a.stream_bf16));
    char* out = static_cast<char*>(a.out) + row * a.out_stride * (a.out_dtype == LILY_F32 ? 4u : a.out_dtype == LILY_BF16 ? 2u : 1u);
    const bool with_residual = a.residual != nullptr;
    float h[CH][8];
    auto at = [&](int c) { return ((uint32_t)c * nt + tid) * 8u; };
    auto whole = [&](int c) { return RAGGED ? at(c) + 8u <= a.d : at(c) < a.d; };

    // Everything the row needs is asked for before any of it is looked at (weight and bias too: they are the same for all
    // rows and come from the L2).
    Raw rx[CH], rr[CH], rw[CH], rb[CH];
    auto from = [&](int c) { return RAGGED ? at(c) : min(at(c), a.d - 8u); };   // (no branch around a load where none is needed)
    auto ask = [&](Raw (&r)[CH], const void* p, bool bf16) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if (!RAGGED || whole(c)) {
                r[c] = load8(p, from(c), bf16);
            }
        }
    };
    ask(rx, x, a.x_bf16);
    if (with_residual) {
        ask(rr, res, a.stream_bf16);
    }
    if (a.weight != nullptr) {
        ask(rw, a.weight, a.weight_bf16);
    }
    if (a.bias != nullptr) {
        ask(rb, a.bias, a.weight_bf16);
    }
    // Eight values of an operand, `none` where it is not there and zeros behind the row's end.
    auto take = [&](const Raw& raw, const void* p, bool bf16, bool there, float none, int c, float (&v)[8]) {
        const uint32_t i = at(c);
        if (!there) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = none;
            }
        } else if (!RAGGED || whole(c)) {
            widen(raw, bf16, v);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = i + (uint32_t)j < a.d ? load1(p, i + (uint32_t)j, bf16) : 0.0f;
            }
        }
    };
    float total = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const uint32_t i = at(c);
        float r[8];
        take(rx[c], x, a.x_bf16, true, 0.0f, c, h[c]);
        if (with_residual) {
            take(rr[c], res, a.stream_bf16, true, 0.0f, c, r);
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
        float t = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            t += h[c][j];
        }
        total += !RAGGED && i >= a.d ? 0.0f : t;
    }
    const float mean = group_sum(total, part[0], waves) / (float)a.d;
    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            h[c][j] = at(c) + (uint32_t)j < a.d ? h[c][j] - mean : 0.0f;
            ss = __builtin_fmaf(h[c][j], h[c][j], ss);
        }
    }
    const float rstd = 1.0f / sqrtf(group_sum(ss, part[1], waves) / (float)a.d + a.eps);
    if (tid == 0u) {
        if (a.mean != nullptr) {
            a.mean[row] = mean;
        }
        if (a.rstd != nullptr) {
            a.rstd[row] = rstd;
        }
    }
    uint32_t top[CH];   // of a piece, the largest |y| as its bits: a NaN is above every number
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        float w[8], b[8];
        take(rw[c], a.weight, a.weight_bf16, a.weight != nullptr, 1.0f, c, w);
        take(rb[c], a.bias, a.weight_bf16, a.bias != nullptr, 0.0f, c, b);
        top[c] = 0u;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            h[c][j] = __builtin_fmaf(h[c][j] * rstd, w[j], b[j]);
            top[c] = max(top[c], at(c) + (uint32_t)j < a.d ? lilym_f32_bits(h[c][j]) & 0x7fffffffu : 0u);
        }
    }
    if (a.out_dtype == LILY_E4M3) {
        if (a.blocks == 0u) {
            uint32_t most = 0u;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                most = max(most, top[c]);
            }
            most = wave_max_u32(most);
            if (lane == 0u) {
                top_of[wave] = most;
            }
            __syncthreads();
            for (uint32_t q = 0; q < waves; ++q) {
                most = max(most, top_of[q]);
            }
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                top[c] = most;
            }
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const Scale8 by = scale_of(a.blocks != 0u ? sixteen_max_u32(top[c]) : top[c]);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                h[c][j] *= by.inverse;
            }
            const uint32_t block = at(c) / LILY_BLOCK;
            if (a.blocks == 0u ? c == 0 && tid == 0u : (lane & 15u) == 0u && block < a.blocks) {
                a.scales[a.blocks == 0u ? row : row * a.scales_stride + block] = by.scale;
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

// ------------------------------------------------------------------ the backward pass

struct LayerGradArgs {
    const void* grad;
    const void* h;
    const float* mean;
    const float* rstd;
    const void* weight;
    const void* past;
    void* grad_x;
    float* grad_weight;
    float* grad_bias;
    float* part;                // [parts][2][wide]: sums over a part's rows, of grad * x and of grad
    uint64_t grad_stride, h_stride, past_stride, grad_x_stride;   // elements
    uint32_t rows, d, wide, parts;
    uint32_t grad_bf16, h_bf16, weight_bf16, grad_x_bf16, accumulate;
};

template <int CH, bool RAGGED>
__global__ void __launch_bounds__(1024) k_layer_grad(const LayerGradArgs a) {
    __shared__ float part[2][16];
    const uint32_t tid = threadIdx.x, nt = blockDim.x, waves = nt >> 6;
    const uint64_t row = blockIdx.x;
    const char* grad = row_at(a.grad, row, a.grad_stride, a.grad_bf16);
    const char* from_h = row_at(a.h, row, a.h_stride, a.h_bf16);
    const char* past = row_at(a.past, row, a.past_stride, a.grad_x_bf16);
    char* to = const_cast<char*>(row_at(a.grad_x, row, a.grad_x_stride, a.grad_x_bf16));
    const float mean = gload(a.mean + row), rstd = gload(a.rstd + row);
    auto at = [&](int c) { return ((uint32_t)c * nt + tid) * 8u; };
    auto take = [&](const void* p, bool bf16, int c, float (&v)[8]) {
        const uint32_t i = at(c);
        if (i + 8u <= a.d) {
            widen(load8(p, i, bf16), bf16, v);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = RAGGED && i + (uint32_t)j < a.d ? load1(p, i + (uint32_t)j, bf16) : 0.0f;
            }
        }
    };
    float g[CH][8], x[CH][8], sg = 0.0f, sx = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        float w[8];
        take(grad, a.grad_bf16, c, g[c]);
        take(from_h, a.h_bf16, c, x[c]);
        if (a.weight != nullptr) {
            take(a.weight, a.weight_bf16, c, w);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            g[c][j] = a.weight != nullptr ? g[c][j] * w[j] : g[c][j];
            x[c][j] = (x[c][j] - mean) * rstd;
            sg += g[c][j];
            sx = __builtin_fmaf(g[c][j], x[c][j], sx);
        }
    }
    sg = group_sum(sg, part[0], waves) / (float)a.d;
    sx = group_sum(sx, part[1], waves) / (float)a.d;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const uint32_t i = at(c);
        float p[8];
        if (a.past != nullptr) {
            take(past, a.grad_x_bf16, c, p);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float v = rstd * (g[c][j] - sg - x[c][j] * sx);
            g[c][j] = a.past != nullptr ? v + p[j] : v;
        }
        if (i + 8u <= a.d) {
            store8(to, i, g[c], a.grad_x_bf16 ? LILY_BF16 : LILY_F32);
        } else if (RAGGED) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (i + (uint32_t)j < a.d) {
                    store1(to, i + (uint32_t)j, g[c][j], a.grad_x_bf16 ? LILY_BF16 : LILY_F32);
                }
            }
        }
    }
}

// Sums over the rows of a part (blockIdx.y, every a.parts-th row), 64 lanes of eight elements by four rows at a time.
template <bool RAGGED>
__global__ void __launch_bounds__(256) k_layer_columns(const LayerGradArgs a) {
    __shared__ float share[3][64][17];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, i = (blockIdx.x * 64u + lane) * 8u;
    float gw[8] = {}, gb[8] = {};
    for (uint64_t row = blockIdx.y + (uint64_t)wave * a.parts; row < a.rows; row += 4ull * a.parts) {
        const char* grad = row_at(a.grad, row, a.grad_stride, a.grad_bf16);
        const char* from_h = row_at(a.h, row, a.h_stride, a.h_bf16);
        const float mean = gload(a.mean + row), rstd = gload(a.rstd + row);
        float g[8], x[8];
        if (i + 8u <= a.d) {
            widen(load8(grad, i, a.grad_bf16), a.grad_bf16, g);
            widen(load8(from_h, i, a.h_bf16), a.h_bf16, x);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool there = RAGGED && i + (uint32_t)j < a.d;
                g[j] = there ? load1(grad, i + (uint32_t)j, a.grad_bf16) : 0.0f;
                x[j] = there ? load1(from_h, i + (uint32_t)j, a.h_bf16) : 0.0f;
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            gb[j] += g[j];
            gw[j] = __builtin_fmaf(g[j], (x[j] - mean) * rstd, gw[j]);
        }
    }
    if (wave != 0u) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            share[wave - 1u][lane][j] = gw[j];
            share[wave - 1u][lane][8 + j] = gb[j];
        }
    }
    __syncthreads();
    if (wave == 0u && i < a.wide) {
        float* to = a.part + (uint64_t)blockIdx.y * 2u * a.wide + i;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int q = 0; q < 3; ++q) {
                gw[j] += share[q][lane][j];
                gb[j] += share[q][lane][8 + j];
            }
            to[j] = gw[j];
            to[a.wide + j] = gb[j];
        }
    }
}

// The parts joined, in order: 32 columns of one of the two a workgroup, eight runs of parts.
__global__ void __launch_bounds__(256) k_layer_join(const LayerGradArgs a) {
    __shared__ float share[8][32];
    const uint32_t column = threadIdx.x & 31u, run = threadIdx.x >> 5, i = blockIdx.x * 32u + column;
    float* to = blockIdx.y == 0u ? a.grad_weight : a.grad_bias;
    const uint32_t per = (a.parts + 7u) / 8u, last = min((run + 1u) * per, a.parts);
    float sum = 0.0f;
    for (uint32_t p = run * per; p < last; ++p) {
        sum += gload(a.part + ((uint64_t)p * 2u + blockIdx.y) * a.wide + min(i, a.wide - 1u));
    }
    share[run][column] = sum;
    __syncthreads();
    if (run == 0u && i < a.d && to != nullptr) {
        for (uint32_t q = 1; q < 8u; ++q) {
            sum += share[q][column];
        }
        to[i] = a.accumulate != 0u ? to[i] + sum : sum;
    }
}

}  // namespace

hipError_t launch_layer_norm(hipStream_t stream, const lily_layer& n) {
    LayerArgs a = {};
    a.x = n.x_dev;
    a.residual = n.residual_dev;
    a.sum = n.sum_dev;
    a.weight = n.weight_dev;
    a.bias = n.bias_dev;
    a.out = n.out_dev;
    a.scales = n.scales_dev;
    a.mean = n.mean_dev;
    a.rstd = n.rstd_dev;
    a.x_stride = n.x_stride;
    a.residual_stride = n.residual_stride;
    a.sum_stride = n.sum_stride;
    a.out_stride = n.out_stride;
    a.scales_stride = n.scales_stride;
    a.d = n.d;
    a.x_bf16 = n.x_dtype == LILY_BF16;
    a.stream_bf16 = n.stream_dtype == LILY_BF16;
    a.weight_bf16 = n.weight_dtype == LILY_BF16;
    a.out_dtype = n.out_dtype;
    a.blocks = n.scale_block == 0u ? 0u : (n.d + LILY_BLOCK - 1u) / LILY_BLOCK;
    a.eps = n.eps;
    const NormShape shape = norm_shape(n.d);
    const dim3 grid(n.rows), block(shape.threads);
#define LILY_LAYER(CH)                                                             \
    if (n.d % 8u != 0u) {                                                          \
        hipLaunchKernelGGL((k_layer_norm<CH, true>), grid, block, 0, stream, a);   \
    } else {                                                                       \
        hipLaunchKernelGGL((k_layer_norm<CH, false>), grid, block, 0, stream, a);  \
    }
    if (shape.pieces == 1u) {
        LILY_LAYER(1)
    } else if (shape.pieces == 2u) {
        LILY_LAYER(2)
    } else {
        LILY_LAYER(4)
    }
#undef LILY_LAYER
    return hipGetLastError();
}

hipError_t launch_layer_norm_backward(hipStream_t stream, const lily_layer_grad& n, const ProjectWorkspace& ws) {
    LayerGradArgs a = {};
    a.grad = n.grad_dev;
    a.h = n.h_dev;
    a.mean = n.mean_dev;
    a.rstd = n.rstd_dev;
    a.weight = n.weight_dev;
    a.past = n.past_dev;
    a.grad_x = n.grad_x_dev;
    a.grad_weight = n.grad_weight_dev;
    a.grad_bias = n.grad_bias_dev;
    a.grad_stride = n.grad_stride;
    a.h_stride = n.h_stride;
    a.past_stride = n.past_stride;
    a.grad_x_stride = n.grad_x_stride;
    a.rows = n.rows;
    a.d = n.d;
    a.wide = (n.d + 7u) / 8u * 8u;
    a.grad_bf16 = n.grad_dtype == LILY_BF16;
    a.h_bf16 = n.h_dtype == LILY_BF16;
    a.weight_bf16 = n.weight_dtype == LILY_BF16;
    a.grad_x_bf16 = n.grad_x_dtype == LILY_BF16;
    a.accumulate = n.accumulate;
    a.part = ws.part;
    // (the columns' sums first: grad_x may lie where an operand lies)
    if (n.grad_weight_dev != nullptr || n.grad_bias_dev != nullptr) {
        const uint32_t strips = (n.d + 511u) / 512u;
        a.parts = std::min({(n.rows + 3u) / 4u, (2048u + strips - 1u) / strips, (uint32_t)(ws.part_floats / (2ull * a.wide))});
        if (n.d % 8u != 0u) {
            hipLaunchKernelGGL(k_layer_columns<true>, dim3(strips, a.parts), dim3(256), 0, stream, a);
        } else {
            hipLaunchKernelGGL(k_layer_columns<false>, dim3(strips, a.parts), dim3(256), 0, stream, a);
        }
        hipLaunchKernelGGL(k_layer_join, dim3((n.d + 31u) / 32u, 2), dim3(256), 0, stream, a);
    }
    if (n.grad_x_dev != nullptr) {
        const NormShape shape = norm_shape(n.d);
        const dim3 grid(n.rows), block(shape.threads);
#define LILY_LAYER(CH)                                                             \
    if (n.d % 8u != 0u) {                                                          \
        hipLaunchKernelGGL((k_layer_grad<CH, true>), grid, block, 0, stream, a);   \
    } else {                                                                       \
        hipLaunchKernelGGL((k_layer_grad<CH, false>), grid, block, 0, stream, a);  \
    }
        if (shape.pieces == 1u) {
            LILY_LAYER(1)
        } else if (shape.pieces == 2u) {
            LILY_LAYER(2)
        } else {
            LILY_LAYER(4)
        }
#undef LILY_LAYER
    }
    return hipGetLastError();
}

}  // namespace lily
