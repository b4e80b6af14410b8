// layer_norm.hip - the residual's addition with the layer norm, and its backward pass.
//
//     h = x + residual (rounded to the stream's type),  y = (h - mean) / sqrt(var + eps) * w + b
//
// One workgroup per row: a thread keeps its part of the row in registers through both sums (the values', then that of the
// squared distances from their mean, which does not cancel) and the outputs, so a row is read once and written once.  A
// block of 128 elements with a scale of its own is a row of 16 lanes: its largest value takes no memory and no barrier.
//
// Bound by memory: 8192 x 4096, bf16 rows, residual and sum, E4M3 blocks, 52 to 55 us (4.3 to 4.5 TB/s; the RMS norm to E4M3 rows the same on
// the same chip).  4 rows 4.5 us, a launch, a trip to memory and two sums.  Rows of more than 16 384 elements, four pieces a thread with all their
// operands, spill 49 registers (74 where they are no multiple of 8 long).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "launch.h"
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

// Both at once, for rows of 8 to 8192 elements: a workgroup takes `groups` rows at a time, `threads` threads and eight elements a
// thread each, and keeps what its rows add to the gradients of weight and bias in registers; the next rows (in bf16 the next
// two) are on their way while a row's two sums go through LDS.  So grad and h are read once: 16 384 x 4096 in bf16 with `past` 104 us
// and 4 of joining 256 workgroups' parts (537 MB, 5.0 TB/s) against 161 by the two kernels below, which read them twice; 2049 x 2560 in
// f32 17 + 4 against 43, of which the memory's are 11: three turns of three rows a workgroup, each a barrier, its stores and, since f32 has
// registers for one turn ahead, a trip to memory (120 to 126 of 128; of bf16's whole rows one is spilled).
// Rows of 4001, 8000 of them in bf16 with `past`, 65 us (134 where the piece that a row ends in was read an element at a time).
// Longer rows go by k_layer_grad_long or by those two, calls for one of the outputs alone by those two.
enum LayerTypes { LAYER_F32, LAYER_BF16, LAYER_MIXED };   // of grad, h, past and grad_x
template <int TYPES>
struct LayerPiece : Eight<TYPES == LAYER_BF16> {
    __device__ __forceinline__ void ask(const void* row, uint32_t i, bool) { this->load(row, i); }
    __device__ __forceinline__ void take(bool, float (&v)[8]) const { this->widened(v); }
};
template <>
struct LayerPiece<LAYER_MIXED> {
    Raw raw;
    __device__ __forceinline__ void ask(const void* row, uint32_t i, bool bf16) { raw = load8(row, i, bf16); }
    __device__ __forceinline__ void take(bool bf16, float (&v)[8]) const { widen(raw, bf16, v); }
};
// The piece that a row of d elements ends in: of the row's last eight elements, which stand in v, the last ones.
__device__ __forceinline__ void ends_in(uint32_t d, float (&v)[8]) {
    const uint32_t shift = 8u - d % 8u;
    const bool one = (shift & 1u) != 0u, two = (shift & 2u) != 0u, four = (shift & 4u) != 0u;
#pragma unroll
    for (int j = 0; j < 7; ++j) {
        const float here = v[j], behind = v[j + 1];
        v[j] = one ? behind : here;
    }
#pragma unroll
    for (int j = 0; j < 6; ++j) {
        const float here = v[j], behind = v[j + 2];
        v[j] = two ? behind : here;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float here = v[j], behind = v[j + 4];
        v[j] = four ? behind : here;
    }
}
template <bool RAGGED, int TYPES>
__global__ void __launch_bounds__(1024) k_layer_grad_all(const LayerGradArgs a, uint32_t threads, uint32_t groups) {
    constexpr uint32_t AHEAD = TYPES == LAYER_BF16 ? 2u : 1u;   // (registers)
    __shared__ float part[2][2][16];
    extern __shared__ float share[];   // [groups - 1][16][threads]
    const uint32_t tid = threadIdx.x;
    const uint32_t group = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid / threads)), in_row = tid - group * threads, i = in_row * 8u;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6)), from = group * (threads >> 6), to = from + (threads >> 6);   // waves of the group
    const bool whole = i + 8u <= a.d;
    const bool grad_bf16 = TYPES == LAYER_MIXED ? a.grad_bf16 != 0u : TYPES == LAYER_BF16, h_bf16 = TYPES == LAYER_MIXED ? a.h_bf16 != 0u : grad_bf16,
               x_bf16 = TYPES == LAYER_MIXED ? a.grad_x_bf16 != 0u : grad_bf16;
    struct Next {
        LayerPiece<TYPES> grad, h, past;
        float mean, rstd;
    } next[AHEAD];
    // (what lies behind the last whole piece of a row is not asked for; the loads of grad and h stand outside of every branch)
    const uint32_t at = min(i, a.d - 8u);
    auto ask = [&](Next& n, uint64_t row) {
        const uint64_t r = min(row, (uint64_t)a.rows - 1u);
        n.grad.ask(row_at(a.grad, r, a.grad_stride, grad_bf16), at, grad_bf16);
        n.h.ask(row_at(a.h, r, a.h_stride, h_bf16), at, h_bf16);
        if (a.past != nullptr) {
            n.past.ask(row_at(a.past, r, a.past_stride, x_bf16), at, x_bf16);
        }
        n.mean = gload(a.mean + r);
        n.rstd = gload(a.rstd + r);
    };
    auto take = [&](const LayerPiece<TYPES>& piece, bool bf16, float (&v)[8]) {
        piece.take(bf16, v);
        if (RAGGED && !whole) {
            ends_in(a.d, v);
        }
    };
    const uint64_t step = (uint64_t)gridDim.x * groups;
    uint64_t row = (uint64_t)blockIdx.x * groups + group;
#pragma unroll
    for (uint32_t q = 0; q < AHEAD; ++q) {
        ask(next[q], row + q * step);
    }
    float w[8], gw[8] = {}, gb[8] = {};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        w[j] = a.weight != nullptr && i + (uint32_t)j < a.d ? load1(a.weight, i + (uint32_t)j, a.weight_bf16) : 1.0f;
    }
    const float over_d = 1.0f / (float)a.d;
    auto one = [&](Next& n, uint32_t turn) {
        const bool there = row < a.rows && (RAGGED || whole);   // (a piece behind the row's end is nothing)
        const float mean = n.mean, rstd = n.rstd;
        float g[8], x[8], past[8], sg = 0.0f, sx = 0.0f;
        take(n.grad, grad_bf16, g);
        take(n.h, h_bf16, x);
        if (a.past != nullptr) {
            take(n.past, x_bf16, past);
        }
        ask(n, row + AHEAD * step);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool in = there && (!RAGGED || i + (uint32_t)j < a.d);
            g[j] = in ? g[j] : 0.0f;
            x[j] = in ? (x[j] - mean) * rstd : 0.0f;
            gb[j] += g[j];
            gw[j] = __builtin_fmaf(g[j], x[j], gw[j]);
            g[j] *= w[j];
            sg += g[j];
            sx = __builtin_fmaf(g[j], x[j], sx);
        }
        sg = wave_sum_f(sg);
        sx = wave_sum_f(sx);
        if ((tid & 63u) == 0u) {
            part[turn][0][wave] = sg;
            part[turn][1][wave] = sx;
        }
        __syncthreads();
        sg = sx = 0.0f;
        for (uint32_t q = from; q < to; ++q) {
            sg += part[turn][0][q];
            sx += part[turn][1][q];
        }
        sg *= over_d;
        sx *= over_d;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float v = rstd * (g[j] - sg - x[j] * sx);
            g[j] = a.past != nullptr ? v + past[j] : v;
        }
        char* out = const_cast<char*>(row_at(a.grad_x, row, a.grad_x_stride, x_bf16));
        if (there && whole) {
            if (x_bf16) {
                store8(out, i, g, LILY_BF16);
            } else {
                store8(out, i, g, LILY_F32);
            }
        } else if (RAGGED && there) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (i + (uint32_t)j < a.d) {
                    store1(out, i + (uint32_t)j, g[j], x_bf16 ? LILY_BF16 : LILY_F32);
                }
            }
        }
        row += step;
    };
    if constexpr (AHEAD == 2u) {
        // (two turns at a time: the registers of what comes next take turns; a turn behind the last row adds nothing)
        for (uint64_t first = (uint64_t)blockIdx.x * groups; first < a.rows; first += 2u * step) {
            one(next[0], 0u);
            __builtin_amdgcn_sched_barrier(0);
            one(next[AHEAD - 1u], 1u);
            __builtin_amdgcn_sched_barrier(0);
        }
    } else {
        uint32_t turn = 0u;
        for (uint64_t first = (uint64_t)blockIdx.x * groups; first < a.rows; first += step, turn ^= 1u) {
            one(next[0], turn);
        }
    }
    if (group != 0u) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            share[((group - 1u) * 16u + (uint32_t)j) * threads + in_row] = gw[j];
            share[((group - 1u) * 16u + 8u + (uint32_t)j) * threads + in_row] = gb[j];
        }
    }
    __syncthreads();
    if (group == 0u && i < a.wide) {
        float* out = a.part + (uint64_t)blockIdx.x * 2u * a.wide + i;
        for (uint32_t q = 0; q + 1u < groups; ++q) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                gw[j] += share[(q * 16u + (uint32_t)j) * threads + in_row];
                gb[j] += share[(q * 16u + 8u + (uint32_t)j) * threads + in_row];
            }
        }
        if (gridDim.x != 1u) {
            store8(out, 0u, gw, LILY_F32);
            store8(out + a.wide, 0u, gb, LILY_F32);
            return;
        }
        // (nothing to join: 1 x 140 9.7 us, 12.5 by another launch)
        auto give = [&](float* to, const float (&v)[8]) {
            if (to != nullptr) {
#pragma unroll
                for (uint32_t j = 0; j < 8u; ++j) {
                    if (i + j < a.d) {
                        to[i + j] = a.accumulate != 0u ? to[i + j] + v[j] : v[j];
                    }
                }
            }
        };
        give(a.grad_weight, gw);
        give(a.grad_bias, gb);
    }
}

// The same for rows of up to 16 384 elements: a row a workgroup, two pieces a thread, whose sums over the rows lie in LDS, 128 bytes a
// thread.  `past` is asked for when its row's turn comes.  3068 x 10 336 in bf16 with `past` 81 us against 94.5 by the two kernels below,
// 3000 x 12 345 115 against 132, 2000 x 16 384 in f32 114 against 145, with `past` 141 against 157.  That is with 13 registers spilled in bf16 and 23 in
// f32 (56 and 96 bytes a lane).  Rows of f32 that are no multiple of 8 long, and of mixed types, spill more than one reading saves and go by those
// two: 2000 x 14 835 in f32 192 so, 155 by them; mixed 3451 x 14 835 324 and 227.
constexpr uint32_t LONG_THREADS = 1024, LONG_PIECES = 2, LONG_LDS = LONG_THREADS * LONG_PIECES * 64;
template <bool RAGGED, bool BF16>
__global__ void __launch_bounds__(LONG_THREADS) k_layer_grad_long(const LayerGradArgs a) {
    __shared__ float part[2][2][16];
    extern __shared__ f32x4 long_sums[];   // [pieces][weight's, bias's][halves][threads]
    const uint32_t tid = threadIdx.x, wave = tid >> 6;
    uint32_t i[LONG_PIECES], at[LONG_PIECES];
    bool whole[LONG_PIECES];
#pragma unroll
    for (uint32_t c = 0; c < LONG_PIECES; ++c) {
        i[c] = (c * LONG_THREADS + tid) * 8u;
        whole[c] = i[c] + 8u <= a.d;
        at[c] = min(i[c], a.d - 8u);
#pragma unroll
        for (uint32_t q = 0; q < 4u; ++q) {
            long_sums[(c * 4u + q) * LONG_THREADS + tid] = f32x4(0.0f);
        }
    }
    Eight<BF16> grad[LONG_PIECES], h[LONG_PIECES];
    float next_mean, next_rstd;
    auto ask = [&](uint64_t row) {
        const uint64_t r = min(row, (uint64_t)a.rows - 1u);
#pragma unroll
        for (uint32_t c = 0; c < LONG_PIECES; ++c) {
            grad[c].load(row_at(a.grad, r, a.grad_stride, BF16), at[c]);
            h[c].load(row_at(a.h, r, a.h_stride, BF16), at[c]);
        }
        next_mean = gload(a.mean + r);
        next_rstd = gload(a.rstd + r);
    };
    auto take = [&](const Eight<BF16>& piece, uint32_t c, float (&v)[8]) {
        piece.widened(v);
        if (RAGGED && !whole[c]) {
            ends_in(a.d, v);
        }
    };
    const float over_d = 1.0f / (float)a.d;
    ask(blockIdx.x);
    uint32_t turn = 0u;
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1u) {
        float g[LONG_PIECES][8], x[LONG_PIECES][8], sg = 0.0f, sx = 0.0f;
        const float mean = next_mean, rstd = next_rstd;
        Eight<BF16> past[LONG_PIECES];
        Raw weight[LONG_PIECES];   // (from the L2)
#pragma unroll
        for (uint32_t c = 0; c < LONG_PIECES; ++c) {
            take(grad[c], c, g[c]);
            take(h[c], c, x[c]);
            if (a.weight != nullptr) {
                weight[c] = load8(a.weight, at[c], a.weight_bf16);
            }
        }
        if (a.past != nullptr) {
#pragma unroll
            for (uint32_t c = 0; c < LONG_PIECES; ++c) {
                past[c].load(row_at(a.past, row, a.past_stride, BF16), at[c]);
            }
        }
        ask(row + gridDim.x);
#pragma unroll
        for (uint32_t c = 0; c < LONG_PIECES; ++c) {
            float w[8] = {};
            if (a.weight != nullptr) {
                widen(weight[c], a.weight_bf16, w);
                if (RAGGED && !whole[c]) {
                    ends_in(a.d, w);
                }
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                f32x4& gw = long_sums[(c * 4u + (uint32_t)half) * LONG_THREADS + tid];
                f32x4& gb = long_sums[(c * 4u + 2u + (uint32_t)half) * LONG_THREADS + tid];
                f32x4 new_gw = gw, new_gb = gb;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int j = half * 4 + e;
                    const bool in = RAGGED ? i[c] + (uint32_t)j < a.d : whole[c];   // (a piece behind the row's end is nothing)
                    g[c][j] = in ? g[c][j] : 0.0f;
                    x[c][j] = in ? (x[c][j] - mean) * rstd : 0.0f;
                    new_gb[e] += g[c][j];
                    new_gw[e] = __builtin_fmaf(g[c][j], x[c][j], new_gw[e]);
                    g[c][j] *= a.weight != nullptr && in ? w[j] : 1.0f;
                    sg += g[c][j];
                    sx = __builtin_fmaf(g[c][j], x[c][j], sx);
                }
                gw = new_gw;
                gb = new_gb;
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        sg = wave_sum_f(sg);
        sx = wave_sum_f(sx);
        if ((tid & 63u) == 0u) {
            part[turn][0][wave] = sg;
            part[turn][1][wave] = sx;
        }
        if (RAGGED && a.past != nullptr) {   // (a piece that lies over its neighbour's has to be there before that is stored)
            __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
        }
        __syncthreads();
        sg = sx = 0.0f;
        for (uint32_t q = 0; q < LONG_THREADS / 64u; ++q) {
            sg += part[turn][0][q];
            sx += part[turn][1][q];
        }
        sg *= over_d;
        sx *= over_d;
        char* out = const_cast<char*>(row_at(a.grad_x, row, a.grad_x_stride, BF16));
#pragma unroll
        for (uint32_t c = 0; c < LONG_PIECES; ++c) {
            float v[8] = {};
            if (a.past != nullptr) {
                take(past[c], c, v);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float own = rstd * (g[c][j] - sg - x[c][j] * sx);
                v[j] = a.past != nullptr ? own + v[j] : own;
            }
            if (whole[c]) {
                store8(out, i[c], v, BF16 ? LILY_BF16 : LILY_F32);
            } else if (RAGGED) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (i[c] + (uint32_t)j < a.d) {
                        store1(out, i[c] + (uint32_t)j, v[j], BF16 ? LILY_BF16 : LILY_F32);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
#pragma unroll
    for (uint32_t c = 0; c < LONG_PIECES; ++c) {
        if (i[c] < a.wide) {
            float* out = a.part + (uint64_t)blockIdx.x * 2u * a.wide + i[c];
#pragma unroll
            for (uint32_t half = 0; half < 2u; ++half) {
                *reinterpret_cast<f32x4*>(out + half * 4u) = long_sums[(c * 4u + half) * LONG_THREADS + tid];
                *reinterpret_cast<f32x4*>(out + a.wide + half * 4u) = long_sums[(c * 4u + 2u + half) * LONG_THREADS + tid];
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
#pragma unroll 8
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

template <bool RAGGED, bool BF16>
hipError_t launch_long(hipStream_t stream, const LayerGradArgs& a) {
    static LdsAllowed allowed;
    if (const hipError_t e = allowed.say((const void*)k_layer_grad_long<RAGGED, BF16>, LONG_LDS); e != hipSuccess) {
        return e;
    }
    hipLaunchKernelGGL((k_layer_grad_long<RAGGED, BF16>), dim3(a.parts), dim3(LONG_THREADS), LONG_LDS, stream, a);
    return hipGetLastError();
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
    const bool sums = n.grad_weight_dev != nullptr || n.grad_bias_dev != nullptr;
    auto join = [&] { hipLaunchKernelGGL(k_layer_join, dim3((n.d + 31u) / 32u, 2), dim3(256), 0, stream, a); };
    const bool mixed = a.grad_bf16 != a.h_bf16 || a.grad_bf16 != a.grad_x_bf16, ragged = n.d % 8u != 0u;
    if (sums && n.grad_x_dev != nullptr && n.d >= 8u && n.d <= 8192u) {
        const uint32_t threads = norm_shape(n.d).threads, groups = 1024u / threads;
        a.parts = std::min({(n.rows + groups - 1u) / groups, 256u, (uint32_t)(ws.part_floats / (2ull * a.wide))});
        const uint32_t lds = (groups - 1u) * 16u * threads * 4u;
#define LILY_LAYER(RAGGED, TYPES) \
    hipLaunchKernelGGL((k_layer_grad_all<RAGGED, TYPES>), dim3(a.parts), dim3(threads * groups), lds, stream, a, threads, groups)
        if (mixed && ragged) {
            LILY_LAYER(true, LAYER_MIXED);
        } else if (mixed) {
            LILY_LAYER(false, LAYER_MIXED);
        } else if (a.grad_bf16 != 0u && ragged) {
            LILY_LAYER(true, LAYER_BF16);
        } else if (a.grad_bf16 != 0u) {
            LILY_LAYER(false, LAYER_BF16);
        } else if (ragged) {
            LILY_LAYER(true, LAYER_F32);
        } else {
            LILY_LAYER(false, LAYER_F32);
        }
#undef LILY_LAYER
        if (a.parts > 1u) {
            join();
        }
        return hipGetLastError();
    }
    if (sums && n.grad_x_dev != nullptr && !mixed && (a.grad_bf16 != 0u || !ragged) && n.d > 8192u && n.d <= LONG_THREADS * LONG_PIECES * 8u) {
        a.parts = std::min({n.rows, 256u, (uint32_t)(ws.part_floats / (2ull * a.wide))});
        const hipError_t e = a.grad_bf16 == 0u ? launch_long<false, false>(stream, a)
                             : ragged          ? launch_long<true, true>(stream, a)
                                               : launch_long<false, true>(stream, a);
        if (e != hipSuccess) {
            return e;
        }
        join();
        return hipGetLastError();
    }
    // (the columns' sums first: grad_x may lie where an operand lies)
    if (sums) {
        const uint32_t strips = (n.d + 511u) / 512u;
        a.parts = std::min({(n.rows + 3u) / 4u, (2048u + strips - 1u) / strips, (uint32_t)(ws.part_floats / (2ull * a.wide))});
        if (n.d % 8u != 0u) {
            hipLaunchKernelGGL(k_layer_columns<true>, dim3(strips, a.parts), dim3(256), 0, stream, a);
        } else {
            hipLaunchKernelGGL(k_layer_columns<false>, dim3(strips, a.parts), dim3(256), 0, stream, a);
        }
        join();
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
