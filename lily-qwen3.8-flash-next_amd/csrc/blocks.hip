// blocks.hip - a matrix in 8-bit floats with a scale for each 128 elements of a row or each 128 x 128.
//
//     scale = max|x| / 448,  q = E4M3(x / scale)
//
// A lane holds eight neighbouring elements, so 16 lanes hold 128 of a row; values stay in registers between the largest
// one's search and the outputs: read once, written once, bound by memory: 12 288 x 4096 in f32, a scale for 128 x 128, 47 us (5.4 TB/s).
// 61 rows of 2560 3.6 us, a launch and a trip to memory.
#include <hip/hip_runtime.h>

#include "operators.h"
#include "row_pieces.h"

namespace lily {

namespace {

struct BlocksArgs {
    const void* x;
    uint8_t* out;
    float* scales;
    uint64_t x_stride, out_stride, scales_stride;   // elements
    uint32_t rows, d, across, blocks;               // blocks a row, and in all
    uint32_t x_bf16;
};

// Eight elements of a row from i on, zeros behind its end.
__device__ __forceinline__ void eight_at(const BlocksArgs& a, uint64_t row, uint32_t i, float (&v)[8]) {
    const char* x = static_cast<const char*>(a.x) + row * a.x_stride * (a.x_bf16 ? 2u : 4u);
    if (i + 8u <= a.d) {
        widen(load8(x, i, a.x_bf16), a.x_bf16, v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = i + (uint32_t)j < a.d ? load1(x, i + (uint32_t)j, a.x_bf16) : 0.0f;
        }
    }
}
__device__ __forceinline__ uint32_t top_of(const float (&v)[8]) {
    uint32_t top = 0u;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        top = max(top, lilym_f32_bits(v[j]) & 0x7fffffffu);
    }
    return top;
}
__device__ __forceinline__ void give(const BlocksArgs& a, uint64_t row, uint32_t i, const float (&v)[8], float inverse) {
    float q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        q[j] = v[j] * inverse;
    }
    uint8_t* out = a.out + row * a.out_stride;
    if (i + 8u <= a.d) {
        store8(out, i, q, LILY_E4M3);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (i + (uint32_t)j < a.d) {
                store1(out, i + (uint32_t)j, q[j], LILY_E4M3);
            }
        }
    }
}

__global__ void __launch_bounds__(256) k_quantize_rows(const BlocksArgs a) {
    const uint32_t block = blockIdx.x * 16u + (threadIdx.x >> 4), in = threadIdx.x & 15u;
    const uint32_t row = min(block, a.blocks - 1u) / a.across, b = min(block, a.blocks - 1u) % a.across;
    float v[8];
    eight_at(a, row, b * LILY_BLOCK + in * 8u, v);
    const Scale8 by = scale_of(sixteen_max_u32(top_of(v)));
    if (block < a.blocks) {
        give(a, row, b * LILY_BLOCK + in * 8u, v, by.inverse);
        if (in == 0u) {
            a.scales[row * a.scales_stride + b] = by.scale;
        }
    }
}

__global__ void __launch_bounds__(256) k_quantize_tiles(const BlocksArgs a) {
    __shared__ uint32_t part[4];
    const uint32_t down = blockIdx.x / a.across, b = blockIdx.x % a.across, in = threadIdx.x & 15u;
    const uint32_t row0 = down * LILY_BLOCK + (threadIdx.x >> 4), i = b * LILY_BLOCK + in * 8u;
    float v[8][8];
    uint32_t top = 0u;
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        eight_at(a, min(row0 + t * 16u, a.rows - 1u), i, v[t]);   // (the last row again: its values count in the block already)
    }
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        top = max(top, top_of(v[t]));
    }
    top = wave_max_u32(top);
    if ((threadIdx.x & 63u) == 0u) {
        part[threadIdx.x >> 6] = top;
    }
    __syncthreads();
    top = max(max(part[0], part[1]), max(part[2], part[3]));
    const Scale8 by = scale_of(top);
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        if (row0 + t * 16u < a.rows) {
            give(a, row0 + t * 16u, i, v[t], by.inverse);
        }
    }
    if (threadIdx.x == 0u) {
        a.scales[down * a.scales_stride + b] = by.scale;
    }
}

}  // namespace

hipError_t launch_quantize_blocks(hipStream_t stream, const lily_blocks& q) {
    BlocksArgs a = {};
    a.x = q.x_dev;
    a.out = static_cast<uint8_t*>(q.out_dev);
    a.scales = q.scales_dev;
    a.x_stride = q.x_stride;
    a.out_stride = q.out_stride;
    a.scales_stride = q.scales_stride;
    a.rows = q.rows;
    a.d = q.d;
    a.across = (q.d + LILY_BLOCK - 1u) / LILY_BLOCK;
    a.x_bf16 = q.x_dtype == LILY_BF16;
    if (q.block_rows == 1u) {
        a.blocks = q.rows * a.across;
        hipLaunchKernelGGL(k_quantize_rows, dim3((a.blocks + 15u) / 16u), dim3(256), 0, stream, a);
    } else {
        a.blocks = (q.rows + LILY_BLOCK - 1u) / LILY_BLOCK * a.across;
        hipLaunchKernelGGL(k_quantize_tiles, dim3(a.blocks), dim3(256), 0, stream, a);
    }
    return hipGetLastError();
}

}  // namespace lily
