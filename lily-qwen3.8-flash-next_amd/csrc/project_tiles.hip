// project_tiles.hip - the matrix product with an epilogue for more rows (project_tile.h), in bf16 and E4M3 with a scale a row,
// and the join of the parts of d.
//
// Measured (cycles of a 256 x 256 tile, 8192 x 4096 x 4096 in bf16): 4 300 until the first stage is there, 146 000 for 64
// stages, of which the matrix pipe is busy 131 000, and the epilogue, in which all compute units write at once.  212 to 224 us by
// the box, 1.30 to 1.23 PFLOP/s, at 1.8 GHz (the clock follows the power the products take; a large library product runs at
// 1.59 PFLOP/s); with a bf16 residual 236, with bias, SiLU and residual 245 to 253; 8192 x 8192 x 8192 774 to 808 us, 1.42 to 1.36;
// 8192 x 12 288 x 4096 in E4M3 340 us, 2.43 (3.21), widened for an f32 output 685.
#include "project_tile.h"

namespace lily {

namespace {

// The parts of d joined: a thread adds four neighbouring outputs of a row over the parts, in order, and finishes them.
__global__ void __launch_bounds__(256) k_project_join(const ProjectArgs a) {
    const uint32_t fours = part_stride(a.n) / 4u;
    const uint64_t at = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    if (at >= (uint64_t)fours * a.rows) {
        return;
    }
    const uint32_t r = (uint32_t)(at / fours), v = (uint32_t)(at % fours) * 4u;
    Columns c;
    Finish f;
    c.load(a, v);
    f.load(a, r, v);
    const float* from = a.part + (uint64_t)r * part_stride(a.n) + v;
    const uint64_t next = (uint64_t)a.rows * part_stride(a.n);
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t q = 0; q < a.splits; q += 4u) {
        f32x4 p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            p[j] = gload(reinterpret_cast<const f32x4*>(from + min(q + (uint32_t)j, a.splits - 1u) * next));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (q + (uint32_t)j < a.splits) {
                sum += p[j];
            }
        }
    }
    f.store(a, r, v, c, sum);
}

template <class T>
hipError_t launch_tile(hipStream_t stream, const ProjectArgs& a, bool e4m3) {
    const uint32_t m_tiles = (a.rows + T::BM - 1u) / T::BM, n_tiles = (a.n + T::BN - 1u) / T::BN;
    const dim3 grid(m_tiles * n_tiles * a.splits), block(256);
    auto go = [&](const void* kernel, LdsAllowed& allowed, auto launch) -> hipError_t {
        const hipError_t e = allowed.say(kernel, T::LDS_BYTES);
        if (e == hipSuccess) {
            launch();
        }
        return e;
    };
    static LdsAllowed allowed[3];
    hipError_t e;
    if (!e4m3) {
        e = go((const void*)k_project_tiles<PRODUCT_BF16, T>, allowed[0], [&] {
            hipLaunchKernelGGL((k_project_tiles<PRODUCT_BF16, T>), grid, block, T::LDS_BYTES, stream, a, m_tiles, n_tiles);
        });
    } else if (a.out_bf16) {
        e = go((const void*)k_project_tiles<PRODUCT_E4M3, T>, allowed[1], [&] {
            hipLaunchKernelGGL((k_project_tiles<PRODUCT_E4M3, T>), grid, block, T::LDS_BYTES, stream, a, m_tiles, n_tiles);
        });
    } else {
        e = go((const void*)k_project_tiles<PRODUCT_E4M3_WIDE, T>, allowed[2], [&] {
            hipLaunchKernelGGL((k_project_tiles<PRODUCT_E4M3_WIDE, T>), grid, block, T::LDS_BYTES, stream, a, m_tiles, n_tiles);
        });
    }
    if (e != hipSuccess) {
        return e;
    }
    return a.splits > 1u ? launch_project_join(stream, a) : hipGetLastError();
}

}  // namespace

hipError_t launch_project_join(hipStream_t stream, const ProjectArgs& a) {
    const uint64_t threads = (uint64_t)a.rows * (part_stride(a.n) / 4u);
    hipLaunchKernelGGL(k_project_join, dim3((uint32_t)((threads + 255u) / 256u)), dim3(256), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_project_tiles(hipStream_t stream, const ProjectArgs& a, bool e4m3, uint32_t tile) {
    return tile == 256u   ? launch_tile<Tile<32, 2, 2, 4, 4, 1, 2>>(stream, a, e4m3)
           : tile == 128u ? launch_tile<Tile<16, 2, 2, 4, 4, 2, 2>>(stream, a, e4m3)
                          : launch_tile<Tile<16, 2, 2, 2, 2, 2, 4>>(stream, a, e4m3);
}

}  // namespace lily
