// project_blocks.hip - the matrix product of 8-bit floats with a scale for each block of 128, and an epilogue.
//
//     out[r][v] = residual[r][v] + act(sum_b xs[r][b] ws[v / 128][b] sum_{i in b} x[r][i] w[v][i] + bias[v])
//
// The kernels are the plain product's (project_few.hip, project_tile.h): what they take of a row at a time, 128 bytes, is
// one block.  Its products are summed on the matrix cores from zero, and the sum joins the tile's by a multiplication
// with both scales and an addition in f32.  The scales of x arrive in LDS beside the rows they belong to, those of
// the weights are one a wave and line.
#include "project_tile.h"

namespace lily {

namespace {

template <Products P, class T>
hipError_t launch_tile_of(hipStream_t stream, const ProjectArgs& a) {
    const uint32_t m_tiles = (a.rows + T::BM - 1u) / T::BM, n_tiles = (a.n + T::BN - 1u) / T::BN;
    static LdsAllowed allowed;
    if (const hipError_t e = allowed.say((const void*)k_project_tiles<P, T>, T::LDS_BYTES); e != hipSuccess) {
        return e;
    }
    hipLaunchKernelGGL((k_project_tiles<P, T>), dim3(m_tiles * n_tiles * a.splits), dim3(64 * T::WAVES), T::LDS_BYTES, stream, a, m_tiles, n_tiles);
    return a.splits > 1u ? launch_project_join(stream, a) : hipGetLastError();
}
template <class T>
hipError_t launch_tile(hipStream_t stream, const ProjectArgs& a) {
    return a.out_bf16 ? launch_tile_of<PRODUCT_BLOCKS, T>(stream, a) : launch_tile_of<PRODUCT_BLOCKS_WIDE, T>(stream, a);
}

}  // namespace

hipError_t launch_project_blocks(hipStream_t stream, const lily_block_projection& b, const ProjectWorkspace& given) {
    lily_projection p = {};
    p.rows = b.rows;
    p.n = b.n;
    p.d = b.d;
    p.dtype = LILY_E4M3;
    p.x_dev = b.x_dev;
    p.x_stride = b.x_stride;
    p.weight_dev = b.weight_dev;
    p.weight_stride = b.weight_stride;
    p.bias_dev = b.bias_dev;
    p.residual_dev = b.residual_dev;
    p.residual_stride = b.residual_stride;
    p.out_dev = b.out_dev;
    p.out_stride = b.out_stride;
    p.bias_dtype = b.bias_dtype;
    p.residual_dtype = b.residual_dtype;
    p.out_dtype = b.out_dtype;
    p.activation = b.activation;
    ProjectWorkspace ws = given;
    ws.tile = ws.tile == 256u ? 0u : ws.tile;
    ProjectArgs a = project_args(p, ws);
    a.x_blocks = b.x_scales_dev;
    a.w_blocks = b.weight_scales_dev;
    a.x_blocks_stride = b.rows > 1u ? (uint32_t)b.x_scales_stride : 0u;
    a.w_blocks_stride = b.n > LILY_BLOCK ? (uint32_t)b.weight_scales_stride : 0u;
    ProjectPlan plan = project_plan(a, ws);
    if (plan.tile == 256u) {
        plan = {128u, 1u};
    }
    a.splits = plan.splits;
    return plan.tile == 0u    ? launch_project_few(stream, a, PRODUCT_BLOCKS_WIDE)
           : plan.tile == 64u ? launch_tile<Tile<16, 2, 2, 2, 2, 2, 4, true>>(stream, a)
                              : launch_tile<Tile<16, 2, 2, 4, 4, 2, 2, true>>(stream, a);
}

}  // namespace lily
