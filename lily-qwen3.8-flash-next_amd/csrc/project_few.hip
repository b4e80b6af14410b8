// project_few.hip - the matrix product with an epilogue for up to 16 rows: the weights are read once at
// the speed of memory, the matrix cores idle.
//
// A workgroup takes 16 outputs' weight rows; its waves share d, a run of whole lines (128 bytes a row)
// each, so that a layer of a few thousand outputs already keeps every compute unit's memory path busy without
// a join between workgroups.  A wave asks for its lines straight into the registers the product takes them
// from, AHEAD of them at a time (16 rows x 64 bytes an instruction, the line's other half with the next).
// The waves' sums meet in LDS.
#include "project.h"

namespace lily {

namespace {

constexpr int FEW_AHEAD = 8;   // lines of a wave in flight

template <Products P>
__global__ void __launch_bounds__(512) k_project_few(const ProjectArgs a) {
    extern __shared__ __align__(16) char lds[];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, waves = blockDim.x >> 6;
    const uint32_t g = lane >> 4, r = lane & 15u, v0 = blockIdx.x * 16u;
    const uint32_t lines = (a.d_bytes + LINE - 1u) / LINE;
    const uint32_t per = (lines + waves - 1u) / waves, from = min(wave * per, lines), to = min(from + per, lines);
    const char* w = a.w + (uint64_t)min(v0 + r, a.n - 1u) * a.w_stride;
    const char* x = a.x + (uint64_t)min(r, a.rows - 1u) * a.x_stride;
    // (a row beyond the last is the last one's values: its sums go nowhere)
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    auto piece = [&](const char* row, uint32_t at) -> u32x4 {
        // beyond d: zeros, in both operands (what lies behind a row may be anything)
        const u32x4 p = gload(reinterpret_cast<const u32x4*>(row + min(at, a.d_bytes - 16u)));
        return at < a.d_bytes ? p : u32x4{0u, 0u, 0u, 0u};
    };
    for (uint32_t l0 = from; l0 < to; l0 += FEW_AHEAD) {
        Frag fw[FEW_AHEAD], fx[FEW_AHEAD];
#pragma unroll
        for (int u = 0; u < FEW_AHEAD; ++u) {
            // (a line past the wave's last is its last again, and its product is left out)
            const uint32_t at = min(l0 + (uint32_t)u, to - 1u) * LINE + g * 16u;
            fw[u].lo = piece(w, at);
            fw[u].hi = piece(w, at + 64u);
            fx[u].lo = piece(x, at);
            fx[u].hi = piece(x, at + 64u);
        }
#pragma unroll
        for (int u = 0; u < FEW_AHEAD; ++u) {
            if (l0 + (uint32_t)u < to) {
                acc = product<P>(fw[u], fx[u], acc);
            }
        }
    }
    f32x4* sums = reinterpret_cast<f32x4*>(lds);
    if (waves > 1u) {
        if (wave != 0u) {
            sums[(wave - 1u) * 64u + lane] = acc;
        }
        __syncthreads();
        if (wave != 0u) {
            return;
        }
        for (uint32_t q = 0; q + 1u < waves; ++q) {
            acc += sums[q * 64u + lane];
        }
    }
    if (r < a.rows) {
        const uint32_t v = v0 + g * 4u;
        finish(a, r, v, columns_at(a, v), a.x_scales != nullptr ? gload(a.x_scales + r) : 1.0f, acc);
    }
}

}  // namespace

hipError_t launch_project_few(hipStream_t stream, const ProjectArgs& a, bool e4m3) {
    const uint32_t lines = (a.d_bytes + LINE - 1u) / LINE;
    uint32_t waves = 1;
    while (waves < 8u && waves * (uint32_t)FEW_AHEAD < lines) {
        waves *= 2u;
    }
    const dim3 grid((a.n + 15u) / 16u), block(waves * 64u);
    const size_t lds = (size_t)(waves - 1u) * 1024u;
    if (e4m3) {
        hipLaunchKernelGGL((k_project_few<PRODUCT_E4M3_WIDE>), grid, block, lds, stream, a);
    } else {
        hipLaunchKernelGGL((k_project_few<PRODUCT_BF16>), grid, block, lds, stream, a);
    }
    return hipGetLastError();
}

hipError_t launch_project(hipStream_t stream, const lily_projection& p, const ProjectWorkspace& ws) {
    const uint32_t e = p.dtype == LILY_BF16 ? 2u : 1u;
    ProjectArgs a = {};
    a.x = static_cast<const char*>(p.x_dev);
    a.w = static_cast<const char*>(p.weight_dev);
    a.x_scales = p.x_scales_dev;
    a.w_scales = p.weight_scales_dev;
    a.bias = p.bias_dev;
    a.residual = p.residual_dev;
    a.out = p.out_dev;
    a.x_stride = p.rows > 1u ? p.x_stride * e : 0u;
    a.w_stride = p.n > 1u ? p.weight_stride * e : 0u;
    a.residual_stride = p.residual_stride;
    a.out_stride = p.out_stride;
    a.rows = p.rows;
    a.n = p.n;
    a.d_bytes = p.d * e;
    a.bias_bf16 = p.bias_dtype == LILY_BF16;
    a.residual_bf16 = p.residual_dtype == LILY_BF16;
    a.out_bf16 = p.out_dtype == LILY_BF16;
    a.act = p.activation;
    const uint64_t out_size = a.out_bf16 ? 8u : 16u, res_size = a.residual_bf16 ? 8u : 16u;   // of four elements
    a.wide = reinterpret_cast<uintptr_t>(p.out_dev) % out_size == 0u && (p.rows == 1u || p.out_stride % 4u == 0u) &&
             (p.residual_dev == nullptr || (reinterpret_cast<uintptr_t>(p.residual_dev) % res_size == 0u &&
                                            (p.rows == 1u || p.residual_stride % 4u == 0u)));
    a.splits = 1;
    a.part = Handed<uint64_t>{ws.part};
    a.ticket = ws.ticket;
    const bool e4m3 = p.dtype == LILY_E4M3;
    if (p.rows <= 16u) {
        return launch_project_few(stream, a, e4m3);
    }
    return launch_project_tiles(stream, a, e4m3, ws.part_words, ws.tickets, ws.handover);
}

}  // namespace lily
