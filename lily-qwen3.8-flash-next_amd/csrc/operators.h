// operators.h - host-callable launchers of the operators around the head.
#pragma once

#include <hip/hip_runtime_api.h>

#include "../../include/lily_sampler.h"

namespace lily {

// The norm (norm.hip): a row is a workgroup of up to 1024 threads, with pieces of eight elements.
struct NormShape {
    uint32_t pieces, threads;   // pieces a thread holds
};
constexpr NormShape norm_shape(uint32_t d) {
    const uint32_t held = (d + 7u) / 8u, pieces = held <= 1024u ? 1u : held <= 2048u ? 2u : 4u;
    return {pieces, ((held + pieces - 1u) / pieces + 63u) / 64u * 64u};
}
hipError_t launch_rms_norm(hipStream_t stream, const lily_norm& norm);

// The matrix product with an epilogue (project_few.hip, project_tiles.hip); the workspace is the sampler's.
struct ProjectWorkspace {
    float* part;            // sums of parts of d, in 16-byte units
    uint64_t part_floats;
    uint32_t tile = 0;      // 64, 128 or 256: what more than 16 rows get; 0: by an estimate of the time
    uint32_t looks = 4096;  // of a distillation's workgroups for the sums of their row's other slices
    bool strict = false;    // nothing is to rest on the order in which the hardware counts stores
    uint64_t* exchange;     // of a distillation of few rows: those sums, and counters, zeros between two calls
};
hipError_t launch_project(hipStream_t stream, const lily_projection& p, const ProjectWorkspace& ws);

// The layer norm and its backward pass (layer_norm.hip): rows as the norm has them.
hipError_t launch_layer_norm(hipStream_t stream, const lily_layer& layer);
hipError_t launch_layer_norm_backward(hipStream_t stream, const lily_layer_grad& grad, const ProjectWorkspace& ws);

// 8-bit floats with a scale for each block (blocks.hip), and their product (project_blocks.hip).
hipError_t launch_quantize_blocks(hipStream_t stream, const lily_blocks& blocks);
hipError_t launch_project_blocks(hipStream_t stream, const lily_block_projection& p, const ProjectWorkspace& ws);

// Distillation (distill.hip): workgroups of this many threads take slices of a row, of this many ids at most.
constexpr uint32_t DISTILL_SLICE = 32768, DISTILL_THREADS = 512;
constexpr uint32_t DISTILL_ALONE = 768;   // workgroups of few rows: three a compute unit
constexpr uint64_t DISTILL_EXCHANGE = DISTILL_ALONE * 28ull;   // bytes: three words and a counter each
hipError_t launch_distill(hipStream_t stream, const lily_distillation& d, bool backward, const ProjectWorkspace& ws);

}  // namespace lily
