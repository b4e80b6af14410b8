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
};
hipError_t launch_project(hipStream_t stream, const lily_projection& p, const ProjectWorkspace& ws);

}  // namespace lily
