// operators.h - host-callable launchers of the operators around the head.
#pragma once

#include <hip/hip_runtime_api.h>

#include "../../include/lily_sampler.h"

namespace lily {

// The norm (norm.hip).
hipError_t launch_rms_norm(hipStream_t stream, const lily_norm& norm);

// The matrix product with an epilogue (project_few.hip, project_tiles.hip); the workspace is the sampler's.
struct ProjectWorkspace {
    float* part;            // sums of parts of d, in 16-byte units
    uint64_t part_floats;
};
hipError_t launch_project(hipStream_t stream, const lily_projection& p, const ProjectWorkspace& ws);

}  // namespace lily
