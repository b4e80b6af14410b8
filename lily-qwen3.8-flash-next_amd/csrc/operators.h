// operators.h - host-callable launchers of the operators around the head.
#pragma once

#include <hip/hip_runtime_api.h>

#include "../../include/lily_sampler.h"

namespace lily {

// The norm (norm.hip).  `pieces`: rows start at multiples of 16 bytes in every array and d is a
// multiple of 8.
hipError_t launch_rms_norm(hipStream_t stream, const lily_norm& norm, bool pieces);

// The matrix product with an epilogue (project_few.hip, project_tiles.hip); the workspace is the sampler's.
struct ProjectWorkspace {
    uint64_t* part;
    uint64_t part_words;
    uint32_t* ticket;   // zero between launches
    uint32_t tickets;
    uint32_t handover;  // 0 = by the launch's size, 1 = strict, 2 = relaxed
};
hipError_t launch_project(hipStream_t stream, const lily_projection& p, const ProjectWorkspace& ws);

}  // namespace lily
