// project_few.hip - the matrix product with an epilogue for few rows: the weights are read once at the speed of
// memory, the matrix cores idle.
//
// A workgroup takes 16 outputs' weight rows; its waves share d, a run of whole lines (128 bytes a row) each, so that
// a layer of a few thousand outputs already keeps every compute unit's memory path busy without a join between
// workgroups.  A wave works alone: its lines arrive in a ring of its own in LDS, loads that write LDS themselves, eight
// whole lines an instruction (a lane that loads what the product wants of it touches 16 lines with every 16
// lanes: 16 bytes a clock and compute unit, whatever is in flight), and it waits for its own loads only.  The
// waves' sums meet in LDS.
//
// Measured: 4 x 151 936 x 4096 in E4M3 104 to 108 us (622 MB, 5.8 TB/s), 1 x 4096 x 4096 in bf16 7.6 us (33.6 MB, 4.4 TB/s:
// a launch and two trips to memory are 2.8 of them), 12 x 2560 x 2560 4.8 us.
#include "launch.h"
#include "project.h"

namespace lily {

namespace {

__device__ const uint4 few_zeros = {0u, 0u, 0u, 0u};   // what lies beyond d

// RT: blocks of 16 rows of x; DEPTH: lines of a wave in flight.
template <Products P, int RT, int WAVES, int DEPTH>
__global__ void __launch_bounds__(WAVES * 64) k_project_few(const ProjectArgs a) {
    constexpr bool BLOCKS = in_blocks(P);
    constexpr uint32_t ROWS = 16 + 16 * RT, SLOT = ROWS * LINE, LOADS = ROWS / 8;
    extern __shared__ __align__(16) char lds[];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
    const uint32_t g = lane >> 4, r = lane & 15u, v0 = blockIdx.x * 16u;
    const uint32_t lines = (a.d_bytes + LINE - 1u) / LINE;
    const uint32_t per = lines / WAVES, over = lines % WAVES;
    const uint32_t from = wave * per + min(wave, over), count = per + (wave < over ? 1u : 0u);
    // The wave that finishes asks for what the epilogue reads before anything else: behind the sums it would be
    // another trip to memory.
    const uint32_t v = v0 + g * 4u, row0 = wave * 16u + r;
    Columns columns;
    Finish finish;
    const bool finishes = wave < (uint32_t)RT && v < a.n && row0 < a.rows;
    if (finishes) {
        columns.load(a, v);
        finish.load(a, row0, v);
    }
    // Instruction i brings rows 8 i .. 8 i + 7 of a line (16 of the weights, then x), a lane the piece that
    // belongs in its place: the pieces of a row change places by the row's number, so that 16 lanes that read one
    // piece of 16 rows meet 16 groups of banks.  (A row beyond the last is the last one's values: its sums go nowhere.)
    const char* src[LOADS];
#pragma unroll
    for (uint32_t i = 0; i < LOADS; ++i) {
        const uint32_t row = i * 8u + (lane >> 3), piece = (lane & 7u) ^ ((row >> 1) & 7u);
        src[i] = (i < 2u ? a.w + (uint64_t)min(v0 + row, a.n - 1u) * a.w_stride
                         : a.x + (uint64_t)min(row - 16u, a.rows - 1u) * a.x_stride) + piece * 16u + from * LINE;
    }
    typedef __attribute__((address_space(1))) const void* gptr;
    typedef __attribute__((address_space(3))) void* lptr;
    char* ring = lds + wave * (DEPTH * SLOT);
    // With a scale for each block: a row's scales of eight lines at a time (one line's would be a request for each of the rows), a run's
    // behind the rings, the next one's on their way.  A row's eight lie from place row / 8 on, so that 16 rows meet 16 banks.
    constexpr uint32_t RUN_LOADS = 2u * RT, RUN_BYTES = RT * 16u * 32u;
    char* const runs = lds + WAVES * DEPTH * SLOT + wave * (2u * RUN_BYTES);
    auto ask_scales = [&](uint32_t run) {
#pragma unroll
        for (uint32_t i = 0; i < RUN_LOADS; ++i) {
            const uint32_t row = i * 8u + (lane >> 3), l = min(run * 8u + ((lane & 7u) ^ (i & 7u)), count - 1u);
            __builtin_amdgcn_global_load_lds((gptr)(a.x_blocks + (uint64_t)min(row, a.rows - 1u) * a.x_blocks_stride + from + l),
                                             (lptr)(runs + (run & 1u) * RUN_BYTES + i * 256u), 4, 0, 0);
        }
    };
    WeightScales w_scales = {BLOCKS ? a.w_blocks + (uint64_t)(v0 / LILY_BLOCK) * a.w_blocks_stride + from : nullptr, count, 0.0f};
    auto ask = [&](uint32_t l, uint32_t slot) {
        char* base = ring + slot * SLOT;
        const uint32_t at = l * LINE;
        if ((from + l + 1u) * LINE <= a.d_bytes) {
#pragma unroll
            for (uint32_t i = 0; i < LOADS; ++i) {
                __builtin_amdgcn_global_load_lds((gptr)(src[i] + at), (lptr)(base + i * 1024u), 16, 0, 0);
            }
        } else {   // the line that d ends in: pieces beyond it are zeros, in both operands
            const char* zeros = reinterpret_cast<const char*>(&few_zeros);
#pragma unroll
            for (uint32_t i = 0; i < LOADS; ++i) {
                const uint32_t piece = (lane & 7u) ^ (((i * 8u + (lane >> 3)) >> 1) & 7u);
                const char* p = (from + l) * LINE + piece * 16u < a.d_bytes ? src[i] + at : zeros;
                __builtin_amdgcn_global_load_lds((gptr)p, (lptr)(base + i * 1024u), 16, 0, 0);
            }
        }
    };
    if (BLOCKS && count != 0u) {
        w_scales.ask(0u);
        ask_scales(0u);
    }
#pragma unroll
    for (uint32_t j = 0; j < DEPTH; ++j) {
        if (j < count) {
            ask(j, j);
        }
    }
    if constexpr (BLOCKS) {
        w_scales.settle();
    }
    f32x4 acc[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const uint32_t off = r * LINE + ((g ^ (r >> 1)) << 4);
    uint32_t slot = 0;
    for (uint32_t l = 0; l < count; ++l) {
        if (BLOCKS && l + DEPTH <= count && (l & 7u) == 1u && l + 7u < count) {   // (a run's scales were asked for in between)
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((DEPTH - 1) * LOADS + RUN_LOADS) : "memory");
        } else if (l + DEPTH <= count) {
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((DEPTH - 1) * LOADS) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        const char* base = ring + slot * SLOT + off;
        auto frag = [&](uint32_t block) {
            Frag f;
            f.lo = *reinterpret_cast<const u32x4*>(base + block * 16u * LINE);
            f.hi = *reinterpret_cast<const u32x4*>(lds + ((uint32_t)(base - lds) ^ 64u) + block * 16u * LINE);
            return f;
        };
        const Frag fw = frag(0);
        Frag fx[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            fx[t] = frag(1u + (uint32_t)t);
        }
        float scale[RT];
        if constexpr (BLOCKS) {
            const float* scales = reinterpret_cast<const float*>(runs + (l >> 3 & 1u) * RUN_BYTES);
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                scale[t] = scales[((uint32_t)t * 16u + r) * 8u + ((l ^ ((uint32_t)t * 2u + (r >> 3))) & 7u)];
            }
        }
        __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0): the slot has been read
        __builtin_amdgcn_sched_barrier(0);
        if (BLOCKS && (l & 7u) == 0u && l + 8u < count) {
            ask_scales(l / 8u + 1u);
        }
        if (l + DEPTH < count) {
            ask(l + DEPTH, slot);
        }
        if constexpr (BLOCKS) {
            if (l != 0u && (l & 63u) == 0u) {
                w_scales.ask(l);
                w_scales.settle();
            }
            const float w = w_scales.of(l);
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const f32x4 line = product<P>(fw, fx[t], f32x4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    acc[t][j] = __builtin_fmaf(line[j], scale[t] * w, acc[t][j]);
                }
            }
        } else {
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                acc[t] = product<P>(fw, fx[t], acc[t]);
            }
        }
        slot = slot + 1u == DEPTH ? 0u : slot + 1u;
    }
    __syncthreads();   // (every ring is the sums' place now)
    f32x4* sums = reinterpret_cast<f32x4*>(lds);
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        sums[(wave * RT + (uint32_t)t) * 64u + lane] = acc[t];
    }
    __syncthreads();
    if (finishes) {   // block `wave` of the rows
        f32x4 sum = sums[wave * 64u + lane];
#pragma unroll
        for (uint32_t q = 1; q < WAVES; ++q) {
            sum += sums[(q * RT + wave) * 64u + lane];
        }
        finish.store(a, row0, v, columns, sum);
    }
}

template <Products P, int RT, int WAVES, int DEPTH>
hipError_t launch_few_of(hipStream_t stream, const ProjectArgs& a) {
    constexpr uint32_t lds = WAVES * (DEPTH * (16 + 16 * RT) * LINE + (in_blocks(P) ? 2 * RT * 16 * 32 : 0));
    static_assert(lds >= WAVES * RT * 1024, "the sums' place");
    static LdsAllowed allowed;
    if (const hipError_t e = allowed.say((const void*)k_project_few<P, RT, WAVES, DEPTH>, lds); e != hipSuccess) {
        return e;
    }
    hipLaunchKernelGGL((k_project_few<P, RT, WAVES, DEPTH>), dim3((a.n + 15u) / 16u), dim3(WAVES * 64), lds, stream, a);
    return hipGetLastError();
}
template <int RT, int WAVES, int DEPTH>
hipError_t launch_few(hipStream_t stream, const ProjectArgs& a, Products products) {
    return products == PRODUCT_BF16        ? launch_few_of<PRODUCT_BF16, RT, WAVES, DEPTH>(stream, a)
           : products == PRODUCT_E4M3_WIDE ? launch_few_of<PRODUCT_E4M3_WIDE, RT, WAVES, DEPTH>(stream, a)
                                           : launch_few_of<PRODUCT_BLOCKS_WIDE, RT, WAVES, DEPTH>(stream, a);
}

}  // namespace

// (waves x lines of a wave in flight, d = 4096 bf16, n = 4096 / 151 936 in E4M3, us: 8 x 2 7.5 / 105, 8 x 4 7.7 / 150, 4 x 4
// 7.8 / 103; 64 rows 4 x 2 10.1, 8 x 1 10.3, 4 x 4 10.4)
hipError_t launch_project_few(hipStream_t stream, const ProjectArgs& a, Products products) {
    return a.rows <= 16u   ? launch_few<1, 8, 2>(stream, a, products)
           : a.rows <= 32u ? launch_few<2, 8, 2>(stream, a, products)
                           : launch_few<4, 4, 2>(stream, a, products);
}

hipError_t launch_project(hipStream_t stream, const lily_projection& p, const ProjectWorkspace& ws) {
    ProjectArgs a = project_args(p, ws);
    const bool e4m3 = p.dtype == LILY_E4M3;
    const ProjectPlan plan = project_plan(a, ws);
    a.splits = plan.splits;
    return plan.tile == 0u ? launch_project_few(stream, a, e4m3 ? PRODUCT_E4M3_WIDE : PRODUCT_BF16) : launch_project_tiles(stream, a, e4m3, plan.tile);
}

}  // namespace lily
