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
#pragma unroll
    for (uint32_t j = 0; j < DEPTH; ++j) {
        if (j < count) {
            ask(j, j);
        }
    }
    f32x4 acc[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const uint32_t off = r * LINE + ((g ^ (r >> 1)) << 4);
    uint32_t slot = 0;
    for (uint32_t l = 0; l < count; ++l) {
        if (l + DEPTH <= count) {
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
        __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0): the slot has been read
        __builtin_amdgcn_sched_barrier(0);
        if (l + DEPTH < count) {
            ask(l + DEPTH, slot);
        }
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            acc[t] = product<P>(fw, fx[t], acc[t]);
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

template <int RT, int WAVES, int DEPTH>
hipError_t launch_few(hipStream_t stream, const ProjectArgs& a, bool e4m3) {
    constexpr uint32_t lds = WAVES * DEPTH * (16 + 16 * RT) * LINE;
    static_assert(lds >= WAVES * RT * 1024, "the sums' place");
    const dim3 grid((a.n + 15u) / 16u), block(WAVES * 64);
    static LdsAllowed allowed[2];
    const void* kernel = e4m3 ? (const void*)k_project_few<PRODUCT_E4M3_WIDE, RT, WAVES, DEPTH>
                              : (const void*)k_project_few<PRODUCT_BF16, RT, WAVES, DEPTH>;
    if (const hipError_t e = allowed[e4m3 ? 1 : 0].say(kernel, lds); e != hipSuccess) {
        return e;
    }
    if (e4m3) {
        hipLaunchKernelGGL((k_project_few<PRODUCT_E4M3_WIDE, RT, WAVES, DEPTH>), grid, block, lds, stream, a);
    } else {
        hipLaunchKernelGGL((k_project_few<PRODUCT_BF16, RT, WAVES, DEPTH>), grid, block, lds, stream, a);
    }
    return hipGetLastError();
}

}  // namespace

// (waves x lines of a wave in flight, d = 4096 bf16, n = 4096 / 151 936 in E4M3, us: 8 x 2 7.5 / 105, 8 x 4 7.7 / 150, 4 x 4
// 7.8 / 103; 64 rows 4 x 2 10.1, 8 x 1 10.3, 4 x 4 10.4)
hipError_t launch_project_few(hipStream_t stream, const ProjectArgs& a, bool e4m3) {
    return a.rows <= 16u   ? launch_few<1, 8, 2>(stream, a, e4m3)
           : a.rows <= 32u ? launch_few<2, 8, 2>(stream, a, e4m3)
                           : launch_few<4, 4, 2>(stream, a, e4m3);
}

hipError_t launch_project(hipStream_t stream, const lily_projection& p, const ProjectWorkspace& ws) {
    ProjectArgs a = project_args(p, ws);
    const bool e4m3 = p.dtype == LILY_E4M3;
    const ProjectPlan plan = project_plan(a, ws);
    a.splits = plan.splits;
    return plan.tile == 0u ? launch_project_few(stream, a, e4m3) : launch_project_tiles(stream, a, e4m3, plan.tile);
}

}  // namespace lily
