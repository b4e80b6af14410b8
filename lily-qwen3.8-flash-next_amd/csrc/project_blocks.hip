// project_blocks.hip - the matrix product of 8-bit floats with a scale for each block of 128, and an epilogue.
//
//     out[r][v] = residual[r][v] + act(sum_b xs[r][b] ws[v / 128][b] sum_{i in b} x[r][i] w[v][i] + bias[v])
//
// The kernels are the plain product's (project_few.hip, project_tile.h): what they take of a row at a time, 128 bytes, is
// one block.  Its products are summed on the matrix cores from zero, and the sum joins the tile's by a multiplication
// with both scales and an addition in f32, behind the next products.  The scales of x arrive in LDS eight blocks at a time (a load for
// each block of each row took as long as the rows: 8192 x 12 288 x 4096 507 us, 437 so); those of the weights are one a wave and line,
// 64 lines' in a lane each.
//
// 4 x 151 936 x 4096 to f32 100 to 102 us (622 MB, 6.2 TB/s), 100 x 10 007 x 4096 17 us where the memory takes 7.5, 8192 x 12 288 x
// 4096 at 2.1 PFLOP/s, two thirds of what the matrix cores reach in E4M3.
#include "project_tile.h"

namespace lily {

namespace {

// The large tile, 256 x 256 by eight waves of 128 x 64: the sums take half of a wave's registers and have to be ordinary ones (what scales
// them reads and writes them), so that neither four waves of 128 x 128 nor the quarters of project_tile.h have room for them.  Two waves
// share a matrix pipe: one scales and reads while the other multiplies.
//
// A wave holds its four blocks of weights of a stage and takes its eight blocks of rows one after the other, the next one on its way
// from LDS.  LDS holds two stages.  A stage's weights and first rows (blocks 0 to 3) are asked for when block 3 begins, two stages
// ahead, its other rows when block 7 does; both are waited for one and a half stages later, at the same two places.  Nothing in a
// stage is conditional, its loads beyond the last line are the last line's again: a branch in the middle of a stage made the compiler
// move additions across it, 112 registers of sums waiting (312 bytes of scratch).
//
// 8192 x 12 288 x 4096 385 to 398 us by the chip, 2.1 PFLOP/s; the product with a scale a row, which has nothing to scale between two lines,
// takes 349 on the same chip.  The matrix cores are busy 49% of its cycles (63% there), the vector unit with 96 000 instructions a SIMD about
// as long: neither bounds it, they stand behind one another.  Both waves of a SIMD pass the same two barriers a stage, and so read, multiply and
// add at much the same time.  A third product between a sum and its addition, or waves of two priorities, change nothing (389 to 391).
template <class T>
__global__ void __launch_bounds__(512, 2) k_blocks_large(const ProjectArgs a, uint32_t m_tiles, uint32_t n_tiles) {
    constexpr int S = 16, MB = 8, NB = 4, XL = 2, WL = 4;   // blocks of a wave; loads of a wave: half of the rows', all of the weights'
    constexpr uint32_t X_BYTES = T::BM * LINE, STAGE = X_BYTES + T::BN * LINE;
    static_assert(T::WAVES == 8 && T::WM == 2 && T::MT == MB && T::NT == NB && T::S == S && T::STAGES == 2 * (int)STAGE, "the tile that this is written for");
    extern __shared__ __align__(16) char lds[];
    typedef Block<S> Operand;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
    const uint32_t wm = wave / T::WN, wn = wave % T::WN, r_in = lane % (uint32_t)S;
    const TilePlace place = place_of<T>(a, m_tiles, n_tiles);
    const uint32_t m0 = place.m0, n0 = place.n0, steps = (a.d_bytes + LINE - 1u) / LINE;
    const char* x_rows = a.x + (uint64_t)m0 * a.x_stride;
    const char* w_rows = a.w + (uint64_t)n0 * a.w_stride;
    // A load of a wave brings eight rows; half h of the rows: the 64 of that half of either wave of rows.
    auto x_row = [&](int h, int i) { return (uint32_t)i * 128u + (uint32_t)h * 64u + wave * 8u; };
    auto w_row = [&](int i) { return (uint32_t)i * 64u + wave * 8u; };
    const uint32_t piece = ((lane & 7u) ^ ((lane >> 4) & 3u) ^ ((wave & 1u) << 2)) * 16u;   // a row's pieces change places: piece ^ (row / 2) % 8
    uint32_t x_at[2][XL], w_at[WL];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < XL; ++i) {
            x_at[h][i] = min(x_row(h, i) + (lane >> 3), a.rows - 1u - m0) * (uint32_t)a.x_stride + piece;
        }
    }
#pragma unroll
    for (int i = 0; i < WL; ++i) {
        w_at[i] = min(w_row(i) + (lane >> 3), a.n - 1u - n0) * (uint32_t)a.w_stride + piece;
    }
    typedef __attribute__((address_space(1))) const void* gptr;
    typedef __attribute__((address_space(3))) void* lptr;
    auto x_buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(x_rows), 0, -1, 0x00020000);
    auto w_buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(w_rows), 0, -1, 0x00020000);
    auto ask_x = [&](uint32_t s, int h) {
#pragma unroll
        for (int i = 0; i < XL; ++i) {
            char* to = lds + (s & 1u) * STAGE + x_row(h, i) * LINE;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(x_buffer, (lptr)to, 16, (int)x_at[h][i], (int)(min(s, steps - 1u) * LINE), 0, 0);
        }
    };
    auto ask_w = [&](uint32_t s) {
#pragma unroll
        for (int i = 0; i < WL; ++i) {
            char* to = lds + (s & 1u) * STAGE + X_BYTES + w_row(i) * LINE;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(w_buffer, (lptr)to, 16, (int)w_at[i], (int)(min(s, steps - 1u) * LINE), 0, 0);
        }
    };
    // Scales: as in project_tile.h, eight stages' a load.
    const uint32_t block = min((n0 + wn * (uint32_t)(NB * S)) / LILY_BLOCK, (a.n - 1u) / LILY_BLOCK);
    WeightScales w_scales = {a.w_blocks + (uint64_t)block * a.w_blocks_stride, steps, 0.0f};
    w_scales.ask(0u);
    auto ask_scales = [&](uint32_t run, uint32_t k) {
        const uint32_t row = wave * (uint32_t)(T::SCALE_LOADS * 8) + k * 8u, in = row + (lane >> 3);
        const uint32_t stage = min(run * (uint32_t)T::RUN + ((lane & 7u) ^ ((in >> 3) & 7u)), steps - 1u);
        const float* from = a.x_blocks + (uint64_t)min(m0 + in, a.rows - 1u) * a.x_blocks_stride + stage;
        __builtin_amdgcn_global_load_lds((gptr)from, (lptr)(lds + T::STAGES + (run & 1u) * (uint32_t)T::SCALES + row * (uint32_t)(T::RUN * 4)), 4, 0, 0);
    };
    // A lane's operands, and its scales: row + 16 i has its piece of a run two places on.
    const uint32_t off = r_in * LINE + ((Operand::first_piece(lane) ^ ((r_in >> 1) & 7u)) << 4);
    uint32_t x_from = wm * (uint32_t)(MB * S) * LINE + off, w_from = X_BYTES + wn * (uint32_t)(NB * S) * LINE + off;
    const uint32_t scale_row = (uint32_t)T::STAGES + (wm * (uint32_t)(MB * S) + r_in) * (uint32_t)(T::RUN * 4), scale_turn = r_in >> 3;
    Operand fw[NB], fx[2];
    float scale[2];
    auto read = [&](Operand& f, uint32_t from, int row) {
#pragma unroll
        for (int q = 0; q < Operand::PIECES; ++q) {
            f.p[q] = *reinterpret_cast<const u32x4*>(lds + (from ^ ((uint32_t)q * Operand::NEXT_PIECE)) + (uint32_t)row * LINE);
        }
    };
    auto read_scale = [&](uint32_t s, int i) {
        const uint32_t turn = (s ^ scale_turn ^ (uint32_t)(2 * i)) & 7u;
        scale[i & 1] = *reinterpret_cast<const float*>(lds + scale_row + (s / (uint32_t)T::RUN & 1u) * (uint32_t)T::SCALES +
                                                       (uint32_t)(i * S * T::RUN * 4) + turn * 4u);
    };
    f32x4 acc[2][MB / 2][2][NB / 2], line[4];
#pragma unroll
    for (int b = 0; b < MB * NB; ++b) {
        acc[b / 16][b / 4 % 4][b / 2 % 2][b % 2] = f32x4(0.0f);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        line[q] = f32x4(0.0f);
    }
    // The sums of a block's line are scaled into the tile's two products later (of the last two of a stage, in the next one).
    float by = 0.0f, by_before = 0.0f;   // of this block of rows and of the one before
    auto add = [&](int t, float f) {
        f32x4& c = acc[t / 16][t / 4 % 4][t / 2 % 2][t % 2];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            c[e] = __builtin_fmaf(line[t % 4][e], f, c[e]);
        }
    };
#pragma unroll
    for (int k = 0; k < T::SCALE_LOADS; ++k) {
        ask_scales(0u, (uint32_t)k);
    }
    ask_w(0u);
    ask_x(0u, 0);
    ask_x(0u, 1);
    ask_scales(0u, 0u);   // (again: what the waits below count)
    ask_w(1u);
    ask_x(1u, 0);
    ask_x(1u, 1);
    asm volatile("s_waitcnt vmcnt(11)\n\ts_barrier" ::: "memory");
    read(fx[0], x_from, 0);
    read_scale(0u, 0);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        read(fw[j], w_from, j * S);
    }
    w_scales.settle();
#pragma clang loop unroll(disable)
    for (uint32_t s = 0; s < steps; ++s) {
        if (s != 0u && (s & 63u) == 0u) {
            w_scales.ask(s);
            w_scales.settle();
        }
        const float w = w_scales.of(s);
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            if (i == 3) {   // this stage's other rows have landed; its weights' and first rows' places are free
                asm volatile("s_waitcnt vmcnt(9) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
                ask_scales(s / (uint32_t)T::RUN + 1u, s % (uint32_t)T::SCALE_LOADS);   // (twice each)
                ask_w(s + 2u);
                ask_x(s + 2u, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (i == MB - 1) {   // the next stage's weights and first rows have landed; this one's other rows' place is free
                asm volatile("s_waitcnt vmcnt(9) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
                ask_x(s + 2u, 1);
                __builtin_amdgcn_sched_barrier(0);
                x_from ^= STAGE;
                w_from ^= STAGE;
            }
            by_before = by;
            by = scale[i & 1] * w;
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const int t = i * NB + j;
                line[t % 4] = step<PRODUCT_BLOCKS, S>(fw[j], fx[i & 1], f32x4(0.0f), 0);
                __builtin_amdgcn_sched_barrier(0);
                if (j == 0) {   // (what is read next: the first wait of a block is for the reads of the block before)
                    read(fx[(i + 1) & 1], x_from, i < MB - 1 ? (i + 1) * S : 0);
                    read_scale(i < MB - 1 ? s : s + 1u, (i + 1) % MB);
                }
                if (i == MB - 1) {
                    read(fw[j], w_from, j * S);
                }
                add((t + MB * NB - 2) % (MB * NB), j < 2 ? by_before : by);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    add(MB * NB - 2, by);
    add(MB * NB - 1, by);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    give_out<T>(a, acc, lds, m0 + wm * (uint32_t)(MB * S), n0 + wn * (uint32_t)(NB * S), wave, lane, 0u);
}

template <Products P, class T>
hipError_t launch_tile(hipStream_t stream, const ProjectArgs& a) {
    const uint32_t m_tiles = (a.rows + T::BM - 1u) / T::BM, n_tiles = (a.n + T::BN - 1u) / T::BN;
    static LdsAllowed allowed;
    if (const hipError_t e = allowed.say((const void*)k_project_tiles<P, T>, T::LDS_BYTES); e != hipSuccess) {
        return e;
    }
    hipLaunchKernelGGL((k_project_tiles<P, T>), dim3(m_tiles * n_tiles * a.splits), dim3(64 * T::WAVES), T::LDS_BYTES, stream, a, m_tiles, n_tiles);
    return a.splits > 1u ? launch_project_join(stream, a) : hipGetLastError();
}
hipError_t launch_large(hipStream_t stream, const ProjectArgs& a) {
    typedef Tile<16, 2, 4, 8, 4, 1, 2, true> T;
    const uint32_t m_tiles = (a.rows + T::BM - 1u) / T::BM, n_tiles = (a.n + T::BN - 1u) / T::BN;
    static LdsAllowed allowed;
    if (const hipError_t e = allowed.say((const void*)k_blocks_large<T>, T::LDS_BYTES); e != hipSuccess) {
        return e;
    }
    hipLaunchKernelGGL((k_blocks_large<T>), dim3(m_tiles * n_tiles), dim3(64 * T::WAVES), T::LDS_BYTES, stream, a, m_tiles, n_tiles);
    return hipGetLastError();
}

// What the estimate of the plan (project_plan.h) goes by, from what the kernels take here (rows x n x d, three sets of operands in turn,
// the estimate in brackets):
//   few rows     the widened products, not the loads, bound it: 32 x 4096 x 4096 8.6 (7.7), 64 rows 10.6 to 12.6 (11.0), but
//                32 x 151 936 x 4096 202 (189) where 64 x 64 takes 123 (118)
//   64 x 64      256 x 4096 x 4096 14.2 (14.5) against 19.7 by 128 x 128, 100 x 10 007 x 4096 17.2 (20.2) against 17.8, 512 x 4096 x 4096
//                19.6 (20.2) against 22, 128 x 4096 x 4096 in two parts 13.5 (13.8), in four 16 (15.1)
//   128 x 128    256 x 12 288 x 4096 24.4 (23.3) against 28.8 by 64 x 64, 1024 x 4096 x 4096 25.6 (26.2) against 34 and 53 by 256 x 256,
//                1024 x 12 288 x 4096 57.5 (60.6) against 61
//   256 x 256    8192 x 12 288 x 4096 385 to 396 (390) against 444, 8192 x 8192 x 2048 143 to 150 (145) against 162, 4096 x 4096 x 14 336 210 (211)
//                against 249; with a residual 8192 x 12 288 x 4096 456 (432) against 490, 4096 x 4096 x 4096 72 (74) against 81
// An f32 output's widened products: 64 x 64 up to 512 x 4096 x 4096 (28.2, where 128 x 64 takes 30), then 128 x 64, whose waves widen six
// blocks for eight blocks' products, where 64 x 64 widens eight: 1024 x 4096 x 4096 43 against 51, 8192 x 12 288 x 4096 900 against 1066.
// (128 x 128 by four waves, eight widened for sixteen, has no registers for it and took 1650; 128 x 128 by eight waves 913.)
ProjectRates block_rates(const ProjectArgs& a) {
    ProjectRates rate;
    rate.few = 40e3;
    rate.start64 = 6.8;
    rate.line64_one = a.out_bf16 ? 0.23 : 0.45;
    rate.line64 = a.out_bf16 ? 0.20 : 0.33;
    rate.tile64 = 0.3;
    rate.start128 = 9.0;
    rate.line128_one = a.out_bf16 ? 0.42 : 0.6;
    rate.line128 = 0.50;
    rate.tile128 = 1.2;
    rate.line256 = 1.8;
    rate.tile256 = 7.0;
    rate.tile256_residual = 14.0;
    rate.outputs128 = a.out_bf16 ? 128u : 64u;
    rate.large = a.out_bf16 && a.d_bytes % LINE == 0u;
    return rate;
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
    ProjectArgs a = project_args(p, given);
    a.x_blocks = b.x_scales_dev;
    a.w_blocks = b.weight_scales_dev;
    a.x_blocks_stride = b.rows > 1u ? (uint32_t)b.x_scales_stride : 0u;
    a.w_blocks_stride = b.n > LILY_BLOCK ? (uint32_t)b.weight_scales_stride : 0u;
    ProjectWorkspace ws = given;
    const ProjectRates rates = block_rates(a);
    if (ws.tile == 256u && !rates.large) {
        ws.tile = 128u;
    }
    const ProjectPlan plan = project_plan(a, ws, rates);
    a.splits = plan.splits;
    return plan.tile == 0u     ? launch_project_few(stream, a, PRODUCT_BLOCKS_WIDE)
           : plan.tile == 256u ? launch_large(stream, a)
           : plan.tile == 64u  ? (a.out_bf16 ? launch_tile<PRODUCT_BLOCKS, Tile<16, 2, 2, 2, 2, 2, 4, true>>(stream, a)
                                             : launch_tile<PRODUCT_BLOCKS_WIDE, Tile<16, 2, 2, 2, 2, 2, 4, true>>(stream, a))
           : a.out_bf16        ? launch_tile<PRODUCT_BLOCKS, Tile<16, 2, 2, 4, 4, 2, 2, true>>(stream, a)
                               : launch_tile<PRODUCT_BLOCKS_WIDE, Tile<16, 2, 2, 4, 2, 2, 2, true>>(stream, a);
}

}  // namespace lily
