// project_plan.h - a matrix product's arguments, and which kernel it gets: the host's part of it, without a device.
#pragma once

#include <algorithm>
#include <cstdint>

#include "operators.h"

namespace lily {

constexpr uint32_t LINE = 128;   // bytes of a row that are taken at a time

struct ProjectArgs {
    const char* x;
    const char* w;
    const float* x_scales;      // or null
    const float* w_scales;      // or null
    const void* bias;           // or null
    const void* residual;       // or null
    void* out;
    uint64_t x_stride, w_stride;               // bytes
    uint64_t residual_stride, out_stride;      // elements
    uint32_t rows, n, d_bytes;
    uint32_t bias_bf16, residual_bf16, out_bf16, act;
    uint32_t splits;            // parts of d, each a workgroup's
    float* part;                // their sums, [splits][rows][part_stride(n)]
    // scales of blocks: of 128 elements of a row of x, of 128 x 128 weights
    const float* x_blocks;      // [rows][x_blocks_stride]
    const float* w_blocks;      // [over(n, 128)][w_blocks_stride]
    uint32_t x_blocks_stride, w_blocks_stride;   // floats
};

constexpr uint32_t part_stride(uint32_t n) { return (n + 3u) / 4u * 4u; }

inline ProjectArgs project_args(const lily_projection& p, const ProjectWorkspace& ws) {
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
    a.splits = 1;
    a.part = ws.part;
    return a;
}

// Which kernel, and how many parts of d: by an estimate of each one's time in us, from what they take on the chip
// (rows x n x d in bf16, three sets of operands in turn, the estimate in brackets):
//   few rows     a compute unit takes in 85 GB/s through LDS: 64 x 4096 x 4096 10.1 (10.5), 64 x 16384 x 2048 19.4 (18.2)
//   64 x 64      a line of d 0.22 where a compute unit has one tile, 0.21 a round of tiles: 256 x 4096 x 4096 17.8 (18.1),
//                512 x 4096 x 4096 28.6 (30.9), 64 x 16384 x 2048 16.4 (16.2: memory)
//   128 x 128    a line 0.48 a round, 0.38 where tiles are few: 1024 x 4096 x 4096 36.7 (36.7), 8192 x 4096 x 4096 259 (252)
//   256 x 256    1.45 a line, and 13 for every tile's epilogue, which nothing hides, 29 with a residual: 8192 x 4096 x 4096
//                213 (214), with a residual 238 (246) where 128 x 128 takes 255 to 265 (264); 8192 x 8192 x 2048 240 (240) against
//                266 (252), but with a residual 302 (304) against 292 (276)
// Parts of d: a launch more (1.5), and the parts' sums written and read at 5.5 TB/s: 64 x 1000 x 8192 in eight 10.6 (10.5)
// against 25.5 in one; 300 x 4096 x 4096 in two of 128 x 128 22.2 (23.3), where 64 x 64 takes 28.1 in one and 25.9 in two
// and 128 x 128 30.4 in one; 512 x 4096 x 4096 25.9 (29.9); 100 x 10 007 x 4096 in E4M3, 79 tiles of 128 x 128, in two
// 16.6 (16.5), in three 16.9 (16.9), in four, a second round, 20.0 (21.5).  Memory at 5.6 TB/s bounds all of them.
// Rows that do not start at lines of 128 bytes take two requests a line, 1.4 times as long where tiles are few, 1.15 times where
// compute units have several: the same with rows of 4128 bytes 19.3 in three parts (18.9), 20.2 in two (18.9), 23.4 in one of
// 64 x 64 (22.8); 5000 x 7000 x 1504 bf16 125 by 128 x 128 (125), 135 by 256 x 256 (145).
// Weights that come from memory every time (700 MB of them in turn, where three sets of 32 MB stay in the last-level cache) take
// longer and change no choice above: 64 x 4096 x 4096 14.2 by few rows and by 64 x 64, 256 rows 22.4 and 23.2 by 64 x 64 and
// 128 x 128, 1024 rows 42 by 128 x 128, 65 by 64 x 64.
// The rates are those of bf16 and of the 8-bit products.  E4M3 with an f32 output widens its operands, four products and their
// conversions for a line's two in bf16, which the estimate does not know: it is up to half of what these take, and its choice,
// against the best of the others (700 MB in turn): 64 x 4096 x 4096 few rows 9.4, 64 x 64 13.1; 256 rows 64 x 64 18.6, 128 x 128 23.8;
// 1024 rows 128 x 128 39, 64 x 64 46; 128 x 151 936 x 4096 128 x 128 181, 64 x 64 228; but 4096 rows 256 x 256 124, 128 x 128 113; 8192
// rows 236 and 221; 8192 x 12 288 x 4096 687 and 642; and 32 x 151 936 x 4096 few rows 190, 64 x 64 144.
struct ProjectPlan {
    uint32_t tile = 0;     // 0: few rows
    uint32_t splits = 1;
};
// What the estimate goes by, us: what a launch takes before and behind its lines, a line of d for a round of tiles, a round's epilogue.
struct ProjectRates {
    double few = 85e3;                                      // bytes a compute unit takes in
    double start64 = 4.0, line64_one = 0.22, line64 = 0.21, tile64 = 0.0;   // (`one`: the least that a line takes)
    double start128 = 6.0, line128_one = 0.38, line128 = 0.48, tile128 = 0.0;
    double line256 = 1.45, tile256 = 13.0, tile256_residual = 29.0;
    uint32_t outputs128 = 128;                              // of a tile of 128 rows
    bool large = true;                                      // is there a tile of 256?
};
inline ProjectPlan project_plan(const ProjectArgs& a, const ProjectWorkspace& ws, const ProjectRates& rate = ProjectRates()) {
    const double rows = a.rows, n = a.n, bytes = a.d_bytes;
    const uint32_t lines = (a.d_bytes + LINE - 1u) / LINE;
    const double memory = ((rows + n) * bytes + rows * n * (a.out_bf16 ? 2.0 : 4.0)) / 5.6e6;
    auto over = [](uint32_t x, uint32_t y) { return (x + y - 1u) / y; };
    auto rounds = [](uint64_t tiles) { return (double)((tiles + 255u) / 256u); };
    auto straight = [](const char* p, uint64_t stride) { return (reinterpret_cast<uintptr_t>(p) | stride) % LINE == 0u; };
    const bool crossing = !(straight(a.x, a.x_stride) && straight(a.w, a.w_stride));
    auto crossed = [&](bool few) { return !crossing ? 1.0 : few ? 1.4 : 1.15; };
    const double residual = a.residual == nullptr ? 0.0 : rows * n * (a.residual_bf16 ? 2.0 : 4.0) / 5.6e6;
    ProjectPlan best;
    double least = 1e30;
    auto offer = [&](uint32_t tile, uint32_t splits, double us) {
        if (us < least && (ws.tile == 0u || ws.tile == tile || a.rows <= 16u)) {
            least = us;
            best.tile = tile;
            best.splits = splits;
        }
    };
    if (a.rows <= 64u) {
        const double blocks = a.rows <= 16u ? 2.0 : a.rows <= 32u ? 3.0 : 5.0;   // of 16 rows a workgroup takes in
        offer(0u, 1u, 2.8 + std::max(memory, rounds(over(a.n, 16u)) * blocks * 16.0 * bytes / rate.few));
        if (a.rows <= 16u) {
            return best;   // (nothing else reads the weights once)
        }
    }
    const uint64_t t64 = (uint64_t)over(a.rows, 64u) * over(a.n, 64u), t128 = (uint64_t)over(a.rows, 128u) * over(a.n, rate.outputs128),
                   t256 = (uint64_t)over(a.rows, 256u) * over(a.n, 256u);
    for (uint32_t k = 1; k <= 16u; ++k) {
        if (k > 1u && (lines < 4u * k || (double)k * rows * part_stride(a.n) > (double)ws.part_floats)) {
            break;
        }
        const double each = lines / (double)k, join = k > 1u ? 1.5 + k * rows * n * 8.0 / 5.5e6 : 0.0;
        const double turns64 = rounds(t64 * k), turns128 = t128 * k <= 256u ? (double)(t128 * k) / 256.0 : rounds(t128 * k);
        offer(64u, k, std::max(3.0 + memory, rate.start64 + each * crossed(turns64 <= 2.0) * std::max(rate.line64_one, rate.line64 * turns64) + rate.tile64 * turns64) +
                          residual + join);
        offer(128u, k, std::max(3.0 + memory, rate.start128 + each * crossed(turns128 <= 1.0) * std::max(rate.line128_one, rate.line128 * turns128) + rate.tile128 * turns128) +
                           residual + join);
    }
    if (rate.large) {
        offer(256u, 1u, 2.0 + std::max(memory, rounds(t256) * ((a.residual != nullptr ? rate.tile256_residual : rate.tile256) + lines * rate.line256)));
    }
    return best;
}

}  // namespace lily
