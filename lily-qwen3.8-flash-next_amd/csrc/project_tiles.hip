// project_tiles.hip - the matrix product with an epilogue for more rows: tiles on the matrix cores.
//
// Four waves share a tile of rows x outputs, each a block of MT x NT products of 16 x 16.  d goes by stages of
// 128 bytes a row.  A wave's block is taken in quarters, two halves of its rows against two halves of its
// outputs, so that half the operands a stage needs are in registers while the other half is on its way
// from LDS:
//
//     quarter   rows   outputs    meanwhile read from LDS
//     0         first  p          the other outputs of this stage
//     1         first  1 - p      the second rows of this stage
//     2         second 1 - p      the first rows of the next stage
//     3         second p          outputs 1 - p of the next stage, which begins with them (p changes with the stage)
//
// LDS holds two stages in four units: what quarters 2 and 3 of the stage before read (Y: first rows, outputs
// p) and what quarters 0 and 1 read (X: second rows, outputs 1 - p).  Loads write LDS themselves (a wave's
// instruction fills 1 KB: 8 rows of 128 bytes); a unit is asked for as soon as the whole workgroup has read what lay
// there, which is six quarters before it is read.  One barrier for two quarters.
//
// A staged row's eight pieces change places by the row's number (piece ^ (row / 2) % 8): the 16 lanes that
// read one piece of 16 rows then meet 16 different groups of banks.
#include "launch.h"
#include "project.h"

namespace lily {

namespace {

__device__ const uint4 line_of_zeros = {0u, 0u, 0u, 0u};   // what lies beyond d

template <int WM_, int WN_, int MT_, int NT_, int RESIDENT_>
struct Tile {
    static constexpr int WM = WM_, WN = WN_, MT = MT_, NT = NT_, RESIDENT = RESIDENT_;
    static constexpr int MH = MT / 2, NH = NT / 2;                     // products of a half
    static constexpr int BM = WM * MT * 16, BN = WN * NT * 16;
    static constexpr int XR = WM * MH * 16, WR = WN * NH * 16;         // rows of a unit: of x, of the weights
    static constexpr int UNIT = (XR + WR) * (int)LINE;
    static constexpr int XL = XR / 32, WL = WR / 32, LOADS = XL + WL;  // loads of a wave and unit
    static constexpr int LDS_BYTES = 4 * UNIT;
    static_assert(WM * WN == 4 && XR % 32 == 0 && WR % 32 == 0, "whole loads a wave");
};

template <int V>
struct Parity {
    static constexpr int value = V;
};

template <Products P, class T>
__global__ void __launch_bounds__(256, T::RESIDENT) k_project_tiles(const ProjectArgs a, uint32_t m_tiles, uint32_t n_tiles) {
    constexpr int MH = T::MH, NH = T::NH;
    extern __shared__ __align__(16) char lds[];
    __shared__ uint32_t last;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const uint32_t wm = wave / T::WN, wn = wave % T::WN, g = lane >> 4, r16 = lane & 15u;
    // Consecutive workgroups go to consecutive XCDs: each XCD gets a run of tiles of its own (they share
    // its L2), in groups of four tiles of rows.
    const uint32_t tiles = m_tiles * n_tiles, all = tiles * a.splits;
    const uint32_t xcd = blockIdx.x & 7u, slot = blockIdx.x >> 3, each = all / 8u, more = all % 8u;
    const uint32_t job = xcd * each + min(xcd, more) + slot;
    const uint32_t split = job / tiles, tile = job % tiles;
    constexpr uint32_t GROUP_M = 4;
    const uint32_t band = tile / (GROUP_M * n_tiles), in_band = tile % (GROUP_M * n_tiles);
    const uint32_t band_m = min(GROUP_M, m_tiles - band * GROUP_M);
    const uint32_t m0 = (band * GROUP_M + in_band % band_m) * T::BM, n0 = in_band / band_m * T::BN;

    const uint32_t stages_all = (a.d_bytes + LINE - 1u) / LINE;
    const uint32_t per = stages_all / a.splits, over = stages_all % a.splits;
    const uint32_t first = split * per + min(split, over), steps = per + (split < over ? 1u : 0u);

    // Where a lane's pieces come from: 32-bit offsets from the tile's first rows, for both halves.
    const char* x_rows = a.x + (uint64_t)m0 * a.x_stride;
    const char* w_rows = a.w + (uint64_t)n0 * a.w_stride;
    uint32_t x_at[2][T::XL], w_at[2][T::WL], k_at[T::LOADS];
#pragma unroll
    for (int i = 0; i < T::LOADS; ++i) {
        const bool is_x = i < T::XL;
        const uint32_t row = (uint32_t)((is_x ? i : i - T::XL) * 32) + wave * 8u + (lane >> 3);   // of the unit's part
        const uint32_t piece = (lane & 7u) ^ ((row >> 1) & 7u);
        k_at[i] = piece * 16u;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t half = is_x ? (uint32_t)MH * 16u : (uint32_t)NH * 16u;
            const uint32_t tile_row = row / half * (2u * half) + (uint32_t)h * half + row % half;
            if (is_x) {
                x_at[h][i] = min(tile_row, a.rows - 1u - m0) * (uint32_t)a.x_stride + piece * 16u;
            } else {
                w_at[h][i - T::XL] = min(tile_row, a.n - 1u - n0) * (uint32_t)a.w_stride + piece * 16u;
            }
        }
    }
    typedef __attribute__((address_space(1))) const void* gptr;
    typedef __attribute__((address_space(3))) void* lptr;
    // Asks for a unit of stage s: rows' half hx, outputs' half hw, into LDS place `unit`.
    auto ask = [&](uint32_t s, int hx, int hw, int unit) {
        const uint32_t k0 = (first + s) * LINE;
        char* base = lds + unit * T::UNIT + wave * 1024u;
        if (k0 + LINE <= a.d_bytes) {
            const char* xk = x_rows + k0;
            const char* wk = w_rows + k0;
#pragma unroll
            for (int i = 0; i < T::XL; ++i) {
                __builtin_amdgcn_global_load_lds((gptr)(xk + (uint64_t)x_at[hx][i]), (lptr)(base + i * 4096), 16, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < T::WL; ++i) {
                __builtin_amdgcn_global_load_lds((gptr)(wk + (uint64_t)w_at[hw][i]), (lptr)(base + (T::XL + i) * 4096), 16, 0, 0);
            }
        } else {   // the stage that d ends in: pieces beyond it are zeros
            const char* zeros = reinterpret_cast<const char*>(&line_of_zeros);
#pragma unroll
            for (int i = 0; i < T::LOADS; ++i) {
                const char* from = i < T::XL ? x_rows + k0 + (uint64_t)x_at[hx][i < T::XL ? i : 0]
                                             : w_rows + k0 + (uint64_t)w_at[hw][i < T::XL ? 0 : i - T::XL];
                from = k0 + k_at[i] < a.d_bytes ? from : zeros;
                __builtin_amdgcn_global_load_lds((gptr)from, (lptr)(base + i * 4096), 16, 0, 0);
            }
        }
    };
    // A lane's operands out of a unit.
    const uint32_t off = r16 * LINE + ((g ^ (r16 >> 1)) << 4);
    const uint32_t x_off = wm * (uint32_t)(MH * 16) * LINE + off, w_off = (uint32_t)T::XR * LINE + wn * (uint32_t)(NH * 16) * LINE + off;
    Frag fx[2][MH], fw[2][NH];
    auto read_x = [&](int h, int unit) {
#pragma unroll
        for (int i = 0; i < MH; ++i) {
            const uint32_t at = (uint32_t)(unit * T::UNIT + i * 16 * (int)LINE) + x_off;
            fx[h][i].lo = *reinterpret_cast<const u32x4*>(lds + at);
            fx[h][i].hi = *reinterpret_cast<const u32x4*>(lds + (at ^ 64u));
        }
    };
    auto read_w = [&](int h, int unit) {
#pragma unroll
        for (int i = 0; i < NH; ++i) {
            const uint32_t at = (uint32_t)(unit * T::UNIT + i * 16 * (int)LINE) + w_off;
            fw[h][i].lo = *reinterpret_cast<const u32x4*>(lds + at);
            fw[h][i].hi = *reinterpret_cast<const u32x4*>(lds + (at ^ 64u));
        }
    };
    f32x4 acc[2][MH][2][NH];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < MH; ++i) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
#pragma unroll
                for (int j = 0; j < NH; ++j) {
                    acc[h][i][q][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                }
            }
        }
    }
    auto quarter = [&](int hx, int hw) {
#pragma unroll
        for (int i = 0; i < MH; ++i) {
#pragma unroll
            for (int j = 0; j < NH; ++j) {
                acc[hx][i][hw][j] = product<P>(fw[hw][j], fx[hx][i], acc[hx][i][hw][j]);
            }
        }
    };
    // Waits until this wave's reads are done and all but the `later` youngest of its loads have landed, then
    // for the other waves.
    auto meet = [&](bool two_units_behind) {
        __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0)
        if (two_units_behind) {
            asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * T::LOADS) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    // Units: Y of an even stage 0, X 1; of an odd stage 2 and 3.
    auto stage = [&](uint32_t s, auto parity) {
        constexpr int p = decltype(parity)::value, Y = 2 * p, X = Y + 1, Y_NEXT = 2 - 2 * p;
        meet(s + 1u < steps);                       // X of this stage has landed; Y's place is free
        if (s + 2u < steps) {
            ask(s + 2u, 0, p, Y);
        }
        read_w(1 - p, X);
        __builtin_amdgcn_sched_barrier(0);
        quarter(0, p);
        __builtin_amdgcn_sched_barrier(0);
        read_x(1, X);
        __builtin_amdgcn_sched_barrier(0);
        quarter(0, 1 - p);
        __builtin_amdgcn_sched_barrier(0);
        meet(s + 2u < steps);                       // Y of the next stage has landed; X's place is free
        if (s + 2u < steps) {
            ask(s + 2u, 1, 1 - p, X);
        }
        if (s + 1u < steps) {
            read_x(0, Y_NEXT);
        }
        __builtin_amdgcn_sched_barrier(0);
        quarter(1, 1 - p);
        __builtin_amdgcn_sched_barrier(0);
        if (s + 1u < steps) {
            read_w(1 - p, Y_NEXT);
        }
        __builtin_amdgcn_sched_barrier(0);
        quarter(1, p);
        __builtin_amdgcn_sched_barrier(0);
    };
    if (steps != 0u) {
        ask(0, 0, 0, 0);
        ask(0, 1, 1, 1);
        if (steps > 1u) {
            ask(1, 0, 1, 2);
            ask(1, 1, 0, 3);
            asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(3 * T::LOADS) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        }
        read_x(0, 0);
        read_w(0, 0);
        uint32_t s = 0;
        for (; s + 1u < steps; s += 2u) {
            stage(s, Parity<0>{});
            stage(s + 1u, Parity<1>{});
        }
        if (s < steps) {
            stage(s, Parity<0>{});
        }
    }

    if (a.splits > 1u) {
        // The parts' sums meet in the workspace, a lane's where its lane of every other part finds them; the
        // last part to arrive adds them in order.
        const uint64_t block = (uint64_t)T::BM * T::BN / 2u;   // 64-bit words
        const uint64_t mine = ((uint64_t)tile * a.splits + split) * block + (uint64_t)tid;
        uint32_t q = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < MH; ++i) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int j = 0; j < NH; ++j) {
                        const f32x4 v = acc[h][i][e][j];
                        handed_store(a.part, mine + (uint64_t)q * 512u,
                                     (uint64_t)lilym_f32_bits(v[0]) | (uint64_t)lilym_f32_bits(v[1]) << 32);
                        handed_store(a.part, mine + (uint64_t)q * 512u + 256u,
                                     (uint64_t)lilym_f32_bits(v[2]) | (uint64_t)lilym_f32_bits(v[3]) << 32);
                        ++q;
                    }
                }
            }
        }
        if (!last_to_arrive(a.ticket + tile, a.splits, last, a.relaxed != 0u)) {
            return;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < MH; ++i) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int j = 0; j < NH; ++j) {
                        acc[h][i][e][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                    }
                }
            }
        }
        for (uint32_t part = 0; part < a.splits; ++part) {
            const uint64_t at = ((uint64_t)tile * a.splits + part) * block + (uint64_t)tid;
            q = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int i = 0; i < MH; ++i) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
#pragma unroll
                        for (int j = 0; j < NH; ++j) {
                            const uint64_t u = handed_load(a.part, at + (uint64_t)q * 512u);
                            const uint64_t v = handed_load(a.part, at + (uint64_t)q * 512u + 256u);
                            acc[h][i][e][j] += f32x4{lilym_bits_f32((uint32_t)u), lilym_bits_f32((uint32_t)(u >> 32)),
                                                     lilym_bits_f32((uint32_t)v), lilym_bits_f32((uint32_t)(v >> 32))};
                            ++q;
                        }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int j = 0; j < NH; ++j) {
            const uint32_t v = n0 + wn * (uint32_t)(T::NT * 16) + (uint32_t)((e * NH + j) * 16) + g * 4u;
            const Columns c = columns_at(a, v);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int i = 0; i < MH; ++i) {
                    const uint32_t r = m0 + wm * (uint32_t)(T::MT * 16) + (uint32_t)((h * MH + i) * 16) + r16;
                    if (r < a.rows) {
                        finish(a, r, v, c, a.x_scales != nullptr ? gload(a.x_scales + r) : 1.0f, acc[h][i][e][j]);
                    }
                }
            }
        }
    }
}

template <class T>
hipError_t launch_tile(hipStream_t stream, ProjectArgs& a, bool e4m3, uint64_t part_words, uint32_t tickets, uint32_t handover) {
    const uint32_t m_tiles = (a.rows + T::BM - 1u) / T::BM, n_tiles = (a.n + T::BN - 1u) / T::BN;
    const uint64_t tiles = (uint64_t)m_tiles * n_tiles;
    const uint32_t stages = (a.d_bytes + LINE - 1u) / LINE;
    // Parts of d: enough to fill the chip once, none shorter than eight stages, what the workspace holds.
    uint32_t splits = 1;
    const uint32_t places = 256u * T::RESIDENT;
    while (splits < 16u && tiles * splits * 2u <= places && stages / (splits * 2u) >= 8u && tiles <= tickets &&
           tiles * (splits * 2u) * (T::BM * T::BN / 2u) <= part_words) {
        splits *= 2u;
    }
    a.splits = splits;
    a.relaxed = handover == 2u || (handover == 0u && tiles * splits > 256u) ? 1u : 0u;
    const dim3 grid((uint32_t)(tiles * splits)), block(256);
    auto go = [&](const void* kernel, LdsAllowed& allowed, auto launch) -> hipError_t {
        const hipError_t e = allowed.say(kernel, T::LDS_BYTES);
        if (e == hipSuccess) {
            launch();
        }
        return e;
    };
    static LdsAllowed allowed[3];
    hipError_t e;
    if (!e4m3) {
        e = go((const void*)k_project_tiles<PRODUCT_BF16, T>, allowed[0], [&] {
            hipLaunchKernelGGL((k_project_tiles<PRODUCT_BF16, T>), grid, block, T::LDS_BYTES, stream, a, m_tiles, n_tiles);
        });
    } else if (a.out_bf16) {
        e = go((const void*)k_project_tiles<PRODUCT_E4M3, T>, allowed[1], [&] {
            hipLaunchKernelGGL((k_project_tiles<PRODUCT_E4M3, T>), grid, block, T::LDS_BYTES, stream, a, m_tiles, n_tiles);
        });
    } else {
        e = go((const void*)k_project_tiles<PRODUCT_E4M3_WIDE, T>, allowed[2], [&] {
            hipLaunchKernelGGL((k_project_tiles<PRODUCT_E4M3_WIDE, T>), grid, block, T::LDS_BYTES, stream, a, m_tiles, n_tiles);
        });
    }
    if (e != hipSuccess) {
        return e;
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_project_tiles(hipStream_t stream, ProjectArgs& a, bool e4m3, uint64_t part_words, uint32_t tickets,
                                uint32_t handover) {
    const uint64_t big = (uint64_t)((a.rows + 255u) / 256u) * ((a.n + 255u) / 256u);
    if (a.rows > 128u && big >= 128u) {
        return launch_tile<Tile<2, 2, 8, 8, 1>>(stream, a, e4m3, part_words, tickets, handover);
    }
    if (a.rows > 64u) {
        return launch_tile<Tile<2, 2, 4, 4, 2>>(stream, a, e4m3, part_words, tickets, handover);
    }
    return launch_tile<Tile<1, 4, 4, 2, 2>>(stream, a, e4m3, part_words, tickets, handover);
}

}  // namespace lily
