// project_tile.h - the kernel of the matrix product with an epilogue for more rows: tiles on the matrix cores.
//
// Four waves share a tile of rows x outputs, each MT x NT blocks of 16 x 16 or, in the large tile, 32 x 32.  d goes by
// stages of 128 bytes a row.  A wave's block is taken in quarters, two halves of its rows against two halves of its
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
#pragma once

#include <utility>

#include "launch.h"
#include "project.h"

namespace lily {

namespace {

__device__ const uint4 line_of_zeros = {0u, 0u, 0u, 0u};   // what lies beyond d

typedef float f32x16 __attribute__((ext_vector_type(16)));

// A block of S x S sums: its operands' pieces, its products one by one, where a lane's sums lie in it.  The wide
// form has a quarter of the instructions and of the separately tracked sums (with 16 x 16 blocks a wave's 256
// registers of sums kept the compiler moving them around: 2 450 us where this takes a tenth).
template <int S>
struct Block;
template <>
struct Block<16> {
    typedef f32x4 Sums;
    static constexpr int PIECES = 2;               // a lane of a line
    u32x4 p[PIECES];
    static __device__ __forceinline__ uint32_t first_piece(uint32_t lane) { return lane >> 4; }   // then every fourth
    static constexpr uint32_t NEXT_PIECE = 64;     // in bytes of a staged row, by exclusive or
    static __device__ __forceinline__ Sums product(bf16x8 w, bf16x8 x, Sums c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x, c, 0, 0, 0); }
    static __device__ __forceinline__ Sums product(i32x8 w, i32x8 x, Sums c) {
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 0, 0, 0, 0, 0, 0);
    }
};
template <>
struct Block<32> {
    typedef f32x16 Sums;
    static constexpr int PIECES = 4;
    u32x4 p[PIECES];
    static __device__ __forceinline__ uint32_t first_piece(uint32_t lane) { return lane >> 5; }   // then every second
    static constexpr uint32_t NEXT_PIECE = 32;
    static __device__ __forceinline__ Sums product(bf16x8 w, bf16x8 x, Sums c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(w, x, c, 0, 0, 0); }
    static __device__ __forceinline__ Sums product(i32x8 w, i32x8 x, Sums c) {
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, x, c, 0, 0, 0, 0, 0, 0);
    }
};
// Products a line of a block takes, and the q-th of them.
template <Products P, int S>
constexpr int STEPS = P == PRODUCT_BF16 ? Block<S>::PIECES : P == PRODUCT_E4M3 || P == PRODUCT_BLOCKS ? Block<S>::PIECES / 2 : Block<S>::PIECES * 2;
template <Products P, int S>
__device__ __forceinline__ typename Block<S>::Sums step(const Block<S>& w, const Block<S>& x, typename Block<S>::Sums c, int q) {
    if constexpr (P == PRODUCT_BF16) {
        return Block<S>::product(__builtin_bit_cast(bf16x8, w.p[q]), __builtin_bit_cast(bf16x8, x.p[q]), c);
    } else if constexpr (P == PRODUCT_E4M3 || P == PRODUCT_BLOCKS) {
        return Block<S>::product(__builtin_bit_cast(i32x8, __builtin_shufflevector(w.p[2 * q], w.p[2 * q + 1], 0, 1, 2, 3, 4, 5, 6, 7)),
                                 __builtin_bit_cast(i32x8, __builtin_shufflevector(x.p[2 * q], x.p[2 * q + 1], 0, 1, 2, 3, 4, 5, 6, 7)), c);
    } else {
        const int e = (q & 1) * 2;
        return Block<S>::product(widened(w.p[q >> 1][e], w.p[q >> 1][e + 1]), widened(x.p[q >> 1][e], x.p[q >> 1][e + 1]), c);
    }
}

template <int S_, int WM_, int WN_, int MT_, int NT_, int RESIDENT_, int DEPTH_, bool BLOCKS_ = false>
struct Tile {
    // BLOCKS: the scales of the rows of x lie behind the stages, those of RUN stages and of the RUN stages that follow
    static constexpr bool BLOCKS = BLOCKS_;
    static constexpr int RUN = 8;
    // DEPTH: stages in LDS (an even number), RESIDENT: workgroups a compute unit is to hold
    static constexpr int S = S_, WM = WM_, WN = WN_, MT = MT_, NT = NT_, RESIDENT = RESIDENT_, DEPTH = DEPTH_;
    static constexpr int MH = MT / 2, NH = NT / 2;                     // blocks of a half
    static constexpr int BM = WM * MT * S, BN = WN * NT * S;
    static constexpr int XR = WM * MH * S, WR = WN * NH * S;           // rows of a unit: of x, of the weights
    static constexpr int UNIT = (XR + WR) * (int)LINE, WAVES = WM * WN;
    static constexpr int XL = XR / (8 * WAVES), WL = WR / (8 * WAVES), LOADS = XL + WL;  // loads of a wave and unit
    static constexpr int SCALES = BLOCKS ? BM * RUN * 4 : 0, SCALE_LOADS = BM / WAVES / 8;   // bytes of a run; loads of a wave, eight rows each
    // The epilogue's: a wave's rows that lie in LDS at once (half of the large tile's), and floats of a row there (a step of
    // four banks from row to row).
    static constexpr int PARTS = S == 32 || WM * WN == 8 ? 2 : 1, PART_ROWS = MT * S / PARTS, ROW = NT * S + 4;
    static constexpr int STAGES = 2 * DEPTH * UNIT, SPREAD = WAVES * PART_ROWS * ROW * 4;   // bytes
    static constexpr int TOUCHED = STAGES + 2 * SCALES, USED = TOUCHED + (S == 32 ? WAVES * 256 : 0);
    static constexpr int LDS_BYTES = SPREAD > USED ? SPREAD : USED;
    static_assert(DEPTH % 2 == 0 && (2 * DEPTH - 1) * LOADS < 64, "loads in flight are counted in six bits");
    static_assert(!BLOCKS || NT * S <= (int)LILY_BLOCK, "a wave's outputs are of one block");
    static_assert(!BLOCKS || (SCALE_LOADS >= 1 && SCALE_LOADS <= RUN - DEPTH), "a run's scales are asked for in time");
    static_assert(XR % (8 * WAVES) == 0 && WR % (8 * WAVES) == 0, "whole loads a wave");
    static_assert(LDS_BYTES <= 160 * 1024, "a compute unit's");
};

template <int V>
struct Constant {
    static constexpr int value = V;
};
// f of the constants 0 .. N - 1
template <class F, int... I>
__device__ __forceinline__ void each_of(F&& f, std::integer_sequence<int, I...>) {
    (f(Constant<I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F&& f) {
    each_of(f, std::make_integer_sequence<int, N>{});
}

// The epilogue: a wave's rows (of the large tile half of them at a time) through its part of LDS, so that a lane has eight
// neighbouring outputs, and the lanes of a row store it whole (256 bytes of bf16 in the large tile, where nothing else
// hides what an epilogue takes).  Its outputs are the same in every row: their scales and biases are read once, the rows go
// by a loop of few operations a value, and what the next rows read is on its way meanwhile.  (Quarters of four outputs a lane,
// rows unrolled, took 39 000 cycles a large tile of bf16 without operands, a fifth of a tile with d = 4096, and 64 000 with a
// bias, SiLU and a residual.)
// A row's 16-byte pieces from the 16th on change places in pairs: lanes 8 to 15 then read the groups of banks that lanes
// 0 to 7 leave.
template <int B>
struct Rows {     // what B rows read
    float scale[B];
    u32x4 lo[B];  // the residual as it lies in memory: eight bf16, or the first four f32
};
typedef u32x4 pj_u32x4_out __attribute__((aligned(2)));
template <class T>
__device__ __forceinline__ void give_out(const ProjectArgs& a, const typename Block<T::S>::Sums (&acc)[2][T::MH][2][T::NH], char* lds, uint32_t m,
                                         uint32_t n, uint32_t wave, uint32_t lane, uint32_t split) {
    constexpr uint32_t ROW = T::ROW, LANES = T::NT * T::S / 8, AT_ONCE = 64 / LANES, TURNS = T::MT * T::S / AT_ONCE;   // lanes of a row, rows at once
    constexpr int B = TURNS < 4 ? TURNS : 4;                                                                         // of them a batch
    constexpr uint32_t PART_TURNS = TURNS / T::PARTS;
    float* mine = reinterpret_cast<float*>(lds) + wave * ((uint32_t)T::PART_ROWS * ROW);
    const uint32_t in_row = lane % LANES, v0 = n + in_row * 8u, r0 = m + lane / LANES;
    const bool whole = v0 + 8u <= a.n;
    auto spread = [&](auto part) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        constexpr int H = 2 / T::PARTS;   // halves of the rows
        each<H * T::MH * 2 * T::NH>([&](auto b) {
            constexpr int h = b.value / (T::MH * 2 * T::NH), i = b.value / (2 * T::NH) % T::MH, e = b.value / T::NH % 2, j = b.value % T::NH;
            const auto& c = acc[part.value * H + h][i][e][j];
            float* row = mine + ((uint32_t)((h * T::MH + i) * T::S) + lane % (uint32_t)T::S) * ROW;
            each<T::S == 32 ? 4 : 1>([&](auto q) {   // runs of four outputs of a lane
                const uint32_t piece = T::S == 32 ? (uint32_t)((e * T::NH + j) * 8 + q.value * 2) + ((lane >> 5) ^ (uint32_t)((e * T::NH + j) / 2))
                                                  : (uint32_t)((e * T::NH + j) * 4) + (lane >> 4);
                *reinterpret_cast<f32x4*>(row + piece * 4u) = f32x4{c[4 * q.value], c[4 * q.value + 1], c[4 * q.value + 2], c[4 * q.value + 3]};
            });
        });
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    if constexpr (T::PARTS == 1) {
        if (a.splits > 1u) {   // a part's sums as they are; k_project_join does the rest
            __syncthreads();   // (the stages' place is the epilogue's)
            spread(Constant<0>{});
#pragma unroll 4
            for (uint32_t turn = 0; turn < TURNS; ++turn) {
                const uint32_t r = r0 + turn * AT_ONCE;
                each<2>([&](auto q) {
                    const uint32_t piece = in_row + q.value * LANES, v = n + piece * 4u;
                    if (r < a.rows && v < a.n) {
                        *(LILY_GLOBAL f32x4*)(a.part + ((uint64_t)split * a.rows + r) * part_stride(a.n) + v) =
                            *reinterpret_cast<const f32x4*>(mine + (turn * AT_ONCE + lane / LANES) * ROW + piece * 4u);
                    }
                });
            }
            return;
        }
    }
    float scale[8];
    uint32_t raw[8];   // of the bias
    each<8>([&](auto k) {
        const uint32_t v = min(v0 + k.value, a.n - 1u);
        scale[k.value] = a.w_scales != nullptr ? gload(a.w_scales + v) : 1.0f;
        raw[k.value] = 0u;
        if (a.bias != nullptr) {
            raw[k.value] = a.bias_bf16 ? (uint32_t)gload(static_cast<const uint16_t*>(a.bias) + v) << 16 : gload(static_cast<const uint32_t*>(a.bias) + v);
        }
    });
    // Rows r0 + AT_ONCE turn and B - 1 after it; and the residual's last four outputs in f32.
    auto residual_at = [&](uint32_t r, uint32_t first) {
        const uint64_t from = (uint64_t)min(r, a.rows - 1u) * a.residual_stride + v0 + first;
        const uint16_t* half = static_cast<const uint16_t*>(a.residual) + from;
        const uint32_t* word = static_cast<const uint32_t*>(a.residual) + from;
        u32x4 w;
        if (whole && a.residual_bf16) {
            w = *(const LILY_GLOBAL pj_u32x4_out*)half;
        } else if (whole) {
            w = *(const LILY_GLOBAL pj_u32x4_any*)word;
        } else {
            uint32_t e[8];
            each<8>([&](auto k) {   // (what lies behind the last output is not read)
                const uint32_t j = min((uint32_t)k.value, a.n - 1u - v0 - min(first, a.n - 1u - v0));
                e[k.value] = a.residual_bf16 ? (uint32_t)gload(half + j) : first + j < a.n - v0 ? gload(word + j) : 0u;
            });
            w = a.residual_bf16 ? u32x4{e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16} : u32x4{e[0], e[1], e[2], e[3]};
        }
        return w;
    };
    auto rows_at = [&](Rows<B>& l, uint32_t turn) {
        if (a.x_scales != nullptr) {
            each<B>([&](auto t) { l.scale[t.value] = gload(a.x_scales + min(r0 + (turn + t.value) * AT_ONCE, a.rows - 1u)); });
        }
        if (a.residual != nullptr) {
            each<B>([&](auto t) { l.lo[t.value] = residual_at(r0 + (turn + t.value) * AT_ONCE, 0u); });
        }
    };
    u32x4 hi[B];
    auto last_at = [&](uint32_t turn) {
        if (a.residual != nullptr && !a.residual_bf16) {
            each<B>([&](auto t) { hi[t.value] = residual_at(r0 + (turn + t.value) * AT_ONCE, 4u); });
        }
    };
    const uint32_t turned = in_row * 2u >> 4;
    const float* first = mine + lane / LANES * ROW + ((in_row * 2u) ^ turned) * 4u;
    const int32_t other = turned != 0u ? -4 : 4;
    auto give = [&](const Rows<B>& l, uint32_t turn) {
        float v[8 * B];
        each<B>([&](auto t) {
            const float* p = first + ((turn + t.value) % PART_TURNS * AT_ONCE) * ROW;
            const f32x4 x = *reinterpret_cast<const f32x4*>(p), y = *reinterpret_cast<const f32x4*>(p + other);
            each<8>([&](auto k) {
                const float sum = k.value < 4 ? x[k.value % 4] : y[k.value % 4];
                v[t.value * 8 + k.value] = sum * l.scale[t.value] * scale[k.value] + lilym_bits_f32(raw[k.value]);
            });
        });
        activate(v, a.act);
        if (a.residual != nullptr && a.residual_bf16) {
            each<8 * B>([&](auto e) {
                const uint32_t w = l.lo[e.value / 8][e.value % 8 / 2];
                v[e.value] += lilym_bits_f32((e.value & 1) ? w & 0xffff0000u : w << 16);
            });
        } else if (a.residual != nullptr) {
            each<8 * B>([&](auto e) {
                v[e.value] += lilym_bits_f32(e.value % 8 < 4 ? l.lo[e.value / 8][e.value % 4] : hi[e.value / 8][e.value % 4]);
            });
        }
        each<B>([&](auto t) {
            constexpr int e = t.value * 8;
            const uint32_t r = r0 + (turn + t.value) * AT_ONCE;
            if (r < a.rows) {
                const uint64_t to = (uint64_t)r * a.out_stride + v0;
                if (!whole) {
                    each<7>([&](auto k) {
                        if (v0 + k.value < a.n) {
                            if (a.out_bf16) {
                                *(LILY_GLOBAL uint16_t*)(static_cast<uint16_t*>(a.out) + to + k.value) = (uint16_t)pj_bf16_pair(v[e + k.value], 0.0f);
                            } else {
                                *(LILY_GLOBAL float*)(static_cast<float*>(a.out) + to + k.value) = v[e + k.value];
                            }
                        }
                    });
                } else if (a.out_bf16) {
                    *(LILY_GLOBAL pj_u32x4_out*)(static_cast<uint16_t*>(a.out) + to) =
                        u32x4{pj_bf16_pair(v[e], v[e + 1]), pj_bf16_pair(v[e + 2], v[e + 3]), pj_bf16_pair(v[e + 4], v[e + 5]),
                              pj_bf16_pair(v[e + 6], v[e + 7])};
                } else {
                    *(LILY_GLOBAL f32x4_any*)(static_cast<float*>(a.out) + to) = f32x4{v[e], v[e + 1], v[e + 2], v[e + 3]};
                    *(LILY_GLOBAL f32x4_any*)(static_cast<float*>(a.out) + to + 4) = f32x4{v[e + 4], v[e + 5], v[e + 6], v[e + 7]};
                }
            }
        });
    };
    // (a loop, and one copy of it: unrolled it runs once a tile and waits for its own instructions, 346 -> 400 us for 8192 x
    // 12288 x 4096 in E4M3.  More rows ahead than the next four change nothing.)
    Rows<B> now = {}, next = {};
    each<B>([&](auto t) { now.scale[t.value] = next.scale[t.value] = 1.0f; });
    auto begin = [&] {
        if (v0 < a.n) {
            rows_at(now, 0u);
            last_at(0u);
        }
    };
    if constexpr (T::PARTS == 2) {   // (the sums are in registers of their own there; the smaller tiles' would be in the way)
        begin();
    }
    __syncthreads();   // (the stages' place is the epilogue's)
    spread(Constant<0>{});
    if constexpr (T::PARTS == 1) {
        begin();
    }
#pragma unroll 1
    for (uint32_t at = 0; at < TURNS; at += (uint32_t)B) {
        uint32_t turn = at;
        asm("" : "+s"(turn));   // (an address is computed where it is used: 64 that grow with the loop took 340 registers)
        if constexpr (T::PARTS == 2) {
            if (turn == PART_TURNS) {
                spread(Constant<1>{});
            }
        }
        if (v0 < a.n) {
            const uint32_t then = min(turn + (uint32_t)B, TURNS - (uint32_t)B);
            rows_at(next, then);
            give(now, turn);
            now = next;
            last_at(then);
        }
    }
}

// A workgroup's tile and part of d.  Consecutive workgroups go to consecutive XCDs: each XCD gets a run of tiles of its own (they
// share its L2), in groups of four tiles of rows.
struct TilePlace {
    uint32_t m0, n0, split;
};
template <class T>
__device__ __forceinline__ TilePlace place_of(const ProjectArgs& a, uint32_t m_tiles, uint32_t n_tiles) {
    const uint32_t tiles = m_tiles * n_tiles, all = tiles * a.splits;
    const uint32_t xcd = blockIdx.x & 7u, slot = blockIdx.x >> 3, each = all / 8u, more = all % 8u;
    const uint32_t job = xcd * each + min(xcd, more) + slot;
    const uint32_t split = job / tiles, tile = job % tiles;
    constexpr uint32_t GROUP_M = 4;
    const uint32_t band = tile / (GROUP_M * n_tiles), in_band = tile % (GROUP_M * n_tiles);
    const uint32_t band_m = min(GROUP_M, m_tiles - band * GROUP_M);
    return {(band * GROUP_M + in_band % band_m) * (uint32_t)T::BM, in_band / band_m * (uint32_t)T::BN, split};
}

template <Products P, class T>
__global__ void __launch_bounds__(64 * T::WAVES, T::RESIDENT * T::WAVES / 4) k_project_tiles(const ProjectArgs a, uint32_t m_tiles, uint32_t n_tiles) {
    constexpr int MH = T::MH, NH = T::NH, S = T::S, DEPTH = T::DEPTH;
    typedef Block<S> Operand;
    typedef typename Operand::Sums Sums;
    extern __shared__ __align__(16) char lds[];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
    const uint32_t wm = wave / T::WN, wn = wave % T::WN, r_in = lane % (uint32_t)S;
    const TilePlace place = place_of<T>(a, m_tiles, n_tiles);
    const uint32_t split = place.split, m0 = place.m0, n0 = place.n0;

    const uint32_t stages_all = (a.d_bytes + LINE - 1u) / LINE;
    const uint32_t per = stages_all / a.splits, over = stages_all % a.splits;
    const uint32_t first = split * per + min(split, over), steps = per + (split < over ? 1u : 0u);

    // Where a lane's pieces come from: 32-bit offsets from the tile's first rows, for both halves.
    const char* x_rows = a.x + (uint64_t)m0 * a.x_stride;
    const char* w_rows = a.w + (uint64_t)n0 * a.w_stride;
    uint32_t x_at[2][T::XL], w_at[2][T::WL];
#pragma unroll
    for (int i = 0; i < T::LOADS; ++i) {
        const bool is_x = i < T::XL;
        const uint32_t row = (uint32_t)((is_x ? i : i - T::XL) * 8 * T::WAVES) + wave * 8u + (lane >> 3);   // of the unit's part
        const uint32_t piece = (lane & 7u) ^ ((row >> 1) & 7u);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t half = is_x ? (uint32_t)(MH * S) : (uint32_t)(NH * S);
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
    // (buffer loads: a lane's offset and the stage's are added by the load itself; the last 32 bits of the resource
    // are a raw buffer's, and nothing is ever asked beyond the rows)
    auto x_buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(x_rows), 0, -1, 0x00020000);
    auto w_buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(w_rows), 0, -1, 0x00020000);
    // Scales of the rows of x: a load brings those of eight rows for a run of stages, eight neighbouring floats a row (a load of
    // one stage's, a line of memory for every lane, takes as long as all of the stage's operands).  A row's eight change places by the
    // row's number, so that lanes that read one stage's of neighbouring rows meet different banks.
    WeightScales w_scales = {};
    if constexpr (T::BLOCKS) {
        const uint32_t block = min((n0 + wn * (uint32_t)(T::NT * S)) / LILY_BLOCK, (a.n - 1u) / LILY_BLOCK);
        w_scales = {a.w_blocks + (uint64_t)block * a.w_blocks_stride + first, steps, 0.0f};
        w_scales.ask(0u);
    }
    auto load_scales = [&](uint32_t run, int k) {
        const uint32_t row = wave * (uint32_t)(T::SCALE_LOADS * 8) + (uint32_t)k * 8u, in = row + (lane >> 3);
        const uint32_t stage = min(run * (uint32_t)T::RUN + ((lane & 7u) ^ ((in >> 3) & 7u)), steps - 1u);
        const float* from = a.x_blocks + (uint64_t)min(m0 + in, a.rows - 1u) * a.x_blocks_stride + first + stage;
        __builtin_amdgcn_global_load_lds((gptr)from, (lptr)(lds + T::STAGES + (run & 1u) * (uint32_t)T::SCALES + row * (uint32_t)(T::RUN * 4)), 4, 0, 0);
    };
    auto load = [&](uint32_t s, int hx, int hw, int unit, int i) {
        const uint32_t k0 = (first + s) * LINE;
        char* base = lds + unit * T::UNIT + wave * 1024u + i * (1024 * T::WAVES);
        if (i < T::XL) {
            __builtin_amdgcn_raw_ptr_buffer_load_lds(x_buffer, (lptr)base, 16, (int)x_at[hx][i < T::XL ? i : 0], (int)k0, 0, 0);
        } else {
            __builtin_amdgcn_raw_ptr_buffer_load_lds(w_buffer, (lptr)base, 16, (int)w_at[hw][i < T::XL ? 0 : i - T::XL], (int)k0, 0, 0);
        }
    };
    auto ask = [&](uint32_t s, int hx, int hw, int unit) {
        const uint32_t k0 = (first + s) * LINE;
        if (k0 + LINE <= a.d_bytes) {
#pragma unroll
            for (int i = 0; i < T::LOADS; ++i) {
                load(s, hx, hw, unit, i);
            }
            return;
        }
        // the stage that d ends in: pieces beyond it are zeros
        char* base = lds + unit * T::UNIT + wave * 1024u;
        const char* zeros = reinterpret_cast<const char*>(&line_of_zeros);
#pragma unroll
        for (int i = 0; i < T::LOADS; ++i) {
            const char* from = i < T::XL ? x_rows + k0 + (uint64_t)x_at[hx][i < T::XL ? i : 0]
                                         : w_rows + k0 + (uint64_t)w_at[hw][i < T::XL ? 0 : i - T::XL];
            const uint32_t row = (uint32_t)((i < T::XL ? i : i - T::XL) * 8 * T::WAVES) + wave * 8u + (lane >> 3);
            from = k0 + ((lane & 7u) ^ ((row >> 1) & 7u)) * 16u < a.d_bytes ? from : zeros;
            __builtin_amdgcn_global_load_lds((gptr)from, (lptr)(base + i * (1024 * T::WAVES)), 16, 0, 0);
        }
    };
    // A lane's operands out of a unit.
    const uint32_t off = r_in * LINE + ((Operand::first_piece(lane) ^ ((r_in >> 1) & 7u)) << 4);
    const uint32_t x_off = wm * (uint32_t)(MH * S) * LINE + off, w_off = (uint32_t)T::XR * LINE + wn * (uint32_t)(NH * S) * LINE + off;
    Operand fx[2][MH], fw[2][NH];
    // the k-th read of a half
    constexpr int XPIECES = MH * Operand::PIECES, XREADS = XPIECES + (T::BLOCKS ? MH : 0), WREADS = NH * Operand::PIECES;
    float scale[2][MH];   // of the rows of x
    auto read = [&](Operand* f, uint32_t from, int k) {
        const int i = k / Operand::PIECES, q = k % Operand::PIECES;
        f[i].p[q] = *reinterpret_cast<const u32x4*>(lds + ((from + (uint32_t)(i * S * (int)LINE)) ^ ((uint32_t)q * Operand::NEXT_PIECE)));
    };
    auto read_x = [&](int h, int unit, int k, uint32_t s) {   // (s: the stage that they are of)
        if constexpr (T::BLOCKS) {
            if (k >= XPIECES) {
                const uint32_t row = wm * (uint32_t)(T::MT * S) + (uint32_t)(h * MH * S + (k - XPIECES) * S) + r_in;
                scale[h][k - XPIECES] = *reinterpret_cast<const float*>(lds + T::STAGES + (s / (uint32_t)T::RUN & 1u) * (uint32_t)T::SCALES +
                                                                        (row * (uint32_t)T::RUN + ((s & 7u) ^ ((row >> 3) & 7u))) * 4u);
                return;
            }
        }
        read(fx[h], (uint32_t)(unit * T::UNIT) + x_off, k);
    };
    auto read_w = [&](int h, int unit, int k) { read(fw[h], (uint32_t)(unit * T::UNIT) + w_off, k); };
    Sums acc[2][MH][2][NH];
    auto clear = [&] {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < MH; ++i) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int j = 0; j < NH; ++j) {
                        acc[h][i][e][j] = Sums(0.0f);
                    }
                }
            }
        }
    };
    clear();
    // A quarter's products, one by one, `reads` reads and `loads` loads spread between the first of them: the
    // matrix pipe is never without work while they are issued.
    // (With scales a line's sums are formed by themselves, and scaled into the tile's while the next quarter's are: what waits
    // for a product's sums waits for the matrix pipe.  `turn`: the places of both.)
    Sums line[2][T::BLOCKS ? MH * NH : 1];
    float by[MH];      // of the line that waits
    auto add = [&](int hx, int hw, int turn, int b) {
        const int i = b / NH, j = b % NH;
#pragma unroll
        for (int e = 0; e < (int)(sizeof(Sums) / 4); ++e) {
            acc[hx][i][hw][j][e] = __builtin_fmaf(line[turn][b][e], by[i], acc[hx][i][hw][j][e]);
        }
    };
    if constexpr (T::BLOCKS) {
#pragma unroll
        for (int i = 0; i < MH; ++i) {
            by[i] = 0.0f;
        }
#pragma unroll
        for (int b = 0; b < MH * NH; ++b) {
            line[1][b] = Sums(0.0f);
        }
    }
    auto quarter = [&](int hx, int hw, int reads, auto&& read_one, int loads, auto&& load_one, int turn, int waits_x, int waits_w, float w) {
        constexpr int STEP = STEPS<P, S>, ALL = STEP * MH * NH;
        float next_by[MH];
        if constexpr (T::BLOCKS) {
#pragma unroll
            for (int i = 0; i < MH; ++i) {
                next_by[i] = scale[hx][i] * w;
            }
        }
#pragma unroll
        for (int t = 0; t < ALL; ++t) {
            const int q = t / (MH * NH), i = t / NH % MH, j = t % NH;
#pragma unroll
            for (int k = 0; k < reads; ++k) {
                if (k * ALL / reads / 2 == t) {
                    read_one(k);
                }
            }
#pragma unroll
            for (int k = 0; k < loads; ++k) {
                if (k * ALL / loads == t) {
                    load_one(k);
                }
            }
            if constexpr (T::BLOCKS) {
                line[turn][i * NH + j] = step<P, S>(fw[hw][j], fx[hx][i], q == 0 ? Sums(0.0f) : line[turn][i * NH + j], q);
                if (q == 0) {
                    add(waits_x, waits_w, 1 - turn, t);
                }
            } else {
                acc[hx][i][hw][j] = step<P, S>(fw[hw][j], fx[hx][i], acc[hx][i][hw][j], q);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (T::BLOCKS) {
#pragma unroll
            for (int i = 0; i < MH; ++i) {
                by[i] = next_by[i];
            }
        }
    };
    auto nothing = [](int) {};
    // Waits until this wave's reads are done and all but the youngest of its loads have landed (those of the
    // DEPTH - 1 stages behind; `full` false: all of them), then for the other waves.
    auto meet = [&](bool full) {
        __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0)
        if (full) {
            asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * (DEPTH - 1) * T::LOADS) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    // Stage s, at place `at` of the DEPTH stages: unit Y at 2 at, X behind it.  `inner`: DEPTH more whole stages follow.
    // (The reads of a stage past the last find what lies there; nothing is made of them.)
    auto stage = [&](uint32_t s, auto place, auto inner) {
        constexpr int at = decltype(place)::value, p = at & 1, Y = 2 * at, X = Y + 1, Y_NEXT = 2 * ((at + 1) % DEPTH);
        constexpr bool INNER = decltype(inner)::value != 0;
        constexpr int LOADS = INNER ? T::LOADS : 0;
        constexpr uint32_t D = DEPTH;
        float w = 1.0f;
        if constexpr (T::BLOCKS) {
            if (s != 0u && (s & 63u) == 0u) {
                w_scales.ask(s);
                w_scales.settle();
            }
            w = w_scales.of(s);
        }
        meet(INNER || s + D <= steps);              // X of this stage has landed; Y's place is free
        if constexpr (T::BLOCKS) {   // (so is that of the scales of the run before; the waits count these as loads, and so wait for more)
            const uint32_t run = s / (uint32_t)T::RUN + 1u, k = s % (uint32_t)T::RUN;
            if (k < (uint32_t)T::SCALE_LOADS && run * (uint32_t)T::RUN < steps) {
                load_scales(run, (int)k);
            }
        }
        if constexpr (!INNER) {
            if (s + D < steps) {
                ask(s + D, 0, p, Y);
            }
        }
        quarter(0, p, WREADS, [&](int k) { read_w(1 - p, X, k); }, LOADS, [&](int k) { load(s + D, 0, p, Y, k); }, 0, 1, 1 - p, w);
        quarter(0, 1 - p, XREADS, [&](int k) { read_x(1, X, k, s); }, 0, nothing, 1, 0, p, w);
        meet(INNER || s + D < steps);               // Y of the next stage has landed; X's place is free
        if constexpr (!INNER) {
            if (s + D < steps) {
                ask(s + D, 1, 1 - p, X);
            }
        }
        quarter(1, 1 - p, XREADS, [&](int k) { read_x(0, Y_NEXT, k, s + 1u); }, LOADS, [&](int k) { load(s + D, 1, 1 - p, X, k); }, 0, 0, 1 - p, w);
        quarter(1, p, WREADS, [&](int k) { read_w(1 - p, Y_NEXT, k); }, 0, nothing, 1, 1, 1 - p, w);
    };
    // (everything that has to be a constant of a stage is one: DEPTH stages one after the other)
    auto stages = [&](uint32_t s, auto inner) {
        auto one = [&](auto place) {
            if constexpr (decltype(place)::value < DEPTH) {
                if (decltype(inner)::value != 0 || s + (uint32_t)decltype(place)::value < steps) {
                    stage(s + (uint32_t)decltype(place)::value, place, inner);
                }
            }
        };
        one(Constant<0>{});
        one(Constant<1>{});
        one(Constant<2>{});
        one(Constant<3>{});
        one(Constant<4>{});
        one(Constant<5>{});
    };
    static_assert(DEPTH <= 6, "stages() lists six");
    if constexpr (T::BLOCKS) {
#pragma unroll
        for (int k = 0; k < T::SCALE_LOADS; ++k) {
            load_scales(0u, k);
        }
    }
#pragma unroll
    for (int j = 0; j < DEPTH; ++j) {
        if ((uint32_t)j < steps) {
            ask((uint32_t)j, 0, j & 1, 2 * j);
            ask((uint32_t)j, 1, 1 - (j & 1), 2 * j + 1);
        }
    }
    if (steps >= (uint32_t)DEPTH) {
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((2 * DEPTH - 1) * T::LOADS) : "memory");
    } else {
        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    }
#pragma unroll
    for (int k = 0; k < XREADS; ++k) {
        read_x(0, 0, k, 0u);
    }
#pragma unroll
    for (int k = 0; k < WREADS; ++k) {
        read_w(0, 0, k);
    }
    if constexpr (T::BLOCKS) {
        w_scales.settle();
    }
    uint32_t s = 0;
    // The residual's lines are asked for, to nobody's use, ten stages before the epilogue reads them: all tiles read and write
    // at once there, and what comes from memory then is waited for (8192 x 4096 x 4096 bf16 with bias, SiLU and residual
    // 254 us without, 249 at the tile's beginning, 245 so).  What they fetch goes to a place of LDS that only the epilogue has
    // a use for, behind the last stages' wait for every load; the waits before count them as loads, and so wait for more.
    constexpr uint32_t TOUCH = 10;
    const bool touches = a.residual != nullptr && m0 + (uint32_t)T::BM <= a.rows && n0 + (uint32_t)T::BN <= a.n;
    auto touch = [&] {
        const uint32_t e = a.residual_bf16 ? 2u : 4u, lines = (uint32_t)(T::NT * S) * e / LINE;   // lines of a wave's outputs of a row
        for (uint32_t k = 0; k < (uint32_t)(T::MT * S) / 64u * lines; ++k) {
            const uint32_t at = k * 64u + lane, row = m0 + wm * (uint32_t)(T::MT * S) + at / lines;
            // (rows may start at any element: the first whole word of what a line holds of a row)
            const uintptr_t p = (reinterpret_cast<uintptr_t>(a.residual) + ((uint64_t)row * a.residual_stride + n0 + wn * (uint32_t)(T::NT * S)) * e + at % lines * LINE + 3u) & ~(uintptr_t)3u;
            __builtin_amdgcn_global_load_lds((gptr)p, (lptr)(lds + T::TOUCHED + wave * 256u), 4, 0, 0);
        }
    };
    const uint32_t touch_at = steps > TOUCH ? (steps - TOUCH) / DEPTH * DEPTH : 0u;
    for (; s + 2u * DEPTH < steps; s += DEPTH) {   // (what these ask for is whole: the stage that d may end in is a later one)
        stages(s, Constant<1>{});
        if constexpr (S == 32) {
            if (s == touch_at && touches) {
                touch();
            }
        }
    }
    for (; s < steps; s += DEPTH) {
        stages(s, Constant<0>{});
    }
    if constexpr (T::BLOCKS) {   // what still waits: the last stage's last quarter
        auto rest = [&](auto p) {
#pragma unroll
            for (int b = 0; b < MH * NH; ++b) {
                add(1, decltype(p)::value, 1, b);
            }
        };
        if ((steps & 1u) != 0u) {
            rest(Constant<0>{});
        } else {
            rest(Constant<1>{});
        }
    }
    give_out<T>(a, acc, lds, m0 + wm * (uint32_t)(T::MT * S), n0 + wn * (uint32_t)(T::NT * S), wave, lane, split);
}

}  // namespace

}  // namespace lily
