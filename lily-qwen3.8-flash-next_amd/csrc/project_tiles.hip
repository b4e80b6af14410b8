// project_tiles.hip - the matrix product with an epilogue for more rows: tiles on the matrix cores.
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
//
// Measured (cycles of a 256 x 256 tile, 8192 x 4096 x 4096 in bf16): 4 300 until the first stage is there, 146 000 for 64
// stages, of which the matrix pipe is busy 131 000, and the epilogue, in which all compute units write at once.  212 to 224 us by
// the box, 1.30 to 1.23 PFLOP/s, at 1.8 GHz (the clock follows the power the products take; a large library product runs at
// 1.59 PFLOP/s); with a bf16 residual 236, with bias, SiLU and residual 245 to 253; 8192 x 8192 x 8192 774 to 808 us, 1.42 to 1.36;
// 8192 x 12 288 x 4096 in E4M3 340 us, 2.43 (3.21), widened for an f32 output 685.
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
constexpr int STEPS = P == PRODUCT_BF16 ? Block<S>::PIECES : P == PRODUCT_E4M3 ? Block<S>::PIECES / 2 : Block<S>::PIECES * 2;
template <Products P, int S>
__device__ __forceinline__ typename Block<S>::Sums step(const Block<S>& w, const Block<S>& x, typename Block<S>::Sums c, int q) {
    if constexpr (P == PRODUCT_BF16) {
        return Block<S>::product(__builtin_bit_cast(bf16x8, w.p[q]), __builtin_bit_cast(bf16x8, x.p[q]), c);
    } else if constexpr (P == PRODUCT_E4M3) {
        return Block<S>::product(__builtin_bit_cast(i32x8, __builtin_shufflevector(w.p[2 * q], w.p[2 * q + 1], 0, 1, 2, 3, 4, 5, 6, 7)),
                                 __builtin_bit_cast(i32x8, __builtin_shufflevector(x.p[2 * q], x.p[2 * q + 1], 0, 1, 2, 3, 4, 5, 6, 7)), c);
    } else {
        const int e = (q & 1) * 2;
        return Block<S>::product(widened(w.p[q >> 1][e], w.p[q >> 1][e + 1]), widened(x.p[q >> 1][e], x.p[q >> 1][e + 1]), c);
    }
}

template <int S_, int WM_, int WN_, int MT_, int NT_, int RESIDENT_, int DEPTH_>
struct Tile {
    // DEPTH: stages in LDS (an even number), RESIDENT: workgroups a compute unit is to hold
    static constexpr int S = S_, WM = WM_, WN = WN_, MT = MT_, NT = NT_, RESIDENT = RESIDENT_, DEPTH = DEPTH_;
    static constexpr int MH = MT / 2, NH = NT / 2;                     // blocks of a half
    static constexpr int BM = WM * MT * S, BN = WN * NT * S;
    static constexpr int XR = WM * MH * S, WR = WN * NH * S;           // rows of a unit: of x, of the weights
    static constexpr int UNIT = (XR + WR) * (int)LINE;
    static constexpr int XL = XR / 32, WL = WR / 32, LOADS = XL + WL;  // loads of a wave and unit
    // The epilogue's: a wave's rows that lie in LDS at once (half of the large tile's), and floats of a row there (a step of
    // four banks from row to row).
    static constexpr int PARTS = S == 32 ? 2 : 1, PART_ROWS = MT * S / PARTS, ROW = NT * S + 4;
    static constexpr int STAGES = 2 * DEPTH * UNIT, SPREAD = 4 * PART_ROWS * ROW * 4;   // bytes
    static constexpr int LDS_BYTES = SPREAD > STAGES ? SPREAD : STAGES;
    static_assert(DEPTH % 2 == 0 && (2 * DEPTH - 1) * LOADS < 64, "loads in flight are counted in six bits");
    static_assert(WM * WN == 4 && XR % 32 == 0 && WR % 32 == 0, "whole loads a wave");
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

template <Products P, class T>
__global__ void __launch_bounds__(256, T::RESIDENT) k_project_tiles(const ProjectArgs a, uint32_t m_tiles, uint32_t n_tiles) {
    constexpr int MH = T::MH, NH = T::NH, S = T::S, DEPTH = T::DEPTH;
    typedef Block<S> Operand;
    typedef typename Operand::Sums Sums;
    extern __shared__ __align__(16) char lds[];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
    const uint32_t wm = wave / T::WN, wn = wave % T::WN, r_in = lane % (uint32_t)S;
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
    uint32_t x_at[2][T::XL], w_at[2][T::WL];
#pragma unroll
    for (int i = 0; i < T::LOADS; ++i) {
        const bool is_x = i < T::XL;
        const uint32_t row = (uint32_t)((is_x ? i : i - T::XL) * 32) + wave * 8u + (lane >> 3);   // of the unit's part
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
    auto load = [&](uint32_t s, int hx, int hw, int unit, int i) {
        const uint32_t k0 = (first + s) * LINE;
        char* base = lds + unit * T::UNIT + wave * 1024u + i * 4096;
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
            const uint32_t row = (uint32_t)((i < T::XL ? i : i - T::XL) * 32) + wave * 8u + (lane >> 3);
            from = k0 + ((lane & 7u) ^ ((row >> 1) & 7u)) * 16u < a.d_bytes ? from : zeros;
            __builtin_amdgcn_global_load_lds((gptr)from, (lptr)(base + i * 4096), 16, 0, 0);
        }
    };
    // A lane's operands out of a unit.
    const uint32_t off = r_in * LINE + ((Operand::first_piece(lane) ^ ((r_in >> 1) & 7u)) << 4);
    const uint32_t x_off = wm * (uint32_t)(MH * S) * LINE + off, w_off = (uint32_t)T::XR * LINE + wn * (uint32_t)(NH * S) * LINE + off;
    Operand fx[2][MH], fw[2][NH];
    // the k-th read of a half
    constexpr int XREADS = MH * Operand::PIECES, WREADS = NH * Operand::PIECES;
    auto read = [&](Operand* f, uint32_t from, int k) {
        const int i = k / Operand::PIECES, q = k % Operand::PIECES;
        f[i].p[q] = *reinterpret_cast<const u32x4*>(lds + ((from + (uint32_t)(i * S * (int)LINE)) ^ ((uint32_t)q * Operand::NEXT_PIECE)));
    };
    auto read_x = [&](int h, int unit, int k) { read(fx[h], (uint32_t)(unit * T::UNIT) + x_off, k); };
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
    auto quarter = [&](int hx, int hw, int reads, auto&& read_one, int loads, auto&& load_one) {
        constexpr int STEP = STEPS<P, S>, ALL = STEP * MH * NH;
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
            acc[hx][i][hw][j] = step<P, S>(fw[hw][j], fx[hx][i], acc[hx][i][hw][j], q);
            __builtin_amdgcn_sched_barrier(0);
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
        meet(INNER || s + D <= steps);              // X of this stage has landed; Y's place is free
        if constexpr (!INNER) {
            if (s + D < steps) {
                ask(s + D, 0, p, Y);
            }
        }
        quarter(0, p, WREADS, [&](int k) { read_w(1 - p, X, k); }, LOADS, [&](int k) { load(s + D, 0, p, Y, k); });
        quarter(0, 1 - p, XREADS, [&](int k) { read_x(1, X, k); }, 0, nothing);
        meet(INNER || s + D < steps);               // Y of the next stage has landed; X's place is free
        if constexpr (!INNER) {
            if (s + D < steps) {
                ask(s + D, 1, 1 - p, X);
            }
        }
        quarter(1, 1 - p, XREADS, [&](int k) { read_x(0, Y_NEXT, k); }, LOADS, [&](int k) { load(s + D, 1, 1 - p, X, k); });
        quarter(1, p, WREADS, [&](int k) { read_w(1 - p, Y_NEXT, k); }, 0, nothing);
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
        read_x(0, 0, k);
    }
#pragma unroll
    for (int k = 0; k < WREADS; ++k) {
        read_w(0, 0, k);
    }
    uint32_t s = 0;
    // The residual's lines are asked for, to nobody's use, ten stages before the epilogue reads them: all tiles read and write
    // at once there, and what comes from memory then is waited for (8192 x 4096 x 4096 bf16 with bias, SiLU and residual
    // 254 us without, 249 at the tile's beginning, 245 so).  What they fetch goes to a place of LDS that only the epilogue has
    // a use for, behind the last stages' wait for every load; the waits before count them as loads, and so wait for more.
    constexpr uint32_t TOUCH = 10;
    const bool touches = a.residual != nullptr && m0 + (uint32_t)T::BM <= a.rows && n0 + (uint32_t)T::BN <= a.n;
    auto touch = [&] {
        static_assert(T::STAGES + 1024 <= T::LDS_BYTES || S != 32, "a place for them");
        const uint32_t e = a.residual_bf16 ? 2u : 4u, lines = e;   // lines of a wave's 128 outputs of a row
        for (uint32_t k = 0; k < 2u * lines; ++k) {
            const uint32_t at = k * 64u + lane, row = m0 + wm * 128u + at / lines;
            // (rows may start at any element: the first whole word of what a line holds of a row)
            const uintptr_t p = (reinterpret_cast<uintptr_t>(a.residual) + ((uint64_t)row * a.residual_stride + n0 + wn * 128u) * e + at % lines * LINE + 3u) & ~(uintptr_t)3u;
            __builtin_amdgcn_global_load_lds((gptr)p, (lptr)(lds + T::STAGES + wave * 256u), 4, 0, 0);
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
    give_out<T>(a, acc, lds, m0 + wm * (uint32_t)(T::MT * S), n0 + wn * (uint32_t)(T::NT * S), wave, lane, split);
}

// The parts of d joined: a thread adds four neighbouring outputs of a row over the parts, in order, and finishes them.
__global__ void __launch_bounds__(256) k_project_join(const ProjectArgs a) {
    const uint32_t fours = part_stride(a.n) / 4u;
    const uint64_t at = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    if (at >= (uint64_t)fours * a.rows) {
        return;
    }
    const uint32_t r = (uint32_t)(at / fours), v = (uint32_t)(at % fours) * 4u;
    Columns c;
    Finish f;
    c.load(a, v);
    f.load(a, r, v);
    const float* from = a.part + (uint64_t)r * part_stride(a.n) + v;
    const uint64_t next = (uint64_t)a.rows * part_stride(a.n);
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t q = 0; q < a.splits; q += 4u) {
        f32x4 p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            p[j] = gload(reinterpret_cast<const f32x4*>(from + min(q + (uint32_t)j, a.splits - 1u) * next));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (q + (uint32_t)j < a.splits) {
                sum += p[j];
            }
        }
    }
    f.store(a, r, v, c, sum);
}

template <class T>
hipError_t launch_tile(hipStream_t stream, const ProjectArgs& a, bool e4m3) {
    const uint32_t m_tiles = (a.rows + T::BM - 1u) / T::BM, n_tiles = (a.n + T::BN - 1u) / T::BN;
    const dim3 grid(m_tiles * n_tiles * a.splits), block(256);
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
    if (a.splits > 1u) {
        const uint64_t threads = (uint64_t)a.rows * (part_stride(a.n) / 4u);
        hipLaunchKernelGGL(k_project_join, dim3((uint32_t)((threads + 255u) / 256u)), dim3(256), 0, stream, a);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_project_tiles(hipStream_t stream, const ProjectArgs& a, bool e4m3, uint32_t tile) {
    return tile == 256u   ? launch_tile<Tile<32, 2, 2, 4, 4, 1, 2>>(stream, a, e4m3)
           : tile == 128u ? launch_tile<Tile<16, 2, 2, 4, 4, 2, 2>>(stream, a, e4m3)
                          : launch_tile<Tile<16, 2, 2, 2, 2, 2, 4>>(stream, a, e4m3);
}

}  // namespace lily
