// logits_rows.hip - penalties for repeated tokens, bias lists and grammar masks applied to whole rows of
// logits, the rows written out as adjusted logits or log-probabilities, with each row's log-sum-exp.
//
//     a = ((l + biases in list order), -inf where barred, penalties where counted) / T,
//     lse = top + log sum exp(a - top),  log-probability = (a - top) - log sum exp(a - top)
//
// The values are those the draws form for their candidates, operation for operation (f32, IEEE
// division), so a draw from the written f32 row without penalties, masks and biases is the draw from the
// raw one with them.
//
// A thread takes four neighbouring ids at a time: a nibble of the bitmap of listed ids, of the mask and of
// the biased ids (a bitmap of the slice in LDS, built from the row's list) each.  Listed and biased ids that
// the mask leaves are evaluated a lane each, a few steps' together.
//
// Log-probabilities need the row's sum before the first value can be written.  A row is cut into slices whose
// values stay in registers: each workgroup leaves its (largest value, sum) as one word, which is the whole message,
// looks for the words of its row's other slices, a bounded number of times, and writes.  Where a word does not
// come (the other workgroup has no place on the chip yet) it forms the other slices' words itself, by the same
// operations, so the result is the same.  Rows too long for that (over 524 288 ids), and rows in slices where the relaxed
// form of the hand-over (last_to_arrive()) is taken out, take a launch for the sums and one that writes: a ticket that releases
// and acquires writes back the outputs behind every one (1 024 rows of 151 936 1 099 us, so 305).
//
// Bound by memory where rows are many: 1 024 rows of 151 936 bf16 to f32 are written, adjusted, in 166 us (933 MB, 5.6
// TB/s, what a copy reaches) and as log-probabilities in 180; under histories of 2 048 ids in 200 and 215, where the
// counts of the listed ids, a line each, are 180 MB more.  Operations come next (37 vector instructions an id with such a
// history; 53, with a division of five operations and a look at the listed ids group by group, took 245 us).  64
// rows take 21 us, 13 of them for what crosses the memory: a batch that is one round of workgroups reads, waits for its
// neighbours' words and writes, one after the other.  4 rows take 11, where each step is a latency.
#include <hip/hip_runtime.h>

#include "device_common.h"
#include "launch.h"

namespace lily {

namespace {

constexpr int GROUP = 4;           // ids a thread takes at a time
constexpr int AHEAD = 4;           // groups of a thread in flight, in a slice of any length
constexpr int HELD = 8;            // groups a thread holds: slices of at most HELD * GROUP * 256 ids
constexpr uint32_t BIAS_PAIRS = 512;   // pairs of a slice kept in LDS
// Workgroups of 256 threads that a batch is cut into: as many as the chip holds.  Slices that are held have more
// registers a thread, and nobody should wait for a workgroup without a place (64 rows of 151 936 bf16, log-probabilities:
// 2 048 workgroups 31 us, 1 216 19).
constexpr uint32_t LOGITS_GROUPS = 2048, LOGITS_GROUPS_HELD = 1024;
constexpr uint32_t LOGITS_SLICE_MIN = 2048;   // ids
constexpr uint32_t LOGITS_HELD = HELD * GROUP * 256;   // ids of a slice that is held
constexpr float LOG2E = 1.4426950408889634f;

enum Form {
    FORM_ADJUSTED = 0,    // written, no sums
    FORM_HELD_ADJUSTED,   // written, and summed, by slices that are held
    FORM_HELD_LOGPROBS,   // log-probabilities by slices that are held
    FORM_SUM,             // summed only: the first launch of two
    FORM_AFTER_ADJUSTED,  // written with the sums of the launch before
    FORM_AFTER_LOGPROBS,
};
constexpr bool is_held(int form) { return form == FORM_HELD_ADJUSTED || form == FORM_HELD_LOGPROBS; }
constexpr bool is_logprobs(int form) { return form == FORM_HELD_LOGPROBS || form == FORM_AFTER_LOGPROBS; }

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x4 u32x4_any __attribute__((aligned(4)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_out __attribute__((ext_vector_type(4), aligned(4)));
typedef u32x2 u32x2_out __attribute__((aligned(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

template <int DT>
struct RawGroup;
template <>
struct RawGroup<LILY_F32> {
    u32x4 w;
    __device__ __forceinline__ void load(const void* from, uint32_t group) {
        w = *(const LILY_GLOBAL u32x4_any*)(static_cast<const char*>(from) + group * 16u);
    }
    __device__ __forceinline__ float at(int j) const { return lilym_bits_f32(w[j]); }
};
template <>
struct RawGroup<LILY_BF16> {
    u32x2 w;
    __device__ __forceinline__ void load(const void* from, uint32_t group) {
        w = *(const LILY_GLOBAL u32x2_any*)(static_cast<const char*>(from) + group * 8u);
    }
    __device__ __forceinline__ float at(int j) const {
        return lilym_bits_f32((j & 1) ? (w[j >> 1] & 0xffff0000u) : (w[j >> 1] << 16));
    }
};

template <int DT>
__device__ __forceinline__ void store_group(void* to, uint32_t group, f32x4 v) {
    if (DT == LILY_F32) {
        *(LILY_GLOBAL f32x4_out*)(static_cast<char*>(to) + group * 16u) = f32x4_out{v[0], v[1], v[2], v[3]};
    } else {
        *(LILY_GLOBAL u32x2_out*)(static_cast<char*>(to) + group * 8u) = u32x2_out{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3])};
    }
}
template <int DT>
__device__ __forceinline__ void store_one(void* row, uint32_t id, float v) {
    if (DT == LILY_F32) {
        *(LILY_GLOBAL float*)(static_cast<float*>(row) + id) = v;
    } else {
        *(LILY_GLOBAL uint16_t*)(static_cast<uint16_t*>(row) + id) = (uint16_t)bf16_pair(v, 0.0f);
    }
}

// What a workgroup knows of the biases of its slice.
struct SliceBias {
    uint32_t n;        // pairs listed, in list order; more than BIAS_PAIRS: the row's own list is read
    uint32_t ids[BIAS_PAIRS];
    float deltas[BIAS_PAIRS];
};
// (the maximum that hands a NaN on needs no quieted operands: an instruction for three values)
__device__ __forceinline__ float largest(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float largest(f32x4 v) { return largest(largest(v[0], v[1]), largest(v[2], v[3])); }

// A thread's sum of exp(v - m), m the largest value it has seen.  (The reference is a value, not its
// multiple by log2 e: rows whose every value is the type's lowest would overflow there.)
struct RowSum {
    float m, s;
    __device__ __forceinline__ void init() {
        m = NEG_INF;
        s = 0.0f;
    }
    __device__ __forceinline__ float raise(float top) {
        const float before = m;
        m = largest(m, top);
        const float ref = largest(m, F32_LOWEST);   // (nothing but -inf so far: its terms are 0)
        s *= __builtin_amdgcn_exp2f((before - ref) * LOG2E);
        return ref;
    }
    __device__ __forceinline__ void add(float v, float ref) { s += __builtin_amdgcn_exp2f((v - ref) * LOG2E); }
    __device__ __forceinline__ void add1(float v) { add(v, raise(v)); }
    __device__ __forceinline__ void add4(f32x4 v) {
        const float ref = raise(largest(v));
#pragma unroll
        for (int j = 0; j < GROUP; ++j) {
            add(v[j], ref);
        }
    }
    // All the values a thread holds, in the place of what was summed before.  The exponents are formed in one operation
    // each, v log2 e - c, c = ref log2 e rounded once: what that rounding took, 2^e, is the same factor for all the terms,
    // and is given back to their sum.  Only for a ref below 2^24, where |e| <= 1 (half a step of c, which lies below 2^25):
    // half a step of 1e10 log2 e is 512, and neither 2^e nor its inverse is a number then.  Elsewhere the
    // difference comes first, as in add().
    __device__ __forceinline__ void hold(const f32x4 (&v)[HELD], float odd) {
        m = odd;
#pragma unroll
        for (int u = 0; u < HELD; ++u) {
            m = largest(m, largest(v[u]));
        }
        const float ref = largest(m, F32_LOWEST);
        float part[GROUP] = {};
        if (fabsf(ref) < 0x1p24f) {
            const float c = ref * LOG2E;
#pragma unroll
            for (int u = 0; u < HELD; ++u) {
#pragma unroll
                for (int j = 0; j < GROUP; ++j) {
                    part[j] += __builtin_amdgcn_exp2f(__builtin_fmaf(v[u][j], LOG2E, -c));
                }
            }
            part[0] += __builtin_amdgcn_exp2f(__builtin_fmaf(odd, LOG2E, -c));
            s = ((part[0] + part[1]) + (part[2] + part[3])) * __builtin_amdgcn_exp2f(-__builtin_fmaf(ref, LOG2E, -c));
        } else {
#pragma unroll
            for (int u = 0; u < HELD; ++u) {
#pragma unroll
                for (int j = 0; j < GROUP; ++j) {
                    part[j] += __builtin_amdgcn_exp2f((v[u][j] - ref) * LOG2E);
                }
            }
            s = ((part[0] + part[1]) + (part[2] + part[3])) + __builtin_amdgcn_exp2f((odd - ref) * LOG2E);
        }
    }
};
struct Sums {
    double s[4];
    float m[4];
    uint64_t words[MAX_SLICES];   // of the row's slices
    uint32_t missing;
};

// The slice's pairs in list order, and a bit for each biased id (bits: (hi - lo + 31) / 32 words).
__device__ __forceinline__ void list_biases(const RowArgs& a, uint32_t lo, uint32_t hi, SliceBias& sb, uint32_t* bits,
                                            uint32_t* wave_count) {
    const uint32_t tid = threadIdx.x, nt = blockDim.x, lane = tid & 63u, wave = tid >> 6;
    for (uint32_t w = tid; w < (hi - lo + 31u) / 32u; w += nt) {
        bits[w] = 0u;
    }
    uint32_t have = 0;
    __syncthreads();
    for (uint32_t j0 = 0; j0 < a.n_bias; j0 += nt) {
        const uint32_t j = j0 + tid;
        uint32_t id = 0xffffffffu;
        float delta = 0.0f;
        if (j < a.n_bias) {
            id = gload(&a.bias[j].id);
            delta = gload(&a.bias[j].delta);
        }
        const bool in = j < a.n_bias && id >= lo && id < hi;
        const uint64_t ballot = __ballot(in);
        if (lane == 0u) {
            wave_count[wave] = (uint32_t)__popcll(ballot);
        }
        __syncthreads();
        uint32_t at = have + (uint32_t)__popcll(ballot & ((1ull << lane) - 1ull));
        for (uint32_t q = 0; q < nt / 64u; ++q) {
            at += q < wave ? wave_count[q] : 0u;
            have += wave_count[q];
        }
        if (in) {
            atomicOr(&bits[(id - lo) >> 5], 1u << ((id - lo) & 31u));
            if (at < BIAS_PAIRS) {
                sb.ids[at] = id;
                sb.deltas[at] = delta;
            }
        }
        __syncthreads();
    }
    if (tid == 0u) {
        sb.n = have;
    }
    __syncthreads();
}

// The division by the temperature, rounded as IEEE has it, and -inf for a NaN.  With the reciprocal in two parts, r the
// nearest number and low what is left of it, q = l r + l low is within a unit in the last place of l / T, its remainder l - q T is
// exact, and q + (l - q T) r is the quotient correctly rounded (Markstein 1990) - four operations for the fourteen of a
// division, as long as nothing on the way is subnormal or overflows upwards: a group with a zero, a tiny or a huge value goes the long
// way.  Values far below zero may overflow: what should be -inf comes out as a NaN, and is worth -inf.  (The remainder
// is formed with the other sign: so zeros would keep theirs.)
struct Temperature {
    float t, r, low;
    bool one, plain;
};
__device__ __forceinline__ Temperature temperature_of(const RowArgs& a) {
    Temperature t;
    t.t = a.temperature;
    t.r = 1.0f / a.temperature;
    t.low = __builtin_fmaf(-t.r, t.t, 1.0f) * t.r;
    t.one = a.temperature == 1.0f;
    t.plain = a.temperature > 0x1p-20f && a.temperature < 0x1p20f;
    return t;
}
__device__ __forceinline__ void divide(f32x4& v, const Temperature& t) {
    if (t.one) {
#pragma unroll
        for (int j = 0; j < GROUP; ++j) {
            v[j] = fmaxf(v[j], NEG_INF);
        }
        return;
    }
    float least = fabsf(v[0]);
#pragma unroll
    for (int j = 1; j < GROUP; ++j) {
        least = __builtin_elementwise_minimum(least, fabsf(v[j]));
    }
    if (t.plain && largest(v) < 0x1p100f && least > 0x1p-100f) {
#pragma unroll
        for (int j = 0; j < GROUP; ++j) {
            const float q = __builtin_fmaf(v[j], t.r, v[j] * t.low), over = __builtin_fmaf(q, t.t, -v[j]);
            v[j] = fmaxf(__builtin_fmaf(-over, t.r, q), NEG_INF);
        }
    } else {
#pragma unroll
        for (int j = 0; j < GROUP; ++j) {
            v[j] = fmaxf(v[j] / t.t, NEG_INF);
        }
    }
}

// One id's value before the temperature, given its logit, count, and whether it is biased and admitted: the
// draws' arithmetic.
__device__ __forceinline__ float adjusted(const RowArgs& a, const SliceBias* sb, uint32_t id, float l, uint32_t count,
                                          bool biased, bool allowed) {
    if (biased) {
        if (sb->n <= BIAS_PAIRS) {
            for (uint32_t j = 0; j < sb->n; ++j) {
                l = sb->ids[j] == id ? l + sb->deltas[j] : l;
            }
        } else {
            for (uint32_t j = 0; j < a.n_bias; ++j) {
                if (gload(&a.bias[j].id) == id) {
                    l += gload(&a.bias[j].delta);
                }
            }
        }
    }
    if (count > 0u) {
        l = l > 0.0f ? l / a.repetition : l * a.repetition;
        l -= a.presence + a.frequency * (float)count;
    }
    return allowed ? l : NEG_INF;
}

// Ids of a wave's steps whose value takes more than its logit, its mask bit and the temperature are gathered
// here and evaluated a lane each (one lane's look at its counts would hold up the other 63), and their values
// go back to the groups they belong to, which are then stored whole: lines written in part, now and a while later,
// cost more than everything else (1 024 rows of 151 936 bf16 under 2 048-id histories to f32: +110 us of 192).
constexpr uint32_t QUEUE = 512;   // ids of a wave: two groups of every lane at least

// What a workgroup's look at its slice, ids [lo, hi) (lo a multiple of 32), goes by.
struct Slice {
    const RowArgs& a;
    const SliceBias* sb;
    const uint32_t* bits;   // of the biased ids
    uint32_t* queue;        // the wave's
    Temperature temperature;
    uint32_t lo, hi, whole; // whole: groups; the ids behind the last one are evaluated by themselves
    bool pen, masked, biased;
    __device__ __forceinline__ Slice(const RowArgs& args, const SliceBias* b, const uint32_t* w, uint32_t* q, uint32_t from, uint32_t to)
        : a(args), sb(b), bits(w), queue(q), temperature(temperature_of(args)), lo(from), hi(to), whole((to - from) / GROUP),
          pen((args.flags & F_PEN) != 0u), masked(args.allow != nullptr), biased(args.n_bias != 0u) {}
};
template <int DT>
__device__ __forceinline__ float value_of(const Slice& s, uint32_t id, bool allowed) {
    const float l = load_logit<DT>(s.a.logits, id);
    const uint32_t count = s.pen ? gload(s.a.counts + id) : 0u;
    const bool add = s.biased && ((s.bits[(id - s.lo) >> 5] >> ((id - s.lo) & 31u)) & 1u) != 0u;
    return fmaxf(adjusted(s.a, s.sb, id, l, count, add, allowed) / s.a.temperature, NEG_INF);
}
// The id behind the last whole group that is this thread's, if any.
__device__ __forceinline__ bool odd_id(const Slice& s, uint32_t& id) {
    id = s.lo + s.whole * GROUP + threadIdx.x;
    return id < s.hi;
}
template <int DT>
__device__ __forceinline__ float odd_value(const Slice& s, uint32_t id) {
    return value_of<DT>(s, id, !s.masked || bit_of(s.a.allow, id));
}

// The values of N groups of every lane, groups w0 + lane, w0 + lane + 256, ... (w0 the same in the wave); groups
// from `whole` on hold nothing of use.
template <int DT, int N>
__device__ __forceinline__ void groups(const Slice& s, uint32_t w0, f32x4 (&v)[N]) {
    static_assert(N * GROUP <= 32 && QUEUE >= 2 * GROUP * 64, "a bit an id of a lane");
    const uint32_t lane = threadIdx.x & 63u, g0 = w0 + lane;
    const char* from = static_cast<const char*>(s.a.logits) + (size_t)s.lo * (DT == LILY_F32 ? 4u : 2u);
    RawGroup<DT> raw[N];
    uint32_t listed[N], admitted[N];
    auto at = [&](int u) { return min(g0 + (uint32_t)u * 256u, s.whole - 1u); };
#pragma unroll
    for (int u = 0; u < N; ++u) {
        raw[u].load(from, at(u));
    }
    if (s.pen) {
        const uint32_t* words = s.a.touched + s.lo / 32u;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            listed[u] = gload(words + at(u) / 8u);
        }
    }
    if (s.masked) {
        const uint32_t* words = s.a.allow + s.lo / 32u;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            admitted[u] = gload(words + at(u) / 8u);
        }
    }
    const uint32_t shift = g0 % 8u * GROUP;   // of the groups' bits in their words, the same for all of them
    uint32_t some = 0, open = 0xffffffffu;    // bits of the lane's ids: listed or biased, admitted
    if (s.pen) {
#pragma unroll
        for (int u = 0; u < N; ++u) {
            some |= (listed[u] >> shift & 15u) << (u * GROUP);
        }
    }
    if (s.biased) {
#pragma unroll
        for (int u = 0; u < N; ++u) {
            some |= (s.bits[at(u) / 8u] >> shift & 15u) << (u * GROUP);
        }
    }
    if (s.masked) {
        open = 0u;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            open |= (admitted[u] >> shift & 15u) << (u * GROUP);
        }
    }
#pragma unroll
    for (int u = 0; u < N; ++u) {
#pragma unroll
        for (int j = 0; j < GROUP; ++j) {
            v[u][j] = raw[u].at(j);
        }
        divide(v[u], s.temperature);
        if (s.masked) {
#pragma unroll
            for (int j = 0; j < GROUP; ++j) {
                const uint32_t all = (uint32_t)((int32_t)(open << (31 - u * GROUP - j)) >> 31);
                v[u][j] = lilym_bits_f32((lilym_f32_bits(v[u][j]) & all) | (lilym_f32_bits(NEG_INF) & ~all));
            }
        }
    }
    const uint32_t mine = g0 < s.whole ? (s.whole - g0 + 255u) / 256u : 0u;   // groups that are there
    some &= open & (mine >= (uint32_t)N ? 0xffffffffu : (1u << (mine * GROUP)) - 1u);
    if (__ballot(some != 0u) == 0ull) {
        return;
    }
    // All of the ids at once, or two groups' after the other where they are too many for the queue.
    const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan_u32((uint32_t)__builtin_popcount(some)), 63);
    const uint32_t width = all <= QUEUE ? 32u : 2u * GROUP;
    for (uint32_t b = 0; b < (uint32_t)(N * GROUP); b += width) {
        const uint32_t part = some & (width == 32u ? 0xffffffffu : ((1u << width) - 1u) << b);
        const uint32_t n = (uint32_t)__builtin_popcount(part), upto = wave_scan_u32(n);
        const uint32_t waiting = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
        uint32_t k = upto - n;
        for (uint32_t rest = part; rest != 0u; rest &= rest - 1u) {
            const uint32_t c = (uint32_t)__builtin_ctz(rest);
            s.queue[k++] = s.lo + (g0 + c / GROUP * 256u) * GROUP + c % GROUP;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        for (uint32_t i = lane; i < waiting; i += 64u) {
            s.queue[i] = lilym_f32_bits(value_of<DT>(s, s.queue[i], true));
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        k = upto - n;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const uint32_t bits = part >> (u * GROUP) & 15u;
            if (__ballot(bits != 0u) != 0ull) {
#pragma unroll
                for (int j = 0; j < GROUP; ++j) {
                    const float x = lilym_bits_f32(s.queue[k]);   // (one behind the last may be looked at, and is not taken)
                    const bool taken = (bits >> j & 1u) != 0u;
                    v[u][j] = taken ? x : v[u][j];
                    k += taken ? 1u : 0u;
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// One pass over the slice: each(group, its values), each_one(id, value).
template <int DT, class EACH, class EACH_ONE>
__device__ __forceinline__ void pass_over(const Slice& s, EACH&& each, EACH_ONE&& each_one) {
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    for (uint32_t w0 = tid - lane; w0 < s.whole; w0 += 256u * AHEAD) {
        f32x4 v[AHEAD];
        groups<DT>(s, w0, v);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const uint32_t g = w0 + lane + (uint32_t)u * 256u;
            if (g < s.whole) {
                each(g, v[u]);
            }
        }
    }
    uint32_t id;
    if (odd_id(s, id)) {
        each_one(id, odd_value<DT>(s, id));
    }
}

// The slice's values in registers, and the thread's sum of them.
template <int DT>
__device__ __forceinline__ RowSum hold(const Slice& s, f32x4 (&v)[HELD], float& odd_v) {
    const uint32_t tid = threadIdx.x;
    if (s.whole != 0u) {
        groups<DT>(s, tid & ~63u, v);
    }
#pragma unroll
    for (int u = 0; u < HELD; ++u) {
        if (s.whole < (uint32_t)(u + 1) * 256u && tid + (uint32_t)u * 256u >= s.whole) {
#pragma unroll
            for (int j = 0; j < GROUP; ++j) {
                v[u][j] = NEG_INF;
            }
        }
    }
    uint32_t odd;
    odd_v = odd_id(s, odd) ? odd_value<DT>(s, odd) : NEG_INF;
    RowSum sum;
    sum.hold(v, odd_v);
    return sum;
}

struct LogitsLaunch {
    void* out;
    uint64_t stride;        // elements
    float* lse;             // or null
    Handed<uint64_t> word;  // [rows][MAX_SLICES] of the slices: largest value << 32 | sum (f32 each); 0 = not there, and
                            // left so between launches
    uint32_t* done;         // [rows] workgroups that have left their word and seen the others', 0 between launches
    uint32_t vocab, slices, per_slice;   // per_slice: a multiple of 32
    uint32_t looks;         // for the words of a row's other slices
    uint32_t in_place;      // the outputs take the logits' place
    uint32_t bias_bits;     // words of dynamic LDS for the biased ids' bitmap (0: no row has a bias list)
};

// A row's log-sum-exp as its largest value and the logarithm of its sum relative to that: a log-probability is
// (a - top) - log_s, exact where the row's values lie together however large they are (rows masked by the
// type's lowest value throughout are even, not nothing).
struct LogSum {
    float top, log_s;   // (an empty row has 0 for both: its values stay -inf)
    float whole;        // the log-sum-exp
    __device__ __forceinline__ float logprob(float a) const { return (a - top) - log_s; }
};
__device__ __forceinline__ LogSum log_sum(double m, double s) {
    LogSum r;
    // (a row with a value sums to 1 at least; one that holds +inf has no sum that means anything, and needs none)
    const bool finite = m > (double)NEG_INF && m < (double)__builtin_huge_valf();
    r.top = m > (double)NEG_INF ? (float)m : 0.0f;
    r.log_s = finite ? (float)log(s) : 0.0f;
    r.whole = (float)(m + (double)r.log_s);
    return r;
}

// The workgroup's (largest value, sum) as a word, in every thread.  (f32 is enough for the sum of a slice: one
// rounding more.  Never 0: a slice with a finite value sums to 1 at least, and one without has -inf for its largest.)
__device__ __forceinline__ uint64_t merge_threads(const RowSum& l, Sums& sh) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    float m = wave_max_dpp(l.m);
    double s = l.m > NEG_INF ? (double)l.s * (double)__builtin_amdgcn_exp2f((l.m - m) * LOG2E) : 0.0;
    s = wave_sum_d(s);
    if (lane == 0u) {
        sh.m[wave] = m;
        sh.s[wave] = s;
    }
    __syncthreads();
    m = fmaxf(fmaxf(sh.m[0], sh.m[1]), fmaxf(sh.m[2], sh.m[3]));
    s = 0.0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        s += sh.m[q] > NEG_INF ? sh.s[q] * (double)__builtin_amdgcn_exp2f((sh.m[q] - m) * LOG2E) : 0.0;
    }
    __syncthreads();
    return (uint64_t)lilym_f32_bits(m) << 32 | lilym_f32_bits((float)s);
}
// The slices' words (a lane a slice, 0 beyond the last) as one (largest value, sum), in every lane of the wave.
__device__ __forceinline__ void merge_slices(uint64_t word, uint32_t slices, double& m_out, double& s_out) {
    const bool mine = (threadIdx.x & 63u) < slices;
    const float m = mine ? lilym_bits_f32((uint32_t)(word >> 32)) : NEG_INF, top = wave_max_dpp(m);
    m_out = (double)top;
    s_out = wave_sum_d(mine && m > NEG_INF ? (double)lilym_bits_f32((uint32_t)word) * (double)__builtin_amdgcn_exp2f((m - top) * LOG2E) : 0.0);
}

template <int DT, int OT, int FORM>
__device__ __forceinline__ void logits_row(const RowArgs& a, uint32_t row_of_launch, uint32_t slice, const LogitsLaunch& q) {
    __shared__ SliceBias sb;
    __shared__ Sums sh;
    __shared__ uint32_t wave_count[4];
    __shared__ uint32_t queues[4][QUEUE + 1];
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    uint32_t* queue = queues[tid >> 6];
    uint32_t* bits = reinterpret_cast<uint32_t*>(dyn_lds);
    const uint32_t row = (uint32_t)a.row;   // of the output
    void* out = static_cast<char*>(q.out) + (size_t)row * q.stride * (OT == LILY_F32 ? 4u : 2u);
    const size_t first = (size_t)row_of_launch * MAX_SLICES;
    auto take = [&](uint32_t which) {   // slice `which`, its biases listed
        const uint32_t lo = which * q.per_slice, hi = min(q.vocab, lo + q.per_slice);
        if (a.n_bias != 0u) {
            list_biases(a, lo, hi, sb, bits, wave_count);
        }
        return Slice(a, &sb, bits, queue, lo, hi);
    };
    const Slice mine = take(slice);
    LogSum lse = {0.0f, 0.0f, 0.0f};
    auto worth = [&](float v) { return is_logprobs(FORM) ? lse.logprob(v) : v; };
    auto write_one = [&](uint32_t id, float v) { store_one<OT>(out, id, worth(v)); };
    char* out_slice = static_cast<char*>(out) + (size_t)mine.lo * (OT == LILY_F32 ? 4u : 2u);
    auto write = [&](uint32_t group, f32x4 v) {
        const f32x4 p = {worth(v[0]), worth(v[1]), worth(v[2]), worth(v[3])};
        store_group<OT>(out_slice, group, p);
    };
    if constexpr (FORM == FORM_ADJUSTED) {
        pass_over<DT>(mine, write, write_one);
    } else if constexpr (FORM == FORM_SUM) {
        RowSum sum;
        sum.init();
        pass_over<DT>(
            mine, [&](uint32_t, f32x4 v) { sum.add4(v); }, [&](uint32_t, float v) { sum.add1(v); });
        const uint64_t word = merge_threads(sum, sh);
        if (tid == 0u) {
            handed_store(q.word, first + slice, word);
        }
    } else if constexpr (!is_held(FORM)) {
        double m, s;
        merge_slices(lane < q.slices ? handed_load(q.word, first + lane) : 0ull, q.slices, m, s);
        lse = log_sum(m, s);
        if (q.lse != nullptr && slice == 0u && tid == 0u) {
            q.lse[row] = lse.whole;
        }
        pass_over<DT>(mine, write, write_one);
    } else {
        // The slice's values in registers, and its word.
        f32x4 v[HELD];
        float odd_v;
        const RowSum sum = hold<DT>(mine, v, odd_v);
        const uint64_t word = merge_threads(sum, sh);
        if (q.slices > 1u && tid == 0u) {
            handed_store(q.word, first + slice, word);
        }
        auto store_all = [&] {
#pragma unroll
            for (int u = 0; u < HELD; ++u) {
                const uint32_t g = tid + (uint32_t)u * 256u;
                if (g < mine.whole) {
                    write(g, v[u]);
                }
            }
            uint32_t odd;
            if (odd_id(mine, odd)) {
                write_one(odd, odd_v);
            }
        };
        // Where the outputs take the logits' place, none is written before the slice's word has arrived: who forms the
        // word itself from the logits, and still finds none behind them, has read logits.  (That the word is in memory
        // when its store counts as done is the hardware's promise, as in last_to_arrive()'s relaxed form, not the memory
        // model's; the same for the count behind which the words are cleared.)
        if (q.slices > 1u && (is_logprobs(FORM) || q.in_place != 0u)) {
            if (tid < 64u) {
                __builtin_amdgcn_s_waitcnt(0);
            }
            __syncthreads();
        }
        if (!is_logprobs(FORM)) {
            store_all();
        }
        // Only who needs the row's sum looks for it: every slice of log-probabilities, else the first.
        if (is_logprobs(FORM) || (slice == 0u && q.lse != nullptr)) {
            if (tid < 64u) {
                uint64_t seen = lane == slice ? word : 0ull;
                bool all = q.slices == 1u;
                for (uint32_t n = 0; n < q.looks && !all; ++n) {
                    if (lane < q.slices && seen == 0ull) {
                        seen = handed_load(q.word, first + lane);
                    }
                    all = __ballot(lane < q.slices && seen == 0ull) == 0ull;
                }
                sh.words[lane] = seen;
                if (lane == 0u) {
                    sh.missing = all ? 0u : 1u;
                }
            }
            __syncthreads();
            if (sh.missing != 0u) {
                // Somebody has no place on the chip yet: the words that are missing from here, the same ones (the
                // threads add the same values in the same order), and then this slice again.
                for (uint32_t other = 0; other < q.slices; ++other) {
                    if (sh.words[other] != 0ull) {
                        continue;
                    }
                    const uint64_t formed = merge_threads(hold<DT>(take(other), v, odd_v), sh);
                    if (tid == 0u) {
                        const uint64_t come = handed_load(q.word, first + other);
                        sh.words[other] = come != 0ull ? come : formed;
                    }
                    __syncthreads();
                }
                if (is_logprobs(FORM)) {
                    hold<DT>(take(slice), v, odd_v);
                }
            }
            double m, s;
            merge_slices(sh.words[lane], q.slices, m, s);
            lse = log_sum(m, s);
            if (q.lse != nullptr && slice == 0u && tid == 0u) {
                q.lse[row] = lse.whole;
            }
        }
        if (is_logprobs(FORM)) {
            store_all();
        }
        // The last workgroup of the row to have left its word and seen what it wanted clears the words.
        if (q.slices > 1u && tid < 64u) {
            uint32_t left = 0;
            if (lane == 0u) {
                __builtin_amdgcn_s_waitcnt(0);   // (the word has arrived)
                left = __hip_atomic_fetch_add(q.done + row_of_launch, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            if ((uint32_t)__builtin_amdgcn_readfirstlane((int)left) == q.slices - 1u) {
                if (lane < q.slices) {
                    handed_store(q.word, first + lane, (uint64_t)0);
                }
                if (lane == 0u) {
                    store_through(q.done + row_of_launch, 0u);
                }
            }
        }
    }
}

__device__ __forceinline__ RowArgs row_of(const LILY_CONST RowArgs* p) {
    RowArgs a;
    __builtin_memcpy(&a, (const RowArgs*)p, sizeof a);
    return a;
}

template <int DT, int OT, int FORM>
__global__ void __launch_bounds__(256) k_logits_rows_table(const RowArgs* table, LogitsLaunch q) {
    const uint32_t row = blockIdx.x / q.slices, slice = blockIdx.x % q.slices;
    const RowArgs a = row_of((const LILY_CONST RowArgs*)table + row);
    logits_row<DT, OT, FORM>(a, row, slice, q);
}
template <int DT, int OT, int FORM>
__global__ void __launch_bounds__(256) k_logits_rows_inline(InlineRows rows, LogitsLaunch q) {
    const LILY_CONST RowArgs* table = (const LILY_CONST RowArgs*)__builtin_amdgcn_kernarg_segment_ptr();
    const uint32_t row = blockIdx.x / q.slices, slice = blockIdx.x % q.slices;
    const RowArgs a = row_of(table + row);
    logits_row<DT, OT, FORM>(a, row, slice, q);
}

template <int DT, int OT, int FORM>
hipError_t launch_form(hipStream_t stream, const RowArgs* table, const InlineRows* few, uint32_t rows, const LogitsLaunch& q) {
    const dim3 grid(rows * q.slices), block(256);
    const size_t lds = (size_t)q.bias_bits * 4u;
    if (few != nullptr) {
        hipLaunchKernelGGL((k_logits_rows_inline<DT, OT, FORM>), grid, block, lds, stream, *few, q);
    } else {
        hipLaunchKernelGGL((k_logits_rows_table<DT, OT, FORM>), grid, block, lds, stream, table, q);
    }
    return hipGetLastError();
}

template <int DT, int OT>
hipError_t launch_typed(hipStream_t stream, const RowArgs* table, const InlineRows* few, uint32_t rows, const LogitsLaunch& q,
                        bool logprobs, bool relaxed) {
    if (!logprobs && q.lse == nullptr) {
        return launch_form<DT, OT, FORM_ADJUSTED>(stream, table, few, rows, q);
    }
    if (q.per_slice <= LOGITS_HELD && (relaxed || q.slices == 1u)) {
        return logprobs ? launch_form<DT, OT, FORM_HELD_LOGPROBS>(stream, table, few, rows, q)
                        : launch_form<DT, OT, FORM_HELD_ADJUSTED>(stream, table, few, rows, q);
    }
    const hipError_t e = launch_form<DT, OT, FORM_SUM>(stream, table, few, rows, q);
    if (e != hipSuccess) {
        return e;
    }
    // (the words stay behind: they are cleared before a held launch looks at them)
    const hipError_t f = logprobs ? launch_form<DT, OT, FORM_AFTER_LOGPROBS>(stream, table, few, rows, q)
                                  : launch_form<DT, OT, FORM_AFTER_ADJUSTED>(stream, table, few, rows, q);
    return f != hipSuccess ? f : launch_fill_u32(stream, reinterpret_cast<uint32_t*>(q.word.p), rows * MAX_SLICES * 2u, 0u);
}

}  // namespace

hipError_t launch_logits_rows(hipStream_t stream, int dtype, uint32_t rows, uint32_t vocab, const RowArgs* table,
                              const InlineRows* few, const LogitsRows& w) {
    LogitsLaunch q = {};
    q.out = w.out;
    q.stride = w.stride;
    q.lse = w.lse;
    q.word = w.word;
    q.done = w.done;
    q.looks = w.looks;
    q.in_place = w.in_place;
#ifdef LILY_STRICT_HANDOVER
    const bool relaxed = false;
#else
    const bool relaxed = w.relaxed;
#endif
    q.vocab = vocab;
    // A launch takes as many rows as the workspace has words for.
    for (uint32_t first = 0; first < rows; first += w.max_rows) {
        const uint32_t n = min(rows - first, w.max_rows);
        const uint32_t groups = !w.logprobs && w.lse == nullptr ? LOGITS_GROUPS : LOGITS_GROUPS_HELD;
        uint32_t slices = min((groups + n - 1u) / n, (vocab + LOGITS_SLICE_MIN - 1u) / LOGITS_SLICE_MIN);
        slices = max(slices, (vocab + LOGITS_HELD - 1u) / LOGITS_HELD);
        slices = max(1u, min(slices, MAX_SLICES));
        q.per_slice = ((vocab + slices - 1u) / slices + 31u) / 32u * 32u;
        q.slices = (vocab + q.per_slice - 1u) / q.per_slice;
        q.bias_bits = w.biased ? q.per_slice / 32u : 0u;
        const RowArgs* part = table != nullptr ? table + first : nullptr;
        hipError_t e;
        if (dtype == LILY_BF16) {
            e = w.out_dtype == LILY_BF16 ? launch_typed<LILY_BF16, LILY_BF16>(stream, part, few, n, q, w.logprobs, relaxed)
                                         : launch_typed<LILY_BF16, LILY_F32>(stream, part, few, n, q, w.logprobs, relaxed);
        } else {
            e = w.out_dtype == LILY_BF16 ? launch_typed<LILY_F32, LILY_BF16>(stream, part, few, n, q, w.logprobs, relaxed)
                                         : launch_typed<LILY_F32, LILY_F32>(stream, part, few, n, q, w.logprobs, relaxed);
        }
        if (e != hipSuccess) {
            return e;
        }
    }
    return hipSuccess;
}

}  // namespace lily
