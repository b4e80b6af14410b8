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
// operations, so the result is the same.  One pass over the logits: 1 024 rows of 151 936 went twice through a row
// in 245 us before, and two launches of 64 rows took 25.  Rows too long for that (over 524 288 ids) take a launch
// for the sums and one that writes.
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
    __device__ __forceinline__ void load(const void* row, uint32_t id) {
        w = *(const LILY_GLOBAL u32x4_any*)(static_cast<const float*>(row) + id);
    }
    __device__ __forceinline__ float at(int j) const { return lilym_bits_f32(w[j]); }
};
template <>
struct RawGroup<LILY_BF16> {
    u32x2 w;
    __device__ __forceinline__ void load(const void* row, uint32_t id) {
        w = *(const LILY_GLOBAL u32x2_any*)(static_cast<const uint16_t*>(row) + id);
    }
    __device__ __forceinline__ float at(int j) const {
        return lilym_bits_f32((j & 1) ? (w[j >> 1] & 0xffff0000u) : (w[j >> 1] << 16));
    }
};

template <int DT>
__device__ __forceinline__ void store_group(void* row, uint32_t id, const float (&v)[GROUP]) {
    if (DT == LILY_F32) {
        *(LILY_GLOBAL f32x4_out*)(static_cast<float*>(row) + id) = f32x4_out{v[0], v[1], v[2], v[3]};
    } else {
        *(LILY_GLOBAL u32x2_out*)(static_cast<uint16_t*>(row) + id) = u32x2_out{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3])};
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
    uint32_t total;    // scratch of the listing
    uint32_t ids[BIAS_PAIRS];
    float deltas[BIAS_PAIRS];
};
// A thread's running sum of exp(v - m), m the largest value it has seen.  (The reference is a value, not its
// multiple by log2 e: rows whose every value is the type's lowest would overflow there.)
struct RowSum {
    float m, s;
    __device__ __forceinline__ void init() {
        m = NEG_INF;
        s = 0.0f;
    }
    __device__ __forceinline__ float raise(float top) {
        const float before = m;
        m = fmaxf(m, top);
        const float ref = fmaxf(m, F32_LOWEST);   // (nothing but -inf so far: its terms are 0)
        s *= __builtin_amdgcn_exp2f((before - ref) * LOG2E);
        return ref;
    }
    __device__ __forceinline__ void add(float v, float ref) { s += __builtin_amdgcn_exp2f((v - ref) * LOG2E); }
    __device__ __forceinline__ void add1(float v) { add(v, raise(v)); }
    __device__ __forceinline__ void add4(const float (&v)[GROUP]) {
        const float ref = raise(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])));
#pragma unroll
        for (int j = 0; j < GROUP; ++j) {
            add(v[j], ref);
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

// The division by the temperature, rounded as IEEE has it.  By its correctly rounded reciprocal r: q0 = l r is
// within 1.5 units in the last place of l / T, q1 = q0 + (l - q0 T) r within one, its remainder l - q1 T is then
// exact, and q1 + (l - q1 T) r is the quotient correctly rounded (Markstein 1990) - five operations for the
// fourteen of a division, as long as nothing on the way leaves the normal numbers: zeros, tiny and huge values and
// infinities go the long way, a group at a time.
struct Temperature {
    float t, r;
    bool one, plain;
};
__device__ __forceinline__ Temperature temperature_of(const RowArgs& a) {
    Temperature t;
    t.t = a.temperature;
    t.r = 1.0f / a.temperature;
    t.one = a.temperature == 1.0f;
    t.plain = a.temperature > 0x1p-60f && a.temperature < 0x1p60f;
    return t;
}
__device__ __forceinline__ void divide(float (&v)[GROUP], const Temperature& t) {
    if (t.one) {
        return;
    }
    float most = fabsf(v[0]), least = fabsf(v[0]);
#pragma unroll
    for (int j = 1; j < GROUP; ++j) {
        most = fmaxf(most, fabsf(v[j]));
        least = fminf(least, fabsf(v[j]));
    }
    if (t.plain && most < 0x1p60f && least > 0x1p-40f) {
#pragma unroll
        for (int j = 0; j < GROUP; ++j) {
            float q = v[j] * t.r;
            q = __builtin_fmaf(__builtin_fmaf(-q, t.t, v[j]), t.r, q);
            v[j] = __builtin_fmaf(__builtin_fmaf(-q, t.t, v[j]), t.r, q);
        }
    } else {
#pragma unroll
        for (int j = 0; j < GROUP; ++j) {
            v[j] /= t.t;
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
constexpr uint32_t QUEUE = 512;   // ids of a wave; a step has 256 at most

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

// The values of N groups of every lane, groups w0 + lane, w0 + lane + nt, ... (w0 the same in the wave); groups
// from `whole` on hold nothing of use.
template <int DT, int N>
__device__ __forceinline__ void groups(const Slice& s, uint32_t w0, float (&v)[N][GROUP]) {
    const uint32_t lane = threadIdx.x & 63u, nt = blockDim.x;
    RawGroup<DT> raw[N];
    uint32_t listed[N], admitted[N];
    auto id_at = [&](int u) { return s.lo + min(w0 + lane + (uint32_t)u * nt, s.whole - 1u) * GROUP; };
#pragma unroll
    for (int u = 0; u < N; ++u) {
        raw[u].load(s.a.logits, id_at(u));
    }
    if (s.pen) {
#pragma unroll
        for (int u = 0; u < N; ++u) {
            listed[u] = gload(s.a.touched + (id_at(u) >> 5));
        }
    }
    if (s.masked) {
#pragma unroll
        for (int u = 0; u < N; ++u) {
            admitted[u] = gload(s.a.allow + (id_at(u) >> 5));
        }
    }
    uint32_t some[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const uint32_t id = id_at(u);
        uint32_t word = s.pen ? listed[u] : 0u;
        if (s.biased) {
            word |= s.bits[(id - s.lo) >> 5];
        }
        const uint32_t open = s.masked ? (admitted[u] >> (id & 31u)) & 15u : 15u;
        some[u] = w0 + lane + (uint32_t)u * nt < s.whole ? (word >> (id & 31u)) & open : 0u;
#pragma unroll
        for (int j = 0; j < GROUP; ++j) {
            v[u][j] = raw[u].at(j);
        }
        if (open != 15u) {
#pragma unroll
            for (int j = 0; j < GROUP; ++j) {
                v[u][j] = (open >> j) & 1u ? v[u][j] : NEG_INF;
            }
        }
        divide(v[u], s.temperature);
#pragma unroll
        for (int j = 0; j < GROUP; ++j) {
            v[u][j] = fmaxf(v[u][j], NEG_INF);   // (a NaN is worth -inf)
        }
    }
    if (!s.pen && !s.biased) {
        return;
    }
    // All steps' ids at once, or as many steps' as the queue holds.
    for (;;) {
        uint32_t at[N], waiting = 0, taken = 0;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            if (__ballot(some[u] != 0u) != 0u) {
                const uint32_t n = (uint32_t)__builtin_popcount(some[u]), upto = wave_scan_u32(n);
                const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
                if (waiting + all <= QUEUE) {
                    at[u] = waiting + upto - n;
                    waiting += all;
                    taken |= 1u << u;
                    uint32_t k = at[u];
                    for (uint32_t rest = some[u]; rest != 0u; rest &= rest - 1u) {
                        s.queue[k++] = id_at(u) + (uint32_t)__builtin_ctz(rest);
                    }
                }
            }
        }
        if (taken == 0u) {
            return;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        for (uint32_t k = lane; k < waiting; k += 64u) {
            s.queue[k] = lilym_f32_bits(value_of<DT>(s, s.queue[k], true));
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int u = 0; u < N; ++u) {
            if (((taken >> u) & 1u) != 0u) {
                uint32_t k = at[u];
#pragma unroll
                for (int j = 0; j < GROUP; ++j) {
                    if ((some[u] >> j) & 1u) {
                        v[u][j] = lilym_bits_f32(s.queue[k++]);
                    }
                }
                some[u] = 0u;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// One pass over the slice: each(id, values of a group), each_one(id, value).
template <int DT, class EACH, class EACH_ONE>
__device__ __forceinline__ void pass_over(const Slice& s, EACH&& each, EACH_ONE&& each_one) {
    const uint32_t tid = threadIdx.x, nt = blockDim.x, lane = tid & 63u;
    for (uint32_t w0 = tid - lane; w0 < s.whole; w0 += nt * AHEAD) {
        float v[AHEAD][GROUP];
        groups<DT>(s, w0, v);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const uint32_t g = w0 + lane + (uint32_t)u * nt;
            if (g < s.whole) {
                each(s.lo + g * GROUP, v[u]);
            }
        }
    }
    uint32_t id;
    if (odd_id(s, id)) {
        each_one(id, odd_value<DT>(s, id));
    }
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
    float top, log_s;
    __device__ __forceinline__ float whole() const { return (float)((double)top + (double)log_s); }
    __device__ __forceinline__ float logprob(float a) const { return a > NEG_INF ? (a - top) - log_s : NEG_INF; }
};
__device__ __forceinline__ LogSum log_sum(double m, double s) {
    LogSum r;
    r.top = (float)m;
    r.log_s = s > 0.0 ? (float)log(s) : 0.0f;   // (0: an empty row; NaN: a row that holds +inf)
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
    __shared__ uint32_t queues[4][QUEUE];
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
    LogSum lse = {0.0f, 0.0f};
    auto worth = [&](float v) { return is_logprobs(FORM) ? lse.logprob(v) : v; };
    auto write_one = [&](uint32_t id, float v) { store_one<OT>(out, id, worth(v)); };
    auto write = [&](uint32_t id, const float (&v)[GROUP]) {
        const float p[GROUP] = {worth(v[0]), worth(v[1]), worth(v[2]), worth(v[3])};
        store_group<OT>(out, id, p);
    };
    if constexpr (FORM == FORM_ADJUSTED) {
        pass_over<DT>(mine, write, write_one);
    } else if constexpr (FORM == FORM_SUM) {
        RowSum sum;
        sum.init();
        pass_over<DT>(
            mine, [&](uint32_t, const float (&v)[GROUP]) { sum.add4(v); }, [&](uint32_t, float v) { sum.add1(v); });
        const uint64_t word = merge_threads(sum, sh);
        if (tid == 0u) {
            handed_store(q.word, first + slice, word);
        }
    } else if constexpr (!is_held(FORM)) {
        double m, s;
        merge_slices(lane < q.slices ? handed_load(q.word, first + lane) : 0ull, q.slices, m, s);
        lse = log_sum(m, s);
        if (q.lse != nullptr && slice == 0u && tid == 0u) {
            q.lse[row] = lse.whole();
        }
        pass_over<DT>(mine, write, write_one);
    } else {
        // The slice's values in registers, and its word.
        float v[HELD][GROUP], odd_v = NEG_INF;
        uint32_t odd;
        RowSum sum;
        sum.init();
        if (mine.whole != 0u) {
            groups<DT>(mine, tid - lane, v);
        }
#pragma unroll
        for (int u = 0; u < HELD; ++u) {
            if (tid + (uint32_t)u * 256u < mine.whole) {
                sum.add4(v[u]);
            }
        }
        if (odd_id(mine, odd)) {
            odd_v = odd_value<DT>(mine, odd);
            sum.add1(odd_v);
        }
        const uint64_t word = merge_threads(sum, sh);
        if (q.slices > 1u && tid == 0u) {
            handed_store(q.word, first + slice, word);
        }
        auto store_all = [&] {
#pragma unroll
            for (int u = 0; u < HELD; ++u) {
                const uint32_t g = tid + (uint32_t)u * 256u;
                if (g < mine.whole) {
                    write(mine.lo + g * GROUP, v[u]);
                }
            }
            if (odd < mine.hi) {
                write_one(odd, odd_v);
            }
        };
        // Where the outputs take the logits' place, none is written before the slice's word has arrived: who forms the
        // word itself from the logits, and still finds none behind them, has read logits.
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
                // threads add the same values in the same order).
                for (uint32_t other = 0; other < q.slices; ++other) {
                    if (sh.words[other] != 0ull) {
                        continue;
                    }
                    RowSum again;
                    again.init();
                    pass_over<DT>(
                        take(other), [&](uint32_t, const float (&w)[GROUP]) { again.add4(w); },
                        [&](uint32_t, float w) { again.add1(w); });
                    const uint64_t formed = merge_threads(again, sh);
                    if (tid == 0u) {
                        const uint64_t come = handed_load(q.word, first + other);
                        sh.words[other] = come != 0ull ? come : formed;
                    }
                    __syncthreads();
                }
            }
            double m, s;
            merge_slices(sh.words[lane], q.slices, m, s);
            lse = log_sum(m, s);
            if (q.lse != nullptr && slice == 0u && tid == 0u) {
                q.lse[row] = lse.whole();
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

// (five waves a SIMD where values are held: by itself the compiler takes the registers of four; 276 -> 246 us for
// 1 024 rows of bf16 log-probabilities.  Six spill: 339)
template <int DT, int OT, int FORM>
__global__ void __launch_bounds__(256, is_held(FORM) ? 5 : 1) k_logits_rows_table(const RowArgs* table, LogitsLaunch q) {
    const uint32_t row = blockIdx.x / q.slices, slice = blockIdx.x % q.slices;
    const RowArgs a = row_of((const LILY_CONST RowArgs*)table + row);
    logits_row<DT, OT, FORM>(a, row, slice, q);
}
template <int DT, int OT, int FORM>
__global__ void __launch_bounds__(256, is_held(FORM) ? 5 : 1) k_logits_rows_inline(InlineRows rows, LogitsLaunch q) {
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
                        bool logprobs) {
    if (!logprobs && q.lse == nullptr) {
        return launch_form<DT, OT, FORM_ADJUSTED>(stream, table, few, rows, q);
    }
    if (q.per_slice <= LOGITS_HELD) {
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
            e = w.out_dtype == LILY_BF16 ? launch_typed<LILY_BF16, LILY_BF16>(stream, part, few, n, q, w.logprobs)
                                         : launch_typed<LILY_BF16, LILY_F32>(stream, part, few, n, q, w.logprobs);
        } else {
            e = w.out_dtype == LILY_BF16 ? launch_typed<LILY_F32, LILY_BF16>(stream, part, few, n, q, w.logprobs)
                                         : launch_typed<LILY_F32, LILY_F32>(stream, part, few, n, q, w.logprobs);
        }
        if (e != hipSuccess) {
            return e;
        }
    }
    return hipSuccess;
}

}  // namespace lily
