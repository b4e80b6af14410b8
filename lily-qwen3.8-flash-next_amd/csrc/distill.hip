// distill.hip - a student's rows of logits against a teacher's top ones: loss, and gradient.
//
// With p the teacher's list, q = softmax(z / T) and S = sum p [+ P], which is 1 but where a list has more than 1 beside the rest:
//     loss = T^2 (sum_j p_j (log p_j - log q_j) [+ P (log P - log Q)]),  grad_v = w T (S q_v - p_v) [outside: w T (S q_v - P q_v / Q)]
//
// A workgroup takes a slice of a row and keeps it in registers, up to 64 values a thread, while the row's slices exchange their sums: a sum
// is one word (largest value, sum of exponentials), which is the whole message, stored and looked for by relaxed atomics at device scope;
// a second one holds the list's ids, which stand apart where the rest counts as one outcome, a third what the list adds to the loss.  So
// rows are read once and written once.
//
// Few rows, whose slices all have a place on the chip, are one launch.  Every workgroup adds up its row's list itself.  One that misses a
// word after a number of looks forms that slice's sums itself, by the same operations.  The words lie in a place of their own that is zeros
// between two calls: the last of a row's workgroups clears them.  37 rows of 151 936 in f32 18 us, 24.5 by the three launches that
// more rows take; 8 of them are the memory's, the others trips to it that wait for each other: the list's ids, the logits they name, the
// words, and the gradient.
//
// Of more rows a small launch adds up the lists and clears the words.  Whoever misses a word (a neighbour has no place on the chip yet) enters
// its slice into a list and ends; a last launch, which finds every word, does the slices of that list, and the losses.  Rows of more than 64
// slices go that way altogether.  2048 rows of 151 936 in bf16 251 us (5.0 TB/s), 1024 in f32 258 (4.8).
//
// The gradient is written as an id outside the list has it, everywhere, and then anew for the list's ids, by the thread that
// holds the entry: of an id that the list names twice (a bitmap of the slice says so) the first one.  Nothing is added by atomics: the
// same call gives the same bits.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "operators.h"
#include "row_pieces.h"

namespace lily {

namespace {

constexpr uint32_t NT_DISTILL = DISTILL_THREADS, DISTILL_WAVES = NT_DISTILL / 64u, TURN = NT_DISTILL * 8u;   // ids of a turn
constexpr uint32_t ENTRIES = LILY_SAMPLE_K_CAP / NT_DISTILL;
constexpr uint32_t WORD_SLICES = 64u;   // slices of a row that a wave looks for
constexpr uint32_t WORDS = 3u;          // of a slice

enum Form {
    FORM_ALONE,   // everything, by slices that wait for each other: few rows
    FORM_HELD,    // sums, and the gradient by slices that wait for each other
    FORM_SUM,     // the sums alone
    FORM_AFTER,   // the gradient from the sums of a launch before, of all slices or of those that are left; losses and stats
    FORM_BACK,    // the gradient from stored stats
};

// What a row's list adds up to.
struct Listed {
    float sum, top;    // its mass; the largest value, which logits without `rest` are relative to
    float left;        // P
    float weight;      // of the row's gradient
    uint32_t live;     // some entry counts, and has a probability
    double mass;       // what its entries' masses m_j come to, in 64 bits
    double entropy;    // sum_j m_j log m_j
};

struct DistillArgs {
    const void* logits;
    const uint32_t* ids;
    const void* values;
    const uint32_t* counts;
    const float* teacher_lse;
    const float* row_weights;
    float* loss;
    float* stats;
    void* grad;
    // [rows][slices][WORDS]: of a slice, (largest value << 32 | sum) outside the list, and in it, and the sum of m_j z_j of the entries
    // that lie in it, in 64 bits (-0.0 for zero); 0 = not there
    uint64_t* words;
    Listed* listed;     // [rows]
    uint32_t* done;     // [rows] (of few rows): how many slices need the row's words no more
    uint32_t* late;     // [0]: how many slices are left to the last launch, then which; null: all of them
    uint32_t rows;      // of the launch
    uint64_t logits_stride, ids_stride, values_stride, grad_stride;   // elements
    uint64_t row0;      // of the call's rows, the launch's first
    uint32_t vocab, slices, k, looks;
    uint32_t probs, rest, values_bf16, grad_bf16;
    float temperature, c2, grad_scale;   // c2 = log2(e) / T
    uint32_t logits_bf16;
    double over_t;      // 1 / T
};

// A sum of exponentials: s times exp(m / T); m a largest value, s relative to it (to 0 where m is -inf).
struct Sum {
    float m, s;
};
__device__ __forceinline__ float reference(float m) { return m == NEG_INF ? 0.0f : m; }
__device__ __forceinline__ float term(float v, float m, float c2) { return __builtin_amdgcn_exp2f((v - reference(m)) * c2); }

// N sums over the workgroup, in every thread.  `part`: [waves][N][2].
template <uint32_t WAVES, int N>
__device__ __forceinline__ void group_sums(Sum (&t)[N], float c2, float* part) {
    const uint32_t wave = threadIdx.x >> 6;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const float m = wave_max_dpp(t[n].m);
        const float s = wave_sum_f(t[n].s * term(t[n].m == NEG_INF ? reference(m) : t[n].m, m, c2));
        if ((threadIdx.x & 63u) == 0u) {
            part[(wave * N + (uint32_t)n) * 2u] = m;
            part[(wave * N + (uint32_t)n) * 2u + 1u] = s;
        }
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {   // (a lane a wave's)
        const uint32_t q = (threadIdx.x % WAVES) * N + (uint32_t)n;
        const float mq = part[q * 2u], m = wave_max_dpp(mq), sq = part[q * 2u + 1u] * term(mq == NEG_INF ? reference(m) : mq, m, c2);
        t[n] = {m, wave_sum_f((threadIdx.x & 63u) < WAVES ? sq : 0.0f)};
    }
}

__device__ __forceinline__ const void* at_row(const void* p, uint64_t row, uint64_t stride, bool bf16) {
    return static_cast<const char*>(p) + row * stride * (bf16 ? 2u : 4u);
}
__device__ __forceinline__ uint32_t list_length(const DistillArgs& a, uint64_t row) {
    return a.counts != nullptr ? min(gload(a.counts + row), a.k) : a.k;
}
// Entry j's id, LILY_NO_TOKEN where it does not count.
__device__ __forceinline__ uint32_t entry_id(const DistillArgs& a, uint64_t row, uint32_t count, uint32_t j) {
    const uint32_t id = j < count ? gload(a.ids + row * a.ids_stride + j) : LILY_NO_TOKEN;
    return id < a.vocab ? id : LILY_NO_TOKEN;
}
// Its value as the formulas have it.
__device__ __forceinline__ float entry_value(const DistillArgs& a, uint64_t row, uint32_t j) {
    const float t = load1(at_row(a.values, row, a.values_stride, a.values_bf16), j, a.values_bf16);
    return a.probs != 0u && t < 0.0f ? 0.0f : t;
}
// exp of an argument in 64 bits, within 2 steps of f32: the exponent's fraction is rounded once, at its own size.
__device__ __forceinline__ float exp_of(double x) {
    const double y = x * 1.4426950408889634, n = rint(y);
    return y > -200.0 && y < 200.0 ? ldexpf(__builtin_amdgcn_exp2f((float)(y - n)), (int)n) : y != y ? __builtin_nanf("") : y < 0.0 ? 0.0f : __builtin_huge_valf();
}
// Its probability, without `rest` times the list's mass (logits then: relative to `top`).
__device__ __forceinline__ float entry_mass(const DistillArgs& a, float t, float top, float lse) {
    return a.probs != 0u ? t : a.rest != 0u ? exp_of((double)t * a.over_t - (double)lse) : term(t, top, a.c2);
}

__device__ __forceinline__ double wave_sum_of(double d) {
    for (int off = 32; off > 0; off >>= 1) {
        d += __shfl_xor(d, off);
    }
    return d;
}
// A wave's parts together, behind a barrier.
template <uint32_t WAVES>
__device__ __forceinline__ double together(const double* part) {
    double d = 0.0;
#pragma unroll
    for (uint32_t q = 0; q < WAVES; ++q) {
        d += part[q];
    }
    return d;
}

// A row's list added up, by a workgroup of WAVES waves: a thread has entries e * 64 WAVES + tid.
template <uint32_t WAVES, uint32_t E>
__device__ __forceinline__ Listed add_up(const DistillArgs& a, uint64_t row, const uint32_t (&id)[E], const float (&t)[E], float lse, float* part) {
    const bool relative = a.probs == 0u && a.rest == 0u;
    Sum mass[1] = {{NEG_INF, 0.0f}};   // (relative to 0, where it is not to the largest value: -inf where no entry counts)
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) {
        if (id[e] != LILY_NO_TOKEN) {
            mass[0].m = relative ? fmaxf(mass[0].m, t[e]) : 0.0f;
        }
    }
    const float own = mass[0].m;
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) {
        mass[0].s += id[e] != LILY_NO_TOKEN ? entry_mass(a, t[e], own, lse) : 0.0f;
    }
    group_sums<WAVES>(mass, a.c2, part);
    Listed l = {};
    l.sum = mass[0].s;
    l.top = mass[0].m;
    l.left = a.rest == 0u ? 0.0f : l.sum < 1.0f || l.sum != l.sum ? 1.0f - l.sum : 0.0f;
    l.weight = a.grad_scale * (a.row_weights != nullptr ? gload(a.row_weights + row) : 1.0f);
    l.live = (a.rest != 0u ? l.top == 0.0f : l.sum > 0.0f || l.sum != l.sum) ? 1u : 0u;
    return l;
}
// Its mass and entropy, a wave's parts in part[0][wave] and part[1][wave].  In 64 bits: a loss near zero is a difference of large logarithms,
// and a mass that is off by a rounding is off by that much of the row's largest logit.
template <uint32_t WAVES, uint32_t E>
__device__ __forceinline__ void entropy_of(const DistillArgs& a, const uint32_t (&id)[E], const float (&t)[E], const Listed& l, float lse,
                                           double (*part)[WAVES]) {
    double mass = 0.0, entropy = 0.0;
    if ((threadIdx.x & ~63u) < a.k) {   // (a wave without entries has nothing to add up)
#pragma unroll
        for (uint32_t e = 0; e < E; ++e) {
            if (id[e] != LILY_NO_TOKEN) {
                const double m = (double)entry_mass(a, t[e], l.top, lse);
                const double log_m = a.probs != 0u  ? log((double)t[e])
                                     : a.rest != 0u ? (double)t[e] * a.over_t - (double)lse
                                                    : ((double)t[e] - (double)reference(l.top)) * a.over_t;
                mass += m;
                entropy += m == 0.0 ? 0.0 : m * log_m;
            }
        }
        mass = wave_sum_of(mass);
        entropy = wave_sum_of(entropy);
    }
    if ((threadIdx.x & 63u) == 0u) {
        part[0][threadIdx.x >> 6] = mass;
        part[1][threadIdx.x >> 6] = entropy;
    }
}

// A row's list added up, its words cleared: a workgroup a row.
__global__ void __launch_bounds__(256) k_distill_lists(const DistillArgs a) {
    __shared__ float part[4 * 2];
    __shared__ double part_d[2][4];
    constexpr uint32_t E = LILY_SAMPLE_K_CAP / 256u;
    const uint32_t tid = threadIdx.x, in_launch = blockIdx.x;
    const uint64_t row = a.row0 + in_launch;
    const uint32_t count = list_length(a, row);
    const float lse = a.teacher_lse != nullptr ? gload(a.teacher_lse + row) : 0.0f;
    uint32_t id[E];
    float t[E];
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) {
        const uint32_t j = e * 256u + tid;
        id[e] = LILY_NO_TOKEN;
        t[e] = 0.0f;
        if (j < a.k) {
            id[e] = entry_id(a, row, count, j);
            t[e] = entry_value(a, row, j);
        }
    }
    if (in_launch == 0u && tid == 0u && a.late != nullptr) {
        a.late[0] = 0u;
    }
    for (uint32_t q = tid; q < a.slices * WORDS; q += 256u) {
        store_through(a.words + (uint64_t)in_launch * a.slices * WORDS + q, (uint64_t)0);
    }
    Listed l = add_up<4u>(a, row, id, t, lse, part);
    if (a.loss != nullptr) {
        entropy_of<4u>(a, id, t, l, lse, part_d);
        __syncthreads();
        l.mass = together<4u>(part_d[0]);
        l.entropy = together<4u>(part_d[1]);
    }
    if (tid == 0u) {
        a.listed[in_launch] = l;
    }
}

// exp(-x) with the product's rounding put right: x may be some tens.
__device__ __forceinline__ float exp_minus(float x) {
    const float y = x * -1.4426950408889634f;
    const float rest = __builtin_fmaf(x, -1.4426950408889634f, -y) + x * -1.925963033500e-8f;   // log2(e) - f32(log2(e))
    const float e = __builtin_amdgcn_exp2f(y);
    return fabsf(y) < 126.0f ? __builtin_fmaf(e, rest * 0.69314718f, e) : e;
}

// What a row's sums come to.
struct RowSums {
    Sum all, out;                                // of the whole row, of what lies outside the list (the same without `rest`)
    float log_all, log_out, inv_all, inv_out;    // logarithms and reciprocals of the sums
    float q_out;                                 // Q
    bool nothing;                                // nothing above -inf outside the list
};
__device__ __forceinline__ Sum joined(Sum x, Sum y, float c2) {
    const float m = fmaxf(x.m, y.m);
    return {m, x.s * term(x.m == NEG_INF ? reference(m) : x.m, m, c2) + y.s * term(y.m == NEG_INF ? reference(m) : y.m, m, c2)};
}
__device__ __forceinline__ RowSums of_sums(const DistillArgs& a, Sum out, Sum in) {
    RowSums r;
    r.out = out;
    r.all = joined(out, in, a.c2);
    const float m = r.all.m;
    r.nothing = out.m == NEG_INF && out.s == 0.0f;
    r.log_all = r.log_out = 0.0f;   // (with_logarithms: the gradient needs none)
    r.inv_all = m == NEG_INF ? __builtin_nanf("") : 1.0f / r.all.s;
    r.inv_out = 1.0f / out.s;
    r.q_out = term(out.m == NEG_INF ? reference(m) : out.m, m, a.c2) * out.s * r.inv_all;
    return r;
}
__device__ __forceinline__ RowSums with_logarithms(RowSums r) {
    r.log_all = r.all.m == NEG_INF ? __builtin_nanf("") : logf(r.all.s);
    r.log_out = r.nothing ? 0.0f : logf(r.out.s);
    return r;
}
__device__ __forceinline__ RowSums of_stats(const DistillArgs& a, uint64_t row) {
    const float* from = a.stats + row * 4u;
    RowSums r;
    r.all = {gload(from), 0.0f};
    r.log_all = gload(from + 1);
    r.out = {a.rest != 0u ? gload(from + 2) : r.all.m, 0.0f};
    r.log_out = a.rest != 0u ? gload(from + 3) : r.log_all;
    r.nothing = r.out.m == NEG_INF && r.log_out == 0.0f;
    r.inv_all = exp_minus(r.log_all);
    r.inv_out = exp_minus(r.log_out);
    r.q_out = __builtin_amdgcn_exp2f((reference(r.out.m) - r.all.m) * a.c2) * exp_minus(r.log_all - r.log_out);
    return r;
}
__device__ __forceinline__ void store_stats(const DistillArgs& a, uint64_t row, const RowSums& r) {
    float* to = a.stats + row * 4u;
    to[0] = r.all.m;
    to[1] = r.log_all;
    to[2] = a.rest != 0u ? r.out.m : 0.0f;
    to[3] = a.rest != 0u ? r.log_out : 0.0f;
}

// The gradient of an id outside the list, factor * exp((z - ref) / T), and of one in it, wt * (inv * exp((z - z0) / T) - p).
struct Gradient {
    bool zeros;
    float wt, ref, factor;
    float inv;   // S over the row's sum of exponentials (a list has more than 1 where its rounded logits meet the sum over the exact row)
};
__device__ __forceinline__ Gradient gradient_of(const DistillArgs& a, const RowSums& r, const Listed& l) {
    Gradient g;
    g.zeros = l.live == 0u || l.weight == 0.0f;
    g.wt = l.weight * a.temperature;
    const float total = l.sum != l.sum || (a.rest != 0u && l.sum > 1.0f) ? l.sum : 1.0f;
    g.inv = r.inv_all * total;
    g.ref = reference(a.rest != 0u ? r.out.m : r.all.m);
    g.factor = g.zeros        ? 0.0f
               : a.rest == 0u ? g.wt * g.inv
               : r.nothing    ? (g.inv != g.inv ? g.inv : 0.0f)   // (a NaN in the row or in its list reaches what is 0, too)
                              : g.wt * (r.q_out * total - l.left) * r.inv_out;
    return g;
}

// The list as the workgroup sees it.
struct SliceList {
    alignas(16) uint32_t ids[LILY_SAMPLE_K_CAP];   // LILY_NO_TOKEN: does not count, or not in the slice
    float z[LILY_SAMPLE_K_CAP], p[LILY_SAMPLE_K_CAP];   // of what lies in the slice: logit, probability
    uint32_t bits[DISTILL_SLICE / 32u];
    uint32_t twice;                    // entries whose id another one had marked before
    uint16_t which[LILY_SAMPLE_K_CAP];
    uint32_t marked[LILY_SAMPLE_K_CAP / 32u], silent[LILY_SAMPLE_K_CAP / 32u];   // a bit for each of these; for each that another one speaks for
};
__device__ __forceinline__ uint64_t word_of(Sum s) { return (uint64_t)lilym_f32_bits(s.m) << 32 | lilym_f32_bits(s.s); }
__device__ __forceinline__ Sum sum_of(uint64_t w) { return {lilym_bits_f32((uint32_t)(w >> 32)), lilym_bits_f32((uint32_t)w)}; }

// A row's sums from its slices' words, the same in every lane of a wave.
__device__ __forceinline__ RowSums of_words(const DistillArgs& a, uint32_t lane, const uint64_t (*words)[WORDS]) {
    Sum o = {NEG_INF, 0.0f}, i = {NEG_INF, 0.0f};
    if (lane < a.slices) {
        o = sum_of(words[lane][0]);
        i = sum_of(words[lane][1]);
    }
    for (uint32_t q = lane + 64u; q < a.slices; q += 64u) {
        o = joined(o, sum_of(words[q][0]), a.c2);
        i = joined(i, sum_of(words[q][1]), a.c2);
    }
    auto over_wave = [&](Sum x) {
        const float m = wave_max_dpp(x.m);
        return Sum{m, wave_sum_f(x.s * term(x.m == NEG_INF ? reference(m) : x.m, m, a.c2))};
    };
    const Sum all_o = over_wave(o), all_i = over_wave(i);
    return of_sums(a, all_o, all_i);
}

// Their third words together, the same in every lane of a wave.
__device__ __forceinline__ double products_of_words(const DistillArgs& a, uint32_t lane, const uint64_t (*words)[WORDS]) {
    double d = 0.0;
    for (uint32_t q = lane; q < a.slices; q += 64u) {
        d += __longlong_as_double((long long)words[q][2]);
    }
    return wave_sum_of(d);
}

// From the wave that formed them to the workgroup.
constexpr uint32_t ROW_SUMS = 8;
__device__ __forceinline__ void hand_over(float* to, const RowSums& r) {
    const float v[ROW_SUMS] = {r.all.m, r.all.s, r.out.m, r.out.s, r.inv_all, r.inv_out, r.q_out, r.nothing ? 1.0f : 0.0f};
#pragma unroll
    for (uint32_t i = 0; i < ROW_SUMS; ++i) {
        to[i] = v[i];
    }
}
__device__ __forceinline__ RowSums handed(const float* from) {
    return {{from[0], from[1]}, {from[2], from[3]}, 0.0f, 0.0f, from[4], from[5], from[6], from[7] != 0.0f};
}

// (FORM_ALONE) A workgroup that needs its row's words no more, and has stored its own, says so; the last one clears them for the next call.
__device__ __forceinline__ uint32_t leave_row(const DistillArgs& a, uint32_t in_launch) {
    return threadIdx.x == 0u ? atomicAdd(a.done + in_launch, 1u) : 0u;
}
__device__ __forceinline__ void clear_row(const DistillArgs& a, uint32_t in_launch, uint64_t* words, uint32_t before) {
    if (threadIdx.x < 64u && (uint32_t)__builtin_amdgcn_readfirstlane((int)before) == a.slices - 1u) {
        for (uint32_t q = threadIdx.x; q < a.slices * WORDS; q += 64u) {
            store_through(words + q, (uint64_t)0);
        }
        if (threadIdx.x == 0u) {
            store_through(a.done + in_launch, 0u);
        }
    }
}

// A row's loss and stats, by a thread.
__device__ __forceinline__ void finish_row(const DistillArgs& a, uint64_t row, const RowSums& sums, const Listed& l, double products) {
    const RowSums r = with_logarithms(sums);
    if (a.stats != nullptr) {
        store_stats(a, row, r);
    }
    if (a.loss != nullptr) {
        // (the sums' part of it: log q = z / T - z0 / T - log(sum); a row of -inf alone has no sum, its logarithm is no number)
        const double log_all = r.log_all != r.log_all ? (double)r.log_all : log((double)r.all.s), top = (double)r.all.m * a.over_t;
        double d = l.entropy - products * a.over_t, left = 0.0;
        if (a.rest != 0u) {
            d += l.mass * (top + log_all);
            left = l.mass < 1.0 || l.mass != l.mass ? 1.0 - l.mass : 0.0;
        } else {
            d = d / l.mass - log(l.mass) + (top + log_all);
        }
        if (left != 0.0) {
            const double log_q = r.nothing ? -INFINITY : (double)reference(r.out.m) * a.over_t - top + log((double)r.out.s) - log_all;
            d += left * (log(left) - log_q);
        }
        a.loss[row] = l.live != 0u ? (float)(d * (double)a.temperature * (double)a.temperature) + (r.log_all != r.log_all ? r.log_all : 0.0f) : 0.0f;
    }
}

// A thread's part of a slice: pieces of eight ids, and an id behind the row's last whole piece.
template <uint32_t TURNS, bool BF16>
struct Part {
    Eight<BF16> raw[TURNS];
    uint32_t lo, hi, whole, last_at;
    float last;

    __device__ __forceinline__ void load(const DistillArgs& a, const void* z, uint32_t slice) {
        const uint32_t tid = threadIdx.x;
        whole = a.vocab / 8u;   // pieces of a row
        lo = slice * (TURNS * TURN);
        hi = min(lo + TURNS * TURN, a.vocab);
        if (whole != 0u) {
#pragma unroll
            for (uint32_t c = 0; c < TURNS; ++c) {
                raw[c].load(z, min(lo / 8u + c * NT_DISTILL + tid, whole - 1u) * 8u);
            }
        }
        last_at = whole * 8u >= lo && whole * 8u + tid < hi ? whole * 8u + tid : LILY_NO_TOKEN;
        last = last_at != LILY_NO_TOKEN ? load1(z, last_at, BF16) : NEG_INF;
    }
    __device__ __forceinline__ bool there(uint32_t c) const { return whole != 0u && lo / 8u + c * NT_DISTILL + threadIdx.x < whole; }
};

// The ids that stand in a slice, in LDS (a thread's entries in its own places) and marked; a thread's entries' logits.  The caller's next
// barrier stands behind it.  `id`: as loaded; of those that do not count LILY_NO_TOKEN afterwards.
template <uint32_t TURNS, bool BF16>
__device__ __forceinline__ void enter(const DistillArgs& a, const void* z, const Part<TURNS, BF16>& part, uint32_t count, SliceList& list,
                                      uint32_t (&id)[ENTRIES], bool (&here)[ENTRIES], float (&mine)[ENTRIES]) {
    const uint32_t tid = threadIdx.x;
    for (uint32_t w = tid; w < TURNS * TURN / 32u; w += NT_DISTILL) {
        list.bits[w] = 0u;
    }
    static_assert(ENTRIES * NT_DISTILL == LILY_SAMPLE_K_CAP, "every entry a place");
    static_assert(TURNS * TURN <= DISTILL_SLICE, "a bit for every id of a slice");
    if (tid < LILY_SAMPLE_K_CAP / 32u) {
        list.marked[tid] = list.silent[tid] = 0u;
    }
    if (tid == 0u) {
        list.twice = 0u;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t e = 0; e < ENTRIES; ++e) {
        const uint32_t j = e * NT_DISTILL + tid, off = id[e] - part.lo;
        id[e] = j < count && id[e] < a.vocab ? id[e] : LILY_NO_TOKEN;
        here[e] = id[e] >= part.lo && id[e] < part.hi;
        mine[e] = NEG_INF;
        list.ids[j] = here[e] ? id[e] : LILY_NO_TOKEN;
        if (here[e]) {
            mine[e] = load1(z, id[e], BF16);
            if ((atomicOr(&list.bits[off >> 5], 1u << (off & 31u)) >> (off & 31u) & 1u) != 0u) {
                list.which[atomicAdd(&list.twice, 1u)] = (uint16_t)j;
                atomicOr(&list.marked[j >> 5], 1u << (j & 31u));
            }
        }
    }
}
__device__ __forceinline__ uint32_t wave_min(uint32_t v) {
    for (int off = 32; off > 0; off >>= 1) {
        v = min(v, (uint32_t)__shfl_xor((int)v, off));
    }
    return v;
}
// Of an id that stands there twice the first entry speaks for all of them, with their probabilities added up in their order.  A wave looks
// at the whole list for one marked entry at a time; the first marked one of an id (which of them are marked, the atomics decide) does the rest.
__device__ __forceinline__ void make_unique(SliceList& list) {
    const uint32_t n = list.twice;
    if (n == 0u) {
        return;
    }
    __syncthreads();
    constexpr uint32_t ROUNDS = LILY_SAMPLE_K_CAP / 64u;
    const uint32_t lane = threadIdx.x & 63u;
    for (uint32_t d = threadIdx.x >> 6; d < n; d += DISTILL_WAVES) {
        const uint32_t j = (uint32_t)__builtin_amdgcn_readfirstlane((int)list.which[d]);
        const uint32_t id = (uint32_t)__builtin_amdgcn_readfirstlane((int)list.ids[j]);
        uint32_t first = LILY_NO_TOKEN, first_marked = LILY_NO_TOKEN;
#pragma unroll 4
        for (uint32_t i = 0; i < ROUNDS; ++i) {
            const bool is = list.ids[i * 64u + lane] == id, marked = (list.marked[i * 2u + (lane >> 5)] >> (lane & 31u) & 1u) != 0u;
            const uint32_t q = i * 64u + lane;
            first = min(first, is ? q : LILY_NO_TOKEN);
            first_marked = min(first_marked, is && marked ? q : LILY_NO_TOKEN);
        }
        first = wave_min(first);
        if (wave_min(first_marked) != j) {
            continue;
        }
        float p = 0.0f;
#pragma clang loop unroll(disable)
        for (uint32_t i = 0; i < ROUNDS; ++i) {   // (the masks once more: 32 registers that hold them leave the chip a workgroup less)
            const bool is = list.ids[i * 64u + lane] == id;
            for (uint64_t left = __ballot(is); left != 0ull; left &= left - 1ull) {
                p += list.p[i * 64u + (uint32_t)__builtin_ctzll(left)];
            }
            if (is && i * 64u + lane != first) {
                atomicOr(&list.silent[(i * 64u + lane) >> 5], 1u << (lane & 31u));
            }
        }
        if (lane == 0u) {
            list.p[first] = p;
        }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t e = 0; e < ENTRIES; ++e) {
        const uint32_t j = e * NT_DISTILL + threadIdx.x;
        if ((list.silent[j >> 5] >> (j & 31u) & 1u) != 0u) {
            list.ids[j] = LILY_NO_TOKEN;
        }
    }
}

// A slice's entries' logits and probabilities, kept in the thread's own places in LDS, and a wave's part of the sum of logits times masses
// in part[wave].
__device__ __forceinline__ void keep(const DistillArgs& a, const Listed& l, float lse, SliceList& list, const bool (&here)[ENTRIES],
                                     const float (&z)[ENTRIES], const float (&t)[ENTRIES], double* part) {
    double d = 0.0;
    if ((threadIdx.x & ~63u) < a.k) {
#pragma unroll
        for (uint32_t e = 0; e < ENTRIES; ++e) {
            if (here[e]) {
                const float m = entry_mass(a, t[e], l.top, lse);
                list.z[e * NT_DISTILL + threadIdx.x] = z[e];
                list.p[e * NT_DISTILL + threadIdx.x] = m * (a.rest != 0u ? 1.0f : 1.0f / l.sum);
                d += m == 0.0f ? 0.0 : (double)m * (double)z[e];
            }
        }
        if (a.loss != nullptr) {
            d = wave_sum_of(d);
        }
    }
    if ((threadIdx.x & 63u) == 0u) {
        part[threadIdx.x >> 6] = d;
    }
}
__device__ __forceinline__ uint64_t word_of(double d) { return (uint64_t)__double_as_longlong(d == 0.0 ? -0.0 : d); }

// A thread's exponentials of a slice, relative to its largest value `own`, and its sums: outside the list, and in it.
template <uint32_t TURNS, bool BF16>
__device__ __forceinline__ void exponentials(const DistillArgs& a, const Part<TURNS, BF16>& part, const SliceList& list, bool sums, float (&x)[TURNS][8],
                                             float& last_x, float& own, Sum (&s)[2]) {
    const uint8_t* named = reinterpret_cast<const uint8_t*>(list.bits);
    const uint32_t tid = threadIdx.x, behind = part.last_at - part.lo;
    const bool counts = part.last_at != LILY_NO_TOKEN && (a.rest == 0u || (list.bits[behind >> 5] >> (behind & 31u) & 1u) == 0u);
    own = counts ? part.last : NEG_INF;
#pragma unroll
    for (uint32_t c = 0; c < TURNS; ++c) {
        part.raw[c].widened(x[c]);
        // What the list names is not outside it (its gradient is formed elsewhere), and what is not there is nothing.
        const uint32_t out = !part.there(c) ? 255u : a.rest != 0u ? named[c * NT_DISTILL + tid] : 0u;
        if (out != 0u) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[c][j] = (out >> j & 1u) != 0u ? NEG_INF : x[c][j];
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            own = fmaxf(own, x[c][j]);
        }
    }
    const float ref = reference(own);
    last_x = counts ? __builtin_amdgcn_exp2f((part.last - ref) * a.c2) : 0.0f;
    float sum = last_x;
#pragma unroll
    for (uint32_t c = 0; c < TURNS; ++c) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[c][j] = __builtin_amdgcn_exp2f((x[c][j] - ref) * a.c2);
            sum += x[c][j];
        }
    }
    s[0] = {own, sum};
    s[1] = {NEG_INF, 0.0f};
    if (sums && a.rest != 0u) {
        for (uint32_t j = tid; j < a.k; j += NT_DISTILL) {
            if (list.ids[j] != LILY_NO_TOKEN) {
                const float v = list.z[j];
                s[1] = joined(s[1], {v, term(v, v, a.c2)}, a.c2);
            }
        }
    }
}


// (FORM_ALONE) The words of the slices `left` of the row that slice `at` belongs to, which have not come: from the logits, by the operations
// of their own workgroups.  What has come by then stands: that workgroup may have stored its gradient over the logits since, and has
// stored the words first.  Not a part of its caller: that keeps its own slice in registers.  `of`: the kernel's arguments.
template <uint32_t TURNS, bool BF16>
__device__ __attribute__((noinline)) void words_of_slices(const DistillArgs* of, uint32_t at, uint64_t left, uint64_t* words) {
    __shared__ SliceList list;
    __shared__ float sums[DISTILL_WAVES * 4];
    __shared__ double products[DISTILL_WAVES];
    const DistillArgs a = *of;
    const uint32_t tid = threadIdx.x, in_launch = at / a.slices;
    const uint64_t row = a.row0 + in_launch;
    const void* z = at_row(a.logits, row, a.logits_stride, BF16);
    const uint32_t count = list_length(a, row);
    const float lse = a.teacher_lse != nullptr ? gload(a.teacher_lse + row) : 0.0f;
    for (; left != 0ull; left &= left - 1ull) {
        const uint32_t slice = (uint32_t)__builtin_ctzll(left);
        uint32_t id[ENTRIES];
        float value[ENTRIES], mine[ENTRIES];
        bool here[ENTRIES];
#pragma unroll
        for (uint32_t e = 0; e < ENTRIES; ++e) {
            id[e] = gload(a.ids + row * a.ids_stride + min(e * NT_DISTILL + tid, a.k - 1u));
            value[e] = entry_value(a, row, min(e * NT_DISTILL + tid, a.k - 1u));
        }
        Part<TURNS, BF16> part;
        part.load(a, z, slice);
        enter(a, z, part, count, list, id, here, mine);
        const Listed l = add_up<DISTILL_WAVES>(a, row, id, value, lse, sums);
        __syncthreads();
        keep(a, l, lse, list, here, mine, value, products);
        make_unique(list);
        Sum s[2];
        float x[TURNS][8], last_x, own;
        exponentials(a, part, list, true, x, last_x, own, s);
        group_sums<DISTILL_WAVES>(s, a.c2, sums);
        if (tid < WORDS) {
            const uint64_t come = load_through(a.words + ((uint64_t)in_launch * a.slices + slice) * WORDS + tid);
            words[slice * WORDS + tid] = come != 0ull ? come : tid == 2u ? word_of(together<DISTILL_WAVES>(products)) : word_of(tid == 0u ? s[0] : s[1]);
        }
        __syncthreads();   // (the list and the sums' places have been read)
    }
}

// Slice `at` (of the launch's rows times slices).  TURNS: pieces of eight a thread holds; a slice is TURNS * TURN ids.
// What a workgroup waits for one after the other is kept short: the list's ids are asked for first, then its slice, behind it the list's
// logits and values; once they are there it waits for its neighbours' words alone.
template <uint32_t TURNS, bool BF16, int FORM>
__device__ __forceinline__ void distill_slice(const DistillArgs& a, uint32_t at) {
    __shared__ SliceList list;
    __shared__ float sums[DISTILL_WAVES * 4];
    __shared__ double entropy[2][DISTILL_WAVES];   // (FORM_ALONE)
    __shared__ uint64_t words[WORD_SLICES][WORDS];
    __shared__ double products[DISTILL_WAVES];
    __shared__ uint64_t missing;
    __shared__ float come[ROW_SUMS];
    // (the backward pass has sums and needs none; a slice that was left is done as it would have been)
    constexpr bool EXPS = FORM != FORM_BACK, SUMS = FORM == FORM_ALONE || FORM == FORM_HELD || FORM == FORM_SUM;
    constexpr bool ADDS = FORM == FORM_ALONE || FORM == FORM_BACK;   // adds up its row's list itself
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t slice = at % a.slices, in_launch = at / a.slices;
    const uint64_t row = a.row0 + in_launch;
    const void* z = at_row(a.logits, row, a.logits_stride, BF16);
    const uint32_t count = list_length(a, row);

    const float lse = a.teacher_lse != nullptr ? gload(a.teacher_lse + row) : 0.0f;
    uint64_t* out = a.words + (uint64_t)in_launch * a.slices * WORDS;
    const bool finishes = FORM == FORM_ALONE && slice == 0u && a.loss != nullptr;   // (the others have no use for the third words)

    uint32_t id[ENTRIES];
    float value[ENTRIES];
#pragma unroll
    for (uint32_t e = 0; e < ENTRIES; ++e) {
        id[e] = gload(a.ids + row * a.ids_stride + min(e * NT_DISTILL + tid, a.k - 1u));
        value[e] = ADDS ? entry_value(a, row, min(e * NT_DISTILL + tid, a.k - 1u)) : 0.0f;
    }
    Part<TURNS, BF16> part;
    part.load(a, z, slice);
    bool here[ENTRIES];   // entries of the slice
    float mine[ENTRIES];
    enter(a, z, part, count, list, id, here, mine);
    Listed l = {};
    if constexpr (ADDS) {
        l = add_up<DISTILL_WAVES>(a, row, id, value, lse, sums);
    } else {
#pragma unroll
        for (uint32_t e = 0; e < ENTRIES; ++e) {
            if (here[e]) {
                value[e] = entry_value(a, row, e * NT_DISTILL + tid);
            }
        }
        l = a.listed[in_launch];
    }
    __syncthreads();
    // (from here on a thread's entries are its own places in LDS: the slice needs the registers)
    keep(a, l, lse, list, here, mine, value, products);
    make_unique(list);

    Sum s[2];   // the slice's, in every thread; its exponentials stay for the gradient
    float x[TURNS][8], last_x = 0.0f, own = NEG_INF;
    if constexpr (EXPS) {
        exponentials(a, part, list, SUMS, x, last_x, own, s);
        if constexpr (SUMS) {
            group_sums<DISTILL_WAVES>(s, a.c2, sums);
        }
    }
    const uint64_t word = !SUMS ? 0ull : tid == 2u ? word_of(together<DISTILL_WAVES>(products)) : word_of(tid == 0u ? s[0] : s[1]);
    RowSums r;
    if constexpr (FORM == FORM_SUM) {
        if (tid < WORDS) {
            out[slice * WORDS + tid] = word;
        }
        return;
    } else if constexpr (FORM == FORM_BACK) {
        r = of_stats(a, row);
    } else if constexpr (FORM == FORM_AFTER) {
        r = of_words(a, lane, reinterpret_cast<const uint64_t (*)[WORDS]>(out));
    } else {
        if (tid < WORDS) {
            store_through(out + slice * WORDS + tid, word);
            words[slice][tid] = word;
        }
        if constexpr (FORM == FORM_ALONE) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (the words have arrived before anything of the gradient has)
            if (a.grad == nullptr && slice != 0u) {
                clear_row(a, in_launch, out, leave_row(a, in_launch));
                return;
            }
        }
        if (finishes) {   // (while the words are on their way)
            entropy_of<DISTILL_WAVES>(a, id, value, l, lse, entropy);
        }
        if (tid < 64u) {
            const bool asks = lane < a.slices && lane != slice;
            uint64_t seen[3] = {0ull, a.rest == 0u ? word_of(Sum{NEG_INF, 0.0f}) : 0ull, finishes ? 0ull : word_of(0.0)};
            uint64_t left = __ballot(asks);
            for (uint32_t n = 0; n < a.looks && left != 0ull; ++n) {
                if (asks) {
#pragma unroll
                    for (uint32_t w = 0; w < WORDS; ++w) {
                        seen[w] = seen[w] == 0ull ? load_through(out + lane * WORDS + w) : seen[w];
                    }
                }
                left = __ballot(asks && (seen[0] == 0ull || seen[1] == 0ull || seen[2] == 0ull));
            }
            if (asks) {
#pragma unroll
                for (uint32_t w = 0; w < WORDS; ++w) {
                    words[lane][w] = seen[w];
                }
            }
            const RowSums w = of_words(a, lane, words);
            if (lane == 0u) {
                missing = left;
                hand_over(come, w);
            }
        }
        __syncthreads();
        if constexpr (FORM == FORM_HELD) {
            if (missing != 0ull) {
                if (tid == 0u) {
                    a.late[1u + atomicAdd(a.late, 1u)] = at;
                }
                return;
            }
        } else if (missing != 0ull) {
            words_of_slices<TURNS, BF16>(reinterpret_cast<const DistillArgs*>((const void*)__builtin_amdgcn_kernarg_segment_ptr()), at, missing, &words[0][0]);
            const RowSums w = of_words(a, lane, words);
            if (tid == 0u) {
                hand_over(come, w);
            }
            __syncthreads();
        }
        r = handed(come);
    }
    uint32_t left_before = 0u;
    if constexpr (FORM == FORM_ALONE) {
        if (a.grad == nullptr) {
            if (tid >= NT_DISTILL - 64u) {
                const double d = products_of_words(a, lane, words);
                l.mass = together<DISTILL_WAVES>(entropy[0]);
                l.entropy = together<DISTILL_WAVES>(entropy[1]);
                if (lane == 0u) {
                    finish_row(a, row, r, l, d);
                }
            }
            clear_row(a, in_launch, out, leave_row(a, in_launch));
            return;
        }
        left_before = leave_row(a, in_launch);
    }
    const Gradient g = gradient_of(a, r, l);
    const uint32_t dtype = a.grad_bf16 != 0u ? LILY_BF16 : LILY_F32;
    void* grad = const_cast<void*>(at_row(a.grad, row, a.grad_stride, a.grad_bf16 != 0u));
    if constexpr (EXPS) {
        // (an infinite or undefined reference has made the sums, and with them the factor, a NaN.  Where there is nothing above -inf the
        // exponentials are zeros: nothing is to be made of a distance from 0, exp of which may be infinite)
        const float factor = g.zeros ? 0.0f : g.factor * term(own == NEG_INF ? g.ref : own, g.ref, a.c2);
#pragma unroll
        for (uint32_t c = 0; c < TURNS; ++c) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[c][j] = factor * x[c][j];
            }
        }
        last_x = factor * last_x;
        if (g.zeros) {   // (whatever the row holds)
            last_x = 0.0f;
#pragma unroll
            for (uint32_t c = 0; c < TURNS; ++c) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    x[c][j] = 0.0f;
                }
            }
        }
    } else {
        last_x = g.zeros ? 0.0f : g.factor * term(part.last, g.ref, a.c2);
    }
#pragma unroll
    for (uint32_t c = 0; c < TURNS; ++c) {
        float v[8] = {};
        if constexpr (EXPS) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = x[c][j];
            }
        } else if (!g.zeros) {
            part.raw[c].widened(v);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = g.factor * __builtin_amdgcn_exp2f((v[j] - g.ref) * a.c2);
            }
        }
        if (part.there(c)) {
            const uint32_t at = part.lo + (c * NT_DISTILL + tid) * 8u;
            if (a.grad_bf16 != 0u) {
                store8(grad, at, v, LILY_BF16);
            } else {
                store8(grad, at, v, LILY_F32);
            }
        }
    }
    if (part.last_at != LILY_NO_TOKEN) {
        store1(grad, part.last_at, last_x, dtype);
    }
    if (!g.zeros) {   // the list's ids anew, behind the stores above
        __syncthreads();
        for (uint32_t j = tid; j < a.k; j += NT_DISTILL) {
            if (list.ids[j] != LILY_NO_TOKEN) {
                store1(grad, list.ids[j], g.wt * (term(list.z[j], r.all.m, a.c2) * g.inv - list.p[j]), dtype);
            }
        }
    }
    if constexpr (FORM == FORM_ALONE) {
        if (slice == 0u && tid >= NT_DISTILL - 64u) {
            const double d = products_of_words(a, lane, words);
            l.mass = together<DISTILL_WAVES>(entropy[0]);
            l.entropy = together<DISTILL_WAVES>(entropy[1]);
            if (lane == 0u) {
                finish_row(a, row, r, l, d);
            }
        }
        clear_row(a, in_launch, out, left_before);
    }
}

// (waves of a SIMD: held in f32 four workgroups a compute unit take 258 us where three, of 67 registers, take 268.  Few rows in one launch have 104 to
// 184 bytes of scratch a lane, the call's of words_of_slices and, of two turns, six registers spilled)
template <uint32_t TURNS, bool BF16, int FORM>
__global__ void __launch_bounds__(NT_DISTILL, TURNS > 4 ? 4 : FORM == FORM_HELD ? 8 : 6) k_distill(const DistillArgs a) {
    if constexpr (FORM != FORM_AFTER) {
        distill_slice<TURNS, BF16, FORM>(a, blockIdx.x);
    } else {
        // a wave a row for what the rows come to, then slices
        const uint32_t finishers = (a.rows + DISTILL_WAVES - 1u) / DISTILL_WAVES;
        if (blockIdx.x < finishers) {
            const uint32_t in_launch = blockIdx.x * DISTILL_WAVES + (threadIdx.x >> 6);
            if (in_launch < a.rows) {
                const uint32_t lane = threadIdx.x & 63u;
                const auto words = reinterpret_cast<const uint64_t (*)[WORDS]>(a.words) + (uint64_t)in_launch * a.slices;
                const RowSums r = of_words(a, lane, words);
                const double d = products_of_words(a, lane, words);
                if (lane == 0u) {
                    finish_row(a, a.row0 + in_launch, r, a.listed[in_launch], d);
                }
            }
            return;
        }
        const uint32_t left = a.late != nullptr ? a.late[0] : a.rows * a.slices;
        for (uint32_t i = blockIdx.x - finishers; i < left; i += gridDim.x - finishers) {
            distill_slice<TURNS, BF16, FORM>(a, a.late != nullptr ? a.late[1u + i] : i);
            __syncthreads();
        }
    }
}

// Turns of a slice.  Four fill the chip best, 32 exponentials a thread; from some 700 rows on in bf16 eight (two workgroups a compute unit)
// have fewer lists to look through and words to wait for: 128 rows of 151 936 31.4 us by four and 33 by eight, 256 51.8 and 55, 512 81 and 82.5, 700
// 103 both, 1024 141 and 139, 2048 with `rest` 271 and 251; 300 of 248 320 with lists of 1000 128 and 134.  (By six 87 and 151 at 512 and 1024; in f32,
// 1024 rows, 253 by four and 263 by eight.)  Three for the backward pass, which holds nothing (219 against 233 by four and 218 by two; lists
// of 1000 entries 94, 98 and 100); it adds up the lists itself, in every slice: 300 rows of 248 320 with lists of 1000 89 against 94 with a launch
// for them, 2048 of 151 936 with lists of 64 221 against 219.
constexpr uint32_t TURNS_BACK = 3, TURNS_HELD = 4, TURNS_MANY = 8;
constexpr uint64_t MANY_GROUPS = 7168;   // by four
template <int FORM>
void launch_form(hipStream_t stream, const DistillArgs& a, uint32_t turns, uint32_t groups) {
    const dim3 grid(groups), block(NT_DISTILL);
#define LILY_DISTILL(TURNS, BF16)                                                                       \
    if (turns == TURNS && (a.logits_bf16 != 0u) == BF16) {                                              \
        hipLaunchKernelGGL((k_distill<TURNS, BF16, FORM>), grid, block, 0, stream, a);                  \
    }
    if constexpr (FORM == FORM_BACK) {
        LILY_DISTILL(TURNS_BACK, true)
        LILY_DISTILL(TURNS_BACK, false)
    }
    if constexpr (FORM == FORM_BACK || FORM == FORM_ALONE) {
        LILY_DISTILL(1u, true)
        LILY_DISTILL(1u, false)
        LILY_DISTILL(2u, true)
        LILY_DISTILL(2u, false)
    } else {
        LILY_DISTILL(TURNS_MANY, true)
        LILY_DISTILL(TURNS_HELD, true)
        LILY_DISTILL(TURNS_HELD, false)
    }
#undef LILY_DISTILL
}

}  // namespace

hipError_t launch_distill(hipStream_t stream, const lily_distillation& d, bool backward, const ProjectWorkspace& ws) {
    DistillArgs a = {};
    a.logits = d.logits_dev;
    a.ids = d.ids_dev;
    a.values = d.values_dev;
    a.counts = d.counts_dev;
    a.teacher_lse = d.teacher_lse_dev;
    a.row_weights = d.row_weights_dev;
    a.loss = d.loss_dev;
    a.stats = d.stats_dev;
    a.grad = d.grad_dev;
    a.logits_stride = d.logits_stride;
    a.ids_stride = d.ids_stride;
    a.values_stride = d.values_stride;
    a.grad_stride = d.grad_stride;
    a.vocab = d.vocab;
    a.k = d.k;
    a.looks = ws.looks;
    a.probs = d.teacher == LILY_TEACHER_PROBS;
    a.rest = d.rest;
    a.values_bf16 = d.values_dtype == LILY_BF16;
    a.grad_bf16 = d.grad_dtype == LILY_BF16;
    a.temperature = d.temperature;
    a.c2 = (float)(1.4426950408889634 / (double)d.temperature);
    a.over_t = 1.0 / (double)d.temperature;
    a.logits_bf16 = d.logits_dtype == LILY_BF16;
    a.grad_scale = d.grad_scale;
    // Few rows are cut finer, as long as every workgroup has a place on the chip; then one launch does everything.
    auto slices = [&](uint64_t turns) { return (d.vocab + turns * TURN - 1u) / (turns * TURN); };
    auto fits = [&](uint64_t turns) { return slices(turns) <= WORD_SLICES && slices(turns) * d.rows <= DISTILL_ALONE; };
    // (what one launch rests on beside whole words is the hardware's: that a workgroup's words have arrived when it counts them so, before its
    // gradient and before it is counted out)
#ifdef LILY_STRICT_HANDOVER
    const bool few = backward && fits(2u);
#else
    const bool few = fits(2u) && (backward || !ws.strict);
#endif
    const bool many = a.logits_bf16 != 0u && (slices(TURNS_HELD) > WORD_SLICES || slices(TURNS_HELD) * d.rows > MANY_GROUPS);
    const uint32_t turns = few && fits(1u) ? 1u : few ? 2u : backward ? TURNS_BACK : many ? TURNS_MANY : TURNS_HELD;
    a.slices = (uint32_t)slices(turns);
    if (few || backward) {
        a.words = ws.exchange;
        a.done = reinterpret_cast<uint32_t*>(ws.exchange + WORDS * DISTILL_ALONE);
        const uint64_t most = 0xffffffffull / ((uint64_t)a.slices * NT_DISTILL) - 1u;   // rows of a launch
        for (uint64_t row = 0; row < d.rows; row += most) {
            const uint32_t rows = (uint32_t)std::min<uint64_t>(most, d.rows - row);
            a.row0 = row;
            if (backward) {
                launch_form<FORM_BACK>(stream, a, turns, rows * a.slices);
            } else {
                launch_form<FORM_ALONE>(stream, a, turns, rows * a.slices);
            }
        }
        return hipGetLastError();
    }
    const bool held = d.grad_dev != nullptr && a.slices <= WORD_SLICES;
    // As many rows at a time as the workspace holds words, lists' sums and lists of slices of.
    const uint64_t each = a.slices * (WORDS * 2ull + 1u) + sizeof(Listed) / 4u;   // floats
    const uint64_t most = std::min<uint64_t>((ws.part_floats - 4u) / each, 0xffffffffull / ((uint64_t)a.slices * NT_DISTILL) - 1u);
    for (uint64_t row = 0; row < d.rows; row += most) {
        const uint32_t rows = (uint32_t)std::min<uint64_t>(most, d.rows - row), groups = rows * a.slices;
        a.row0 = row;
        a.rows = rows;
        a.words = reinterpret_cast<uint64_t*>(ws.part);
        a.listed = reinterpret_cast<Listed*>(ws.part + (uint64_t)groups * (WORDS * 2u));
        a.late = held ? reinterpret_cast<uint32_t*>(a.listed + rows) : nullptr;
        hipLaunchKernelGGL(k_distill_lists, dim3(rows), dim3(256), 0, stream, a);
        if (held) {
            launch_form<FORM_HELD>(stream, a, turns, groups);
        } else {
            launch_form<FORM_SUM>(stream, a, turns, groups);
        }
        const uint32_t finishers = (rows + DISTILL_WAVES - 1u) / DISTILL_WAVES;
        launch_form<FORM_AFTER>(stream, a, turns, finishers + (d.grad_dev == nullptr ? 0u : held ? std::min(groups, 256u) : groups));
    }
    return hipGetLastError();
}

}  // namespace lily
