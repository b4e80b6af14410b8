// distill.hip - a student's rows of logits against a teacher's top ones: loss, and gradient.
//
// With p the teacher's list and q = softmax(z / T):
//     loss = T^2 (sum_j p_j (log p_j - log q_j) [+ P (log P - log Q)]),  grad_v = w T (q_v sum p - p_v) [outside: w T (q_v - P q_v / Q)]
//
// A small launch adds up every row's list.  Then a workgroup takes a slice of a row and keeps it in registers, up to 32 values
// a thread, while the row's slices exchange their sums: a sum is one word (largest value, sum of exponentials), which is the
// whole message, stored and looked for by relaxed atomics at device scope; a second one holds the list's ids, which stand apart where the
// rest counts as one outcome.  So rows are read once and written once.  Whoever misses a word after a number of looks (a neighbour has no
// place on the chip yet) enters its slice into a list and ends; a last launch, which finds every word, does the slices of that list,
// and the losses.  Rows of more than 64 slices go that way altogether.
//
// The gradient is written as an id outside the list has it, everywhere, and then anew for the list's ids, by the thread that
// holds the entry: of an id that the list names twice the first one, found by a bitmap of the slice.  Nothing is added by atomics: the
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

enum Form {
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
    double known;      // of the loss, what does not wait for the row's sum: sum_j p_j (log p_j - z_j / T)
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
    uint64_t* words;    // [rows][slices][2]: of a slice, (largest value << 32 | sum) outside the list, and in it; 0 = not there
    Listed* listed;     // [rows]
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
    for (int n = 0; n < N; ++n) {
        float m = NEG_INF, s = 0.0f;
        for (uint32_t q = 0; q < WAVES; ++q) {
            m = fmaxf(m, part[(q * N + (uint32_t)n) * 2u]);
        }
        for (uint32_t q = 0; q < WAVES; ++q) {
            const float mq = part[(q * N + (uint32_t)n) * 2u];
            s += part[(q * N + (uint32_t)n) * 2u + 1u] * term(mq == NEG_INF ? reference(m) : mq, m, c2);
        }
        t[n] = {m, s};
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
// Its probability up to the list's mass (logits without `rest`: relative to `top`), and as it is.
__device__ __forceinline__ float entry_mass(const DistillArgs& a, float t, float top, float lse) {
    return a.probs != 0u ? t : a.rest != 0u ? exp_of((double)t * a.over_t - (double)lse) : term(t, top, a.c2);
}
__device__ __forceinline__ float entry_probability(const DistillArgs& a, float t, const Listed& l, float lse) {
    return entry_mass(a, t, l.top, lse) * (a.rest != 0u ? 1.0f : 1.0f / l.sum);
}

// A row's list added up, its words cleared: a workgroup a row.
__global__ void __launch_bounds__(256) k_distill_lists(const DistillArgs a) {
    __shared__ float part[4 * 2 * 2];
    __shared__ double part_d[4];
    constexpr uint32_t E = LILY_SAMPLE_K_CAP / 256u;
    const uint32_t tid = threadIdx.x, in_launch = blockIdx.x;
    const uint64_t row = a.row0 + in_launch;
    const uint32_t count = list_length(a, row);
    const float lse = a.teacher_lse != nullptr ? gload(a.teacher_lse + row) : 0.0f;
    const bool relative = a.probs == 0u && a.rest == 0u;
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
    for (uint32_t q = tid; q < a.slices * 2u; q += 256u) {
        store_through(a.words + (uint64_t)in_launch * a.slices * 2u + q, (uint64_t)0);
    }
    Sum mass[2] = {{relative ? NEG_INF : 0.0f, 0.0f}, {NEG_INF, 0.0f}};   // of the list; [1].m: whether any entry counts
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) {
        if (id[e] != LILY_NO_TOKEN) {
            mass[0].m = relative ? fmaxf(mass[0].m, t[e]) : 0.0f;
            mass[1].m = 0.0f;
        }
    }
    const float own = mass[0].m;
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) {
        mass[0].s += id[e] != LILY_NO_TOKEN ? entry_mass(a, t[e], own, lse) : 0.0f;
    }
    group_sums<4u>(mass, a.c2, part);
    const float sum = mass[0].s;
    Listed l = {};
    l.sum = sum;
    l.top = mass[0].m;
    double d = 0.0;   // (in 64 bits: a loss near zero is a difference of large logarithms)
    if (a.loss != nullptr) {
        const void* z = at_row(a.logits, row, a.logits_stride, a.logits_bf16);
        const double log_sum = a.rest != 0u ? 0.0 : log((double)sum);
#pragma unroll
        for (uint32_t e = 0; e < E; ++e) {
            if (id[e] != LILY_NO_TOKEN) {
                const float p = entry_probability(a, t[e], l, lse);
                const double log_p = a.probs != 0u  ? log((double)t[e]) - log_sum
                                     : a.rest != 0u ? (double)t[e] * a.over_t - (double)lse
                                                    : ((double)t[e] - (double)l.top) * a.over_t - log_sum;
                d += p == 0.0f ? 0.0 : (double)p * (log_p - (double)load1(z, id[e], a.logits_bf16) * a.over_t);
            }
        }
        for (int off = 32; off > 0; off >>= 1) {
            d += __shfl_xor(d, off);
        }
        if ((tid & 63u) == 0u) {
            part_d[tid >> 6] = d;
        }
        __syncthreads();
        d = part_d[0] + part_d[1] + part_d[2] + part_d[3];
    }
    if (tid == 0u) {
        l.left = a.rest == 0u ? 0.0f : sum < 1.0f || sum != sum ? 1.0f - sum : 0.0f;
        l.weight = a.grad_scale * (a.row_weights != nullptr ? gload(a.row_weights + row) : 1.0f);
        l.live = mass[1].m == 0.0f && (a.rest != 0u || sum > 0.0f || sum != sum) ? 1u : 0u;
        l.known = d;
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
    r.log_all = m == NEG_INF ? __builtin_nanf("") : logf(r.all.s);
    r.nothing = out.m == NEG_INF && out.s == 0.0f;
    r.log_out = r.nothing ? 0.0f : logf(out.s);
    r.inv_all = m == NEG_INF ? __builtin_nanf("") : 1.0f / r.all.s;
    r.inv_out = 1.0f / out.s;
    r.q_out = term(out.m == NEG_INF ? reference(m) : out.m, m, a.c2) * out.s * r.inv_all;
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

// The gradient of an id outside the list, factor * exp((z - ref) / T), and of one in it, wt * (q - p).
struct Gradient {
    bool zeros;
    float wt, ref, factor;
};
__device__ __forceinline__ Gradient gradient_of(const DistillArgs& a, const RowSums& r, const Listed& l) {
    Gradient g;
    g.zeros = l.live == 0u || l.weight == 0.0f;
    g.wt = l.weight * a.temperature * (l.sum != l.sum ? l.sum : 1.0f);
    g.ref = reference(a.rest != 0u ? r.out.m : r.all.m);
    g.factor = g.zeros        ? 0.0f
               : a.rest == 0u ? g.wt * r.inv_all
               : r.nothing    ? (r.inv_all != r.inv_all ? r.inv_all : 0.0f)
                              : g.wt * (r.q_out - l.left) * r.inv_out;
    return g;
}

// The list as the workgroup sees it.
struct SliceList {
    uint32_t ids[LILY_SAMPLE_K_CAP];   // LILY_NO_TOKEN: does not count
    float z[LILY_SAMPLE_K_CAP], p[LILY_SAMPLE_K_CAP];   // of what lies in the slice: logit, probability
    uint32_t bits[DISTILL_SLICE / 32u];
    uint32_t twice;                    // an id stands there twice
};
// Whether entry j is the first of its id.
__device__ __forceinline__ bool speaks(const SliceList& l, uint32_t j) {
    for (uint32_t q = 0; q < j; ++q) {
        if (l.ids[q] == l.ids[j]) {
            return false;
        }
    }
    return true;
}
// The probabilities of entry j's id, from its first entry on.
__device__ __forceinline__ float added_up(const SliceList& l, uint32_t j, uint32_t k) {
    float p = l.p[j];
    for (uint32_t q = j + 1u; q < k; ++q) {
        p += l.ids[q] == l.ids[j] ? l.p[q] : 0.0f;
    }
    return p;
}

__device__ __forceinline__ uint64_t word_of(Sum s) { return (uint64_t)lilym_f32_bits(s.m) << 32 | lilym_f32_bits(s.s); }
__device__ __forceinline__ Sum sum_of(uint64_t w) { return {lilym_bits_f32((uint32_t)(w >> 32)), lilym_bits_f32((uint32_t)w)}; }

// A row's sums from its slices' words, the same in every lane of a wave.
__device__ __forceinline__ RowSums of_words(const DistillArgs& a, uint32_t lane, const uint64_t (*words)[2]) {
    Sum o = {NEG_INF, 0.0f}, i = {NEG_INF, 0.0f};
    for (uint32_t q = lane; q < a.slices; q += 64u) {
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

// A row's loss and stats, by a wave.
__device__ __forceinline__ void finish_row(const DistillArgs& a, uint32_t in_launch, uint32_t lane) {
    const uint64_t row = a.row0 + in_launch;
    const RowSums r = of_words(a, lane, reinterpret_cast<const uint64_t (*)[2]>(a.words) + (uint64_t)in_launch * a.slices);
    if (lane != 0u) {
        return;
    }
    if (a.stats != nullptr) {
        store_stats(a, row, r);
    }
    if (a.loss != nullptr) {
        // (the sums' part of it: log q = z / T - z0 / T - log(sum); a row of -inf alone has no sum, its logarithm is no number)
        const Listed l = a.listed[in_launch];
        const double log_all = r.log_all != r.log_all ? (double)r.log_all : log((double)r.all.s), top = (double)r.all.m * a.over_t;
        double d = l.known + (double)l.sum * (a.rest != 0u ? 1.0 : 1.0 / (double)l.sum) * (top + log_all);
        if (a.rest != 0u && l.left != 0.0f) {
            const double log_q = r.nothing ? -INFINITY : (double)reference(r.out.m) * a.over_t - top + log((double)r.out.s) - log_all;
            d += (double)l.left * (log((double)l.left) - log_q);
        }
        a.loss[row] = l.live != 0u ? (float)(d * (double)a.temperature * (double)a.temperature) + (r.log_all != r.log_all ? r.log_all : 0.0f) : 0.0f;
    }
}

// Slice `at` (of the launch's rows times slices).  TURNS: pieces of eight a thread holds; a slice is TURNS * TURN ids.
// What a workgroup waits for one after the other is kept short: the list's ids are asked for first, then its slice, behind it the list's
// logits and values; once they are there it waits for its neighbours' words alone.
template <uint32_t TURNS, bool BF16, int FORM>
__device__ __forceinline__ void distill_slice(const DistillArgs& a, uint32_t at) {
    __shared__ SliceList list;
    __shared__ float part[DISTILL_WAVES * 4];
    __shared__ uint64_t words[WORD_SLICES][2];
    __shared__ uint32_t missing;
    constexpr uint32_t SLICE = TURNS * TURN;
    // (the backward pass has sums and needs none; a slice that was left is done as it would have been)
    constexpr bool EXPS = FORM != FORM_BACK, SUMS = FORM == FORM_HELD || FORM == FORM_SUM;
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t slice = at % a.slices, in_launch = at / a.slices;
    const uint64_t row = a.row0 + in_launch;
    const void* z = at_row(a.logits, row, a.logits_stride, BF16);
    const uint32_t whole = a.vocab / 8u;   // whole pieces of a row; the ids behind them are an id a thread
    const uint32_t lo = slice * SLICE, hi = min(lo + SLICE, a.vocab), first = lo / 8u;
    const uint32_t count = list_length(a, row);

    uint32_t id[ENTRIES];
#pragma unroll
    for (uint32_t e = 0; e < ENTRIES; ++e) {
        id[e] = gload(a.ids + row * a.ids_stride + min(e * NT_DISTILL + tid, a.k - 1u));
    }
    Eight<BF16> raw[TURNS];
    if (whole != 0u) {
#pragma unroll
        for (uint32_t c = 0; c < TURNS; ++c) {
            raw[c].load(z, min(first + c * NT_DISTILL + tid, whole - 1u) * 8u);
        }
    }
    const uint32_t last_at = whole * 8u >= lo && whole * 8u + tid < hi ? whole * 8u + tid : LILY_NO_TOKEN;
    const float last = last_at != LILY_NO_TOKEN ? load1(z, last_at, BF16) : NEG_INF;   // the id behind the pieces
    auto there = [&](uint32_t c) { return whole != 0u && first + c * NT_DISTILL + tid < whole; };
    for (uint32_t w = tid; w < SLICE / 32u; w += NT_DISTILL) {
        list.bits[w] = 0u;
    }
    static_assert(SLICE <= DISTILL_SLICE, "a bit for every id of a slice");
    if (tid == 0u) {
        list.twice = 0u;
    }
    __syncthreads();
    bool here[ENTRIES];                        // entries of the slice: of an id that stands there twice, the first
    float mine[ENTRIES], value[ENTRIES];       // their logits, and their values
#pragma unroll
    for (uint32_t e = 0; e < ENTRIES; ++e) {
        const uint32_t j = e * NT_DISTILL + tid, off = id[e] - lo;
        id[e] = j < count && id[e] < a.vocab ? id[e] : LILY_NO_TOKEN;
        here[e] = id[e] >= lo && id[e] < hi;
        mine[e] = NEG_INF;
        value[e] = 0.0f;
        if (j < a.k) {
            list.ids[j] = id[e];
        }
        if (here[e]) {
            mine[e] = load1(z, id[e], BF16);
            value[e] = entry_value(a, row, j);
            if ((atomicOr(&list.bits[off >> 5], 1u << (off & 31u)) >> (off & 31u) & 1u) != 0u) {
                list.twice = 1u;
            }
        }
    }
    __syncthreads();
    const bool twice = list.twice != 0u;
    Listed l = {};
    if constexpr (FORM != FORM_SUM) {
        l = a.listed[in_launch];
        const float lse = a.teacher_lse != nullptr ? gload(a.teacher_lse + row) : 0.0f;
#pragma unroll
        for (uint32_t e = 0; e < ENTRIES; ++e) {
            if (here[e]) {
                list.p[e * NT_DISTILL + tid] = entry_probability(a, value[e], l, lse);
            }
        }
    }
    if (twice) {   // the first of an id speaks for all of them
        __syncthreads();
        float p[ENTRIES];
#pragma unroll
        for (uint32_t e = 0; e < ENTRIES; ++e) {
            here[e] = here[e] && speaks(list, e * NT_DISTILL + tid);
            p[e] = here[e] && FORM != FORM_SUM ? added_up(list, e * NT_DISTILL + tid, a.k) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t e = 0; e < ENTRIES; ++e) {
            if (here[e]) {
                list.p[e * NT_DISTILL + tid] = p[e];
            }
        }
    }
    // (from here on a thread's entries are its own places in LDS: the slice needs the registers)
#pragma unroll
    for (uint32_t e = 0; e < ENTRIES; ++e) {
        const uint32_t j = e * NT_DISTILL + tid;
        if (j < a.k) {
            list.ids[j] = here[e] ? id[e] : LILY_NO_TOKEN;
            list.z[j] = mine[e];
        }
    }

    // The slice's sums, in every thread; its exponentials, relative to the thread's largest value, stay for the gradient.
    Sum s[2] = {{NEG_INF, 0.0f}, {NEG_INF, 0.0f}};
    float x[TURNS][8], last_x = 0.0f, own = NEG_INF;
    if constexpr (EXPS) {
        const uint8_t* named = reinterpret_cast<const uint8_t*>(list.bits);
        const uint32_t behind = last_at - lo;
        const bool counts = last_at != LILY_NO_TOKEN && (a.rest == 0u || (list.bits[behind >> 5] >> (behind & 31u) & 1u) == 0u);
        own = counts ? last : NEG_INF;
#pragma unroll
        for (uint32_t c = 0; c < TURNS; ++c) {
            raw[c].widened(x[c]);
            // What the list names is not outside it (its gradient is formed elsewhere), and what is not there is nothing.
            const uint32_t out = !there(c) ? 255u : a.rest != 0u ? named[c * NT_DISTILL + tid] : 0u;
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
        last_x = counts ? __builtin_amdgcn_exp2f((last - ref) * a.c2) : 0.0f;
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
        if (SUMS && a.rest != 0u) {
            for (uint32_t j = tid; j < a.k; j += NT_DISTILL) {
                if (list.ids[j] != LILY_NO_TOKEN) {
                    const float v = list.z[j];
                    s[1] = joined(s[1], {v, term(v, v, a.c2)}, a.c2);
                }
            }
        }
        if constexpr (SUMS) {
            group_sums<DISTILL_WAVES>(s, a.c2, part);
        }
    }

    uint64_t* out = a.words + (uint64_t)in_launch * a.slices * 2u;
    RowSums r;
    if constexpr (FORM == FORM_SUM) {
        if (tid < 2u) {
            out[slice * 2u + tid] = word_of(tid == 0u ? s[0] : s[1]);
        }
        return;
    } else if constexpr (FORM == FORM_BACK) {
        r = of_stats(a, row);
    } else if constexpr (FORM == FORM_AFTER) {
        r = of_words(a, lane, reinterpret_cast<const uint64_t (*)[2]>(out));
    } else {
        if (tid < 2u) {
            store_through(out + slice * 2u + tid, word_of(tid == 0u ? s[0] : s[1]));
        }
        if (tid < 64u) {
            uint64_t seen[2] = {lane == slice ? word_of(s[0]) : 0ull, lane == slice || a.rest == 0u ? word_of(s[1]) : 0ull};
            bool all = a.slices == 1u;
            for (uint32_t n = 0; n < a.looks && !all; ++n) {
                if (lane < a.slices) {
                    seen[0] = seen[0] == 0ull ? load_through(out + lane * 2u) : seen[0];
                    seen[1] = seen[1] == 0ull ? load_through(out + lane * 2u + 1u) : seen[1];
                }
                all = __ballot(lane < a.slices && (seen[0] == 0ull || seen[1] == 0ull)) == 0ull;
            }
            words[lane][0] = seen[0];
            words[lane][1] = seen[1];
            if (lane == 0u) {
                missing = all ? 0u : 1u;
            }
        }
        __syncthreads();
        if (missing != 0u) {
            if (tid == 0u) {
                a.late[1u + atomicAdd(a.late, 1u)] = at;
            }
            return;
        }
        r = of_words(a, lane, words);
    }
    const Gradient g = gradient_of(a, r, l);
    const uint32_t dtype = a.grad_bf16 != 0u ? LILY_BF16 : LILY_F32;
    void* grad = const_cast<void*>(at_row(a.grad, row, a.grad_stride, a.grad_bf16 != 0u));
    if constexpr (EXPS) {
        // (an infinite or undefined reference has made the sums, and with them the factor, a NaN)
        const float factor = g.zeros ? 0.0f : g.factor * __builtin_amdgcn_exp2f((reference(own) - g.ref) * a.c2);
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
        last_x = g.zeros ? 0.0f : g.factor * term(last, g.ref, a.c2);
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
            raw[c].widened(v);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = g.factor * __builtin_amdgcn_exp2f((v[j] - g.ref) * a.c2);
            }
        }
        if (there(c)) {
            const uint32_t at = (first + c * NT_DISTILL + tid) * 8u;
            if (a.grad_bf16 != 0u) {
                store8(grad, at, v, LILY_BF16);
            } else {
                store8(grad, at, v, LILY_F32);
            }
        }
    }
    if (last_at != LILY_NO_TOKEN) {
        store1(grad, last_at, last_x, dtype);
    }
    if (g.zeros) {
        return;
    }
    // The list's ids anew, behind the stores above.
    __syncthreads();
    for (uint32_t j = tid; j < a.k; j += NT_DISTILL) {
        if (list.ids[j] != LILY_NO_TOKEN) {
            store1(grad, list.ids[j], g.wt * (term(list.z[j], r.all.m, a.c2) * r.inv_all - list.p[j]), dtype);
        }
    }
}

template <uint32_t TURNS, bool BF16, int FORM>
__global__ void __launch_bounds__(NT_DISTILL, TURNS > 4 ? 4 : 6) k_distill(const DistillArgs a) {
    if constexpr (FORM != FORM_AFTER) {
        distill_slice<TURNS, BF16, FORM>(a, blockIdx.x);
    } else {
        // a wave a row for what the rows come to, then slices
        const uint32_t finishers = (a.rows + DISTILL_WAVES - 1u) / DISTILL_WAVES;
        if (blockIdx.x < finishers) {
            const uint32_t in_launch = blockIdx.x * DISTILL_WAVES + (threadIdx.x >> 6);
            if (in_launch < a.rows) {
                finish_row(a, in_launch, threadIdx.x & 63u);
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

// Turns of a slice: where rows are many, as many as a thread holds exponentials of (two workgroups a compute unit in bf16: 2048 rows of
// 151 936 in bf16 266 us by eight, 301 by four, 295 by six, 457 by two; in f32, 1024 rows, 253 by four, 263 by eight), and three for the
// backward pass, which holds nothing (219 against 233 by four and 218 by two; lists of 1000 entries 94, 98 and 100).
constexpr uint32_t TURNS_BACK = 3;
constexpr uint32_t turns_held(bool bf16) { return bf16 ? 8u : 4u; }
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
    } else {
        LILY_DISTILL(turns_held(true), true)
        LILY_DISTILL(turns_held(false), false)
    }
    LILY_DISTILL(1u, true)
    LILY_DISTILL(1u, false)
    LILY_DISTILL(2u, true)
    LILY_DISTILL(2u, false)
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
    // Few rows are cut finer, as long as every workgroup has a place on the chip.
    auto slices = [&](uint64_t turns) { return (d.vocab + turns * TURN - 1u) / (turns * TURN); };
    auto fits = [&](uint64_t turns) { return slices(turns) <= WORD_SLICES && slices(turns) * d.rows <= 768u; };
    const uint32_t turns = fits(1u) ? 1u : fits(2u) ? 2u : backward ? TURNS_BACK : turns_held(a.logits_bf16 != 0u);
    a.slices = (d.vocab + turns * TURN - 1u) / (turns * TURN);
    const bool held = d.grad_dev != nullptr && a.slices <= WORD_SLICES;
    // As many rows at a time as the workspace holds words, lists' sums and lists of slices of.
    const uint64_t each = a.slices * 5ull + sizeof(Listed) / 4u;   // floats
    const uint64_t most = std::min<uint64_t>((ws.part_floats - 4u) / each, 0xffffffffull / ((uint64_t)a.slices * NT_DISTILL) - 1u);
    for (uint64_t row = 0; row < d.rows; row += most) {
        const uint32_t rows = (uint32_t)std::min<uint64_t>(most, d.rows - row), groups = rows * a.slices;
        a.row0 = row;
        a.rows = rows;
        a.words = reinterpret_cast<uint64_t*>(ws.part);
        a.listed = reinterpret_cast<Listed*>(ws.part + (uint64_t)groups * 4u);
        a.late = held && !backward ? reinterpret_cast<uint32_t*>(a.listed + rows) : nullptr;
        hipLaunchKernelGGL(k_distill_lists, dim3(rows), dim3(256), 0, stream, a);
        if (backward) {
            launch_form<FORM_BACK>(stream, a, turns, groups);
            continue;
        }
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
