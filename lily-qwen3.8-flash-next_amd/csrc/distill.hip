// distill.hip - a student's rows of logits against a teacher's top ones: loss, and gradient.
//
// With p the teacher's list and q = softmax(z / T):
//     loss = T^2 (sum_j p_j (log p_j - log q_j) [+ P (log P - log Q)]),  grad_v = w T (q_v sum p - p_v) [outside: w T (q_v - P q_v / Q)]
//
// A workgroup takes a slice of a row, 32 values a thread in registers.  One launch leaves each slice's largest value and sum
// of exponentials (ids in the list apart where the rest counts as one outcome) and the list's logits in the workspace; the
// next combines them, every workgroup for itself, and writes the gradient: first what an id outside the list gets,
// everywhere, then the list's ids anew.  So an id that the list names twice is found by a bitmap of the slice, and nothing
// is added by atomics.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "operators.h"
#include "row_pieces.h"

namespace lily {

namespace {

constexpr uint32_t NT_DISTILL = DISTILL_THREADS, PIECES = DISTILL_SLICE / 8u / NT_DISTILL, ENTRIES = LILY_SAMPLE_K_CAP / NT_DISTILL;
constexpr uint32_t DISTILL_WAVES = NT_DISTILL / 64u;

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
    float* records;     // [rows][slices][4]: largest value and sum outside the list, the same in it
    float* list;        // [rows][k]: the list's logits
    uint64_t logits_stride, ids_stride, values_stride, grad_stride;   // elements
    uint32_t row0, vocab, slices, k;   // row0: of the call's rows, the launch's first
    uint32_t probs, rest, logits_bf16, values_bf16, grad_dtype, backward;
    float temperature, c2, grad_scale;   // c2 = log2(e) / T
};

// A sum of exponentials: s times exp(m / T); m a largest value, s relative to it (to 0 where m is -inf).
struct Sum {
    float m, s;
};
__device__ __forceinline__ float reference(float m) { return m == NEG_INF ? 0.0f : m; }
__device__ __forceinline__ float term(float v, float m, float c2) { return __builtin_amdgcn_exp2f((v - reference(m)) * c2); }

// N sums over the workgroup, in every thread.  `part`: [waves][N][2].
template <int N>
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
        for (uint32_t q = 0; q < DISTILL_WAVES; ++q) {
            m = fmaxf(m, part[(q * N + (uint32_t)n) * 2u]);
        }
        for (uint32_t q = 0; q < DISTILL_WAVES; ++q) {
            const float mq = part[(q * N + (uint32_t)n) * 2u];
            s += part[(q * N + (uint32_t)n) * 2u + 1u] * term(mq == NEG_INF ? reference(m) : mq, m, c2);
        }
        t[n] = {m, s};
    }
}

// Which of the list's ids lie in a slice, who speaks for an id that stands there twice, and what it adds up to.
struct SliceList {
    uint32_t ids[LILY_SAMPLE_K_CAP];     // LILY_NO_TOKEN: does not count
    float p[LILY_SAMPLE_K_CAP];
    uint32_t bits[DISTILL_SLICE / 32u];
    uint32_t twice;
};

__device__ __forceinline__ uint32_t valid_id(const DistillArgs& a, uint64_t row, uint32_t count, uint32_t j) {
    const uint32_t id = j < count ? gload(a.ids + row * a.ids_stride + j) : LILY_NO_TOKEN;
    return id < a.vocab ? id : LILY_NO_TOKEN;
}
__device__ __forceinline__ uint32_t list_length(const DistillArgs& a, uint64_t row) {
    return a.counts != nullptr ? min(gload(a.counts + row), a.k) : a.k;
}
// Whether entry j is the first of its id.
__device__ __forceinline__ bool speaks(const SliceList& l, uint32_t j) {
    for (uint32_t q = 0; q < j; ++q) {
        if (l.ids[q] == l.ids[j]) {
            return false;
        }
    }
    return true;
}

__device__ __forceinline__ const void* at_row(const void* p, uint64_t row, uint64_t stride, bool bf16) {
    return static_cast<const char*>(p) + row * stride * (bf16 ? 2u : 4u);
}

// A thread's share of a slice: pieces of eight, as they lie in memory; what is not there is -inf.
struct Held {
    float v[PIECES][8];
};
__device__ __forceinline__ uint32_t piece_at(uint32_t c) { return (c * NT_DISTILL + threadIdx.x) * 8u; }
__device__ __forceinline__ void hold(const DistillArgs& a, const void* z, uint32_t lo, Held& h) {
    Raw raw[PIECES];
#pragma unroll
    for (uint32_t c = 0; c < PIECES; ++c) {
        const uint32_t i = lo + piece_at(c);
        if (i + 8u <= a.vocab) {
            raw[c] = load8(z, i, a.logits_bf16);
        }
    }
#pragma unroll
    for (uint32_t c = 0; c < PIECES; ++c) {
        const uint32_t i = lo + piece_at(c);
        if (i + 8u <= a.vocab) {
            widen(raw[c], a.logits_bf16, h.v[c]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                h.v[c][j] = i + (uint32_t)j < a.vocab ? load1(z, i + (uint32_t)j, a.logits_bf16) : NEG_INF;
            }
        }
    }
}

__global__ void __launch_bounds__(NT_DISTILL) k_distill_sums(const DistillArgs a) {
    __shared__ SliceList list;
    __shared__ float part[DISTILL_WAVES * 4];
    const uint32_t tid = threadIdx.x, slice = blockIdx.x % a.slices, in_launch = blockIdx.x / a.slices;
    const uint64_t row = (uint64_t)a.row0 + in_launch;
    const uint32_t lo = slice * DISTILL_SLICE;
    const void* z = at_row(a.logits, row, a.logits_stride, a.logits_bf16);
    Held h;
    hold(a, z, lo, h);
    const uint32_t count = list_length(a, row);
    Sum sums[2] = {{NEG_INF, 0.0f}, {NEG_INF, 0.0f}};
    if (a.rest != 0u) {
        list.bits[tid] = 0u;
        if (tid == 0u) {
            list.twice = 0u;
        }
        __syncthreads();
    }
    static_assert(DISTILL_SLICE / 32u == NT_DISTILL, "a word of the bitmap a thread");
    float mine[ENTRIES];
#pragma unroll
    for (uint32_t e = 0; e < ENTRIES; ++e) {
        const uint32_t j = e * NT_DISTILL + tid;
        mine[e] = NEG_INF;
        if (j < a.k) {
            const uint32_t id = valid_id(a, row, count, j), off = id - lo;
            const bool here = id != LILY_NO_TOKEN && id >= lo && off < DISTILL_SLICE;
            list.ids[j] = here ? id : LILY_NO_TOKEN;
            if (here) {
                mine[e] = load1(z, id, a.logits_bf16);
                a.list[(uint64_t)in_launch * a.k + j] = mine[e];
                if (a.rest != 0u && (atomicOr(&list.bits[off >> 5], 1u << (off & 31u)) >> (off & 31u) & 1u) != 0u) {
                    list.twice = 1u;
                }
            }
        }
    }
    if (a.rest != 0u) {
        __syncthreads();
        const bool twice = list.twice != 0u;
#pragma unroll
        for (uint32_t e = 0; e < ENTRIES; ++e) {
            const uint32_t j = e * NT_DISTILL + tid;
            if (j < a.k && list.ids[j] != LILY_NO_TOKEN && (!twice || speaks(list, j))) {
                const float m = fmaxf(sums[1].m, mine[e]);
                sums[1].s = sums[1].s * term(sums[1].m == NEG_INF ? reference(m) : sums[1].m, m, a.c2) + term(mine[e], m, a.c2);
                sums[1].m = m;
            }
        }
        // what the list names is not outside it
        const uint8_t* bytes = reinterpret_cast<const uint8_t*>(list.bits);
#pragma unroll
        for (uint32_t c = 0; c < PIECES; ++c) {
            const uint32_t named = bytes[piece_at(c) >> 3];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                h.v[c][j] = (named >> j & 1u) != 0u ? NEG_INF : h.v[c][j];
            }
        }
    }
#pragma unroll
    for (uint32_t c = 0; c < PIECES; ++c) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            sums[0].m = fmaxf(sums[0].m, h.v[c][j]);
        }
    }
#pragma unroll
    for (uint32_t c = 0; c < PIECES; ++c) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            sums[0].s += term(h.v[c][j], sums[0].m, a.c2);
        }
    }
    group_sums(sums, a.c2, part);
    if (tid == 0u) {
        float* to = a.records + ((uint64_t)in_launch * a.slices + slice) * 4u;
        to[0] = sums[0].m;
        to[1] = sums[0].s;
        to[2] = sums[1].m;
        to[3] = sums[1].s;
    }
}

// exp(-x) with the product's rounding put right: x may be some tens.
__device__ __forceinline__ float exp_minus(float x) {
    const float y = x * -1.4426950408889634f;
    const float rest = __builtin_fmaf(x, -1.4426950408889634f, -y) + x * -1.925963033500e-8f;   // log2(e) - f32(log2(e))
    const float e = __builtin_amdgcn_exp2f(y);
    return fabsf(y) < 126.0f ? __builtin_fmaf(e, rest * 0.69314718f, e) : e;
}

// GRAD false: the loss and stats alone, a workgroup a row.
template <bool GRAD>
__global__ void __launch_bounds__(NT_DISTILL) k_distill_finish(const DistillArgs a) {
    __shared__ SliceList list;
    __shared__ float part[DISTILL_WAVES * 4];
    __shared__ double part_d[DISTILL_WAVES][2];
    const uint32_t tid = threadIdx.x, slices = GRAD ? a.slices : 1u, slice = blockIdx.x % slices, in_launch = blockIdx.x / slices;
    const uint64_t row = (uint64_t)a.row0 + in_launch;
    const uint32_t lo = slice * DISTILL_SLICE;
    const void* z = at_row(a.logits, row, a.logits_stride, a.logits_bf16);
    Held h;
    if (GRAD) {
        hold(a, z, lo, h);
    }
    const uint32_t count = list_length(a, row);
    const float weight = a.grad_scale * (a.row_weights != nullptr ? gload(a.row_weights + row) : 1.0f);
    if (GRAD) {
        list.bits[tid] = 0u;
    }
    if (tid == 0u) {
        list.twice = 0u;
    }
    // the row's sums: outside the list (everything without `rest`), in it
    Sum out = {NEG_INF, 0.0f}, all = {NEG_INF, 0.0f};
    float log_all, log_out, inv_all, inv_out, q_out;   // logarithms and reciprocals of the sums; Q
    bool nothing;                                     // nothing above -inf outside the list
    if (a.backward == 0u) {
        Sum in = {NEG_INF, 0.0f};
        const float* from = a.records + (uint64_t)in_launch * a.slices * 4u;
        for (uint32_t q = tid & 63u; q < a.slices; q += 64u) {
            const Sum o = {gload(from + q * 4u), gload(from + q * 4u + 1u)}, i = {gload(from + q * 4u + 2u), gload(from + q * 4u + 3u)};
            const float mo = fmaxf(out.m, o.m), mi = fmaxf(in.m, i.m);
            out.s = out.s * term(out.m == NEG_INF ? reference(mo) : out.m, mo, a.c2) + o.s * term(o.m == NEG_INF ? reference(mo) : o.m, mo, a.c2);
            in.s = in.s * term(in.m == NEG_INF ? reference(mi) : in.m, mi, a.c2) + i.s * term(i.m == NEG_INF ? reference(mi) : i.m, mi, a.c2);
            out.m = mo;
            in.m = mi;
        }
        auto over_wave = [&](Sum t) {
            const float m = wave_max_dpp(t.m);
            return Sum{m, wave_sum_f(t.s * term(t.m == NEG_INF ? reference(m) : t.m, m, a.c2))};
        };
        out = over_wave(out);
        in = over_wave(in);
        const float m = fmaxf(out.m, in.m);
        all = {m, out.s * term(out.m == NEG_INF ? reference(m) : out.m, m, a.c2) + in.s * term(in.m == NEG_INF ? reference(m) : in.m, m, a.c2)};
        log_all = m == NEG_INF ? __builtin_nanf("") : logf(all.s);
        nothing = out.m == NEG_INF && out.s == 0.0f;
        log_out = nothing ? 0.0f : logf(out.s);
        inv_all = m == NEG_INF ? __builtin_nanf("") : 1.0f / all.s;
        inv_out = 1.0f / out.s;
        q_out = term(out.m == NEG_INF ? reference(m) : out.m, m, a.c2) * out.s * inv_all;
        if (slice == 0u && tid == 0u && a.stats != nullptr) {
            float* to = a.stats + row * 4u;
            to[0] = all.m;
            to[1] = log_all;
            to[2] = a.rest != 0u ? out.m : 0.0f;
            to[3] = a.rest != 0u ? log_out : 0.0f;
        }
    } else {
        const float* from = a.stats + row * 4u;
        all.m = gload(from);
        log_all = gload(from + 1);
        out.m = a.rest != 0u ? gload(from + 2) : all.m;
        log_out = a.rest != 0u ? gload(from + 3) : log_all;
        nothing = out.m == NEG_INF && log_out == 0.0f;
        inv_all = exp_minus(log_all);
        inv_out = exp_minus(log_out);
        q_out = __builtin_amdgcn_exp2f((reference(out.m) - all.m) * a.c2) * exp_minus(log_all - log_out);
    }
    // the teacher's list
    const void* values = at_row(a.values, row, a.values_stride, a.values_bf16);
    float t[ENTRIES], mine[ENTRIES];
    uint32_t id[ENTRIES];
    Sum mass[2] = {{NEG_INF, 0.0f}, {NEG_INF, 0.0f}};   // of the list; [1].m: whether any entry counts
#pragma unroll
    for (uint32_t e = 0; e < ENTRIES; ++e) {
        const uint32_t j = e * NT_DISTILL + tid;
        id[e] = j < a.k ? valid_id(a, row, count, j) : LILY_NO_TOKEN;
        t[e] = 0.0f;
        mine[e] = 0.0f;
        if (id[e] != LILY_NO_TOKEN) {
            t[e] = load1(values, j, a.values_bf16);
            mass[1].m = 0.0f;
            const bool here = id[e] >= lo && id[e] - lo < DISTILL_SLICE;
            if (a.backward == 0u) {
                mine[e] = slice == 0u || here ? gload(a.list + (uint64_t)in_launch * a.k + j) : 0.0f;
            } else if (here) {
                mine[e] = load1(z, id[e], a.logits_bf16);
            }
            if (a.probs != 0u) {
                t[e] = t[e] < 0.0f ? 0.0f : t[e];
            }
        }
        if (GRAD && j < a.k) {
            list.ids[j] = id[e];
        }
    }
    // (with `rest` a logit's probability is relative to the teacher's sum; otherwise to the list's largest)
    if (a.probs == 0u && a.rest == 0u) {
#pragma unroll
        for (uint32_t e = 0; e < ENTRIES; ++e) {
            mass[0].m = fmaxf(mass[0].m, id[e] != LILY_NO_TOKEN ? t[e] : NEG_INF);
        }
    }
    const double over_t = 1.0 / (double)a.temperature;
    const double teacher_lse = a.teacher_lse != nullptr ? (double)gload(a.teacher_lse + row) : 0.0;
    float p[ENTRIES];
#pragma unroll
    for (uint32_t e = 0; e < ENTRIES; ++e) {
        p[e] = 0.0f;
        if (id[e] != LILY_NO_TOKEN) {
            p[e] = a.probs != 0u  ? t[e]
                   : a.rest != 0u ? (float)exp((double)t[e] * over_t - teacher_lse)
                                  : term(t[e], mass[0].m, a.c2);
            mass[0].s += p[e];
        }
    }
    const float own_m = mass[0].m;
    if (a.probs != 0u || a.rest != 0u) {
        mass[0].m = 0.0f;
    }
    group_sums(mass, a.c2, part);
    const bool any = mass[1].m == 0.0f;
    const float sum = mass[0].s, top = mass[0].m;
    const bool live = any && (a.rest != 0u || sum > 0.0f || sum != sum);
    const float per = a.rest != 0u ? 1.0f : 1.0f / sum;
#pragma unroll
    for (uint32_t e = 0; e < ENTRIES; ++e) {
        if (a.probs == 0u && a.rest == 0u) {
            p[e] *= term(own_m == NEG_INF ? reference(top) : own_m, top, a.c2);
        }
        p[e] *= per;
    }
    const float left = a.rest == 0u ? 0.0f : sum < 1.0f || sum != sum ? 1.0f - sum : 0.0f;   // P
    if (!a.backward && slice == 0u && a.loss != nullptr) {
        // in 64 bits: a loss near zero is a difference of large logarithms
        double sum_d = 0.0;
        const double log_sum = log((double)sum), la = log_all != log_all ? (double)log_all : log((double)all.s);
#pragma unroll
        for (uint32_t e = 0; e < ENTRIES; ++e) {
            if (id[e] != LILY_NO_TOKEN && p[e] != 0.0f) {
                const double log_p = a.probs == 0u && a.rest == 0u ? ((double)t[e] - (double)top) * over_t - log_sum
                                     : a.probs == 0u               ? (double)t[e] * over_t - teacher_lse
                                                                   : log((double)t[e]) - (a.rest != 0u ? 0.0 : log_sum);
                sum_d += (double)p[e] * (log_p - (((double)mine[e] - (double)all.m) * over_t - la));
            }
        }
        for (int off = 32; off > 0; off >>= 1) {
            sum_d += __shfl_xor(sum_d, off);
        }
        if ((tid & 63u) == 0u) {
            part_d[tid >> 6][0] = sum_d;
        }
        __syncthreads();
        if (tid == 0u) {
            for (uint32_t q = 1; q < DISTILL_WAVES; ++q) {
                sum_d += part_d[q][0];
            }
            if (a.rest != 0u && left != 0.0f) {
                const double log_q = nothing ? -INFINITY : ((double)reference(out.m) - (double)all.m) * over_t + log((double)out.s) - la;
                sum_d += (double)left * (log((double)left) - log_q);
            }
            // (a row of -inf alone has no sum: its logarithm is no number)
            a.loss[row] = live ? (float)(sum_d * (double)a.temperature * (double)a.temperature) + (log_all != log_all ? log_all : 0.0f) : 0.0f;
        }
    }
    if (!GRAD) {
        return;
    }
    // The gradient of an id outside the list: factor * exp((z - ref) / T).
    const bool zeros = !live || weight == 0.0f;
    const float wt = weight * a.temperature * (sum != sum ? sum : 1.0f);
    float ref, factor;
    if (a.rest != 0u) {
        ref = out.m;
        factor = nothing ? (log_all != log_all ? log_all : 0.0f) : wt * (q_out - left) * inv_out;
    } else {
        ref = all.m;
        factor = wt * inv_all;
    }
    if (zeros) {
        factor = 0.0f;
    }
    void* grad = const_cast<void*>(at_row(a.grad, row, a.grad_stride, a.grad_dtype == LILY_BF16));
#pragma unroll
    for (uint32_t c = 0; c < PIECES; ++c) {
        const uint32_t i = lo + piece_at(c);
        float g[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            g[j] = zeros ? 0.0f : factor * term(h.v[c][j], ref, a.c2);
        }
        if (i + 8u <= a.vocab) {
            store8(grad, i, g, a.grad_dtype);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (i + (uint32_t)j < a.vocab) {
                    store1(grad, i + (uint32_t)j, g[j], a.grad_dtype);
                }
            }
        }
    }
    if (zeros) {
        return;
    }
    // The list's ids anew, behind the barrier that follows the stores above.
#pragma unroll
    for (uint32_t e = 0; e < ENTRIES; ++e) {
        const uint32_t j = e * NT_DISTILL + tid, off = id[e] - lo;
        if (j < a.k) {
            list.p[j] = p[e];
            if (id[e] != LILY_NO_TOKEN && id[e] >= lo && off < DISTILL_SLICE &&
                (atomicOr(&list.bits[off >> 5], 1u << (off & 31u)) >> (off & 31u) & 1u) != 0u) {
                list.twice = 1u;
            }
        }
    }
    __syncthreads();
    const bool twice = list.twice != 0u;
#pragma unroll
    for (uint32_t e = 0; e < ENTRIES; ++e) {
        const uint32_t j = e * NT_DISTILL + tid;
        if (id[e] == LILY_NO_TOKEN || id[e] < lo || id[e] - lo >= DISTILL_SLICE || (twice && !speaks(list, j))) {
            continue;
        }
        float total = p[e];
        if (twice) {
            for (uint32_t q = j + 1u; q < a.k; ++q) {
                total += list.ids[q] == id[e] ? list.p[q] : 0.0f;
            }
        }
        const float q = term(mine[e], all.m, a.c2) * inv_all;
        store1(grad, id[e], wt * (q - total), a.grad_dtype);
    }
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
    a.slices = (d.vocab + DISTILL_SLICE - 1u) / DISTILL_SLICE;
    a.k = d.k;
    a.probs = d.teacher == LILY_TEACHER_PROBS;
    a.rest = d.rest;
    a.logits_bf16 = d.logits_dtype == LILY_BF16;
    a.values_bf16 = d.values_dtype == LILY_BF16;
    a.grad_dtype = d.grad_dtype;
    a.backward = backward;
    a.temperature = d.temperature;
    a.c2 = (float)(1.4426950408889634 / (double)d.temperature);
    a.grad_scale = d.grad_scale;
    // as many rows at a time as the workspace holds
    const uint64_t each = (uint64_t)a.slices * 4u + d.k;
    const uint32_t most = backward ? d.rows : (uint32_t)std::min<uint64_t>(d.rows, ws.part_floats / each);
    for (uint64_t row = 0; row < d.rows; row += most) {
        const uint32_t rows = (uint32_t)std::min<uint64_t>(most, d.rows - row);
        a.row0 = (uint32_t)row;
        a.records = ws.part;
        a.list = ws.part + (uint64_t)rows * a.slices * 4u;
        if (!backward) {
            hipLaunchKernelGGL(k_distill_sums, dim3(rows * a.slices), dim3(NT_DISTILL), 0, stream, a);
        }
        if (d.grad_dev != nullptr) {
            hipLaunchKernelGGL(k_distill_finish<true>, dim3(rows * a.slices), dim3(NT_DISTILL), 0, stream, a);
        } else {
            hipLaunchKernelGGL(k_distill_finish<false>, dim3(rows), dim3(NT_DISTILL), 0, stream, a);
        }
    }
    return hipGetLastError();
}

}  // namespace lily
