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
// the biased ids (a bitmap of the slice in LDS, built from the row's list) each; only groups with a bit set
// look further (one 16-byte load brings the four counts).  Bound by memory.
//
// Log-probabilities need the row's sum before the first value can be written.  Rows that one workgroup each
// fill the chip with go through twice in one launch, the second time out of the caches
// (k_logits_rows<..., FORM_BOTH>); fewer rows are cut into slices, a launch for the sums and one that
// writes.
#include <hip/hip_runtime.h>

#include "device_common.h"
#include "launch.h"

namespace lily {

namespace {

constexpr int GROUP = 4;           // ids a thread takes at a time
constexpr int AHEAD = 4;           // groups of a thread in flight
constexpr uint32_t BIAS_PAIRS = 512;   // pairs of a slice kept in LDS
constexpr uint32_t LOGITS_GROUPS = 2048;      // workgroups of 256 threads that a batch is cut into: the chip holds as many
constexpr uint32_t RELAXED_FROM = 256;        // workgroups above which the slices' hand-over takes its relaxed form
constexpr uint32_t LOGITS_SLICE_MIN = 2048;   // ids
constexpr uint32_t LOGITS_ROWS_WHOLE = 256;   // rows from which on a workgroup of 1 024 threads each fills the chip
constexpr float LOG2E = 1.4426950408889634f;

enum Form {
    FORM_ADJUSTED = 0,   // written, no sums
    FORM_ADJUSTED_SUM,   // written, and summed
    FORM_SUM,            // summed only: the first launch of log-probabilities
    FORM_LOGPROBS,       // written with the sums of the launch before
    FORM_BOTH,           // summed, then written, by the one workgroup of the row
};

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
};
struct Sums {
    double s[16];
    float m[16];
    uint32_t last;
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

// One id's value, given its logit, count, and whether it is biased and admitted: the draws' arithmetic.
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
    l = allowed ? l : NEG_INF;
    l = a.temperature == 1.0f ? l : l / a.temperature;
    return l > NEG_INF ? l : NEG_INF;   // (a NaN is worth -inf)
}

// One pass over ids [lo, hi) (lo a multiple of 32) of the row.
template <int DT, class EACH, class EACH_ONE>
__device__ __forceinline__ void pass_over(const RowArgs& a, uint32_t lo, uint32_t hi, const SliceBias* sb,
                                          const uint32_t* bits, EACH&& each, EACH_ONE&& each_one) {
    const uint32_t tid = threadIdx.x, nt = blockDim.x;
    const bool pen = (a.flags & F_PEN) != 0u, masked = a.allow != nullptr, biased = a.n_bias != 0u;
    const uint32_t whole = (hi - lo) / GROUP;   // groups; the ids behind the last one follow
    for (uint32_t g0 = tid; g0 < whole; g0 += nt * AHEAD) {
        RawGroup<DT> raw[AHEAD];
        uint32_t listed[AHEAD], admitted[AHEAD], to_add[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const uint32_t id = lo + min(g0 + (uint32_t)u * nt, whole - 1u) * GROUP;
            raw[u].load(a.logits, id);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const uint32_t id = lo + min(g0 + (uint32_t)u * nt, whole - 1u) * GROUP;
            listed[u] = pen ? gload(a.touched + (id >> 5)) : 0u;
            admitted[u] = masked ? gload(a.allow + (id >> 5)) : 0xffffffffu;
            to_add[u] = biased ? bits[(id - lo) >> 5] : 0u;
        }
        u32x4 counts[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const uint32_t id = lo + min(g0 + (uint32_t)u * nt, whole - 1u) * GROUP;
            listed[u] = (listed[u] >> (id & 31u)) & 15u;
            admitted[u] = (admitted[u] >> (id & 31u)) & 15u;
            to_add[u] = (to_add[u] >> ((id - lo) & 31u)) & 15u;
            counts[u] = u32x4{0u, 0u, 0u, 0u};
            if (listed[u] != 0u) {   // (counts start at a multiple of 16 bytes)
                counts[u] = gload(reinterpret_cast<const u32x4*>(a.counts + id));
            }
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const uint32_t g = g0 + (uint32_t)u * nt;
            if (g < whole) {
                const uint32_t id = lo + g * GROUP;
                float v[GROUP];
                if ((listed[u] | to_add[u]) != 0u) {
#pragma unroll
                    for (int j = 0; j < GROUP; ++j) {
                        v[j] = adjusted(a, sb, id + (uint32_t)j, raw[u].at(j), counts[u][j], (to_add[u] >> j) & 1u,
                                        (admitted[u] >> j) & 1u);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < GROUP; ++j) {
                        v[j] = adjusted(a, sb, id + (uint32_t)j, raw[u].at(j), 0u, false, (admitted[u] >> j) & 1u);
                    }
                }
                each(id, v);
            }
        }
    }
    const uint32_t id = lo + whole * GROUP + tid;
    if (id < hi) {
        const uint32_t count = pen ? gload(a.counts + id) : 0u;
        const bool add = biased && ((bits[(id - lo) >> 5] >> ((id - lo) & 31u)) & 1u) != 0u;
        each_one(id, adjusted(a, sb, id, load_logit<DT>(a.logits, id), count, add, !masked || bit_of(a.allow, id)));
    }
}

struct LogitsLaunch {
    void* out;
    uint64_t stride;        // elements
    float* lse;             // or null
    Handed<double> part;    // [rows][slices][2] largest value, sum of exp(value - largest)
    uint32_t* ticket;       // [rows], zero between launches
    uint32_t vocab, slices, per_slice;   // per_slice: a multiple of 32
    uint32_t relaxed;
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

// The workgroup's (largest value, sum) in every thread.
__device__ __forceinline__ void merge_threads(const RowSum& l, Sums& sh, double& m_out, double& s_out) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    float m = wave_max_dpp(l.m);
    double s = l.m > NEG_INF ? (double)l.s * (double)__builtin_amdgcn_exp2f((l.m - m) * LOG2E) : 0.0;
    s = wave_sum_d(s);
    if (lane == 0u) {
        sh.m[wave] = m;
        sh.s[wave] = s;
    }
    __syncthreads();
    m = sh.m[0];
    for (uint32_t q = 1; q < waves; ++q) {
        m = fmaxf(m, sh.m[q]);
    }
    s = 0.0;
    for (uint32_t q = 0; q < waves; ++q) {
        s += sh.m[q] > NEG_INF ? sh.s[q] * (double)__builtin_amdgcn_exp2f((sh.m[q] - m) * LOG2E) : 0.0;
    }
    m_out = (double)m;
    s_out = s;
    __syncthreads();
}

// The slices' (largest value, sum) pairs of a row as one; every thread gets it (a lane a slice).
__device__ __forceinline__ void merge_slices(const Handed<double>& part, size_t first, uint32_t slices, double& m_out, double& s_out) {
    const uint32_t lane = threadIdx.x & 63u;
    double m = -__builtin_huge_val(), s = 0.0;
    if (lane < slices) {
        m = handed_load(part, (first + lane) * 2);
        s = handed_load(part, (first + lane) * 2 + 1);
    }
    const double top = wave_max_d(m);
    s = m > -__builtin_huge_val() ? s * (double)__builtin_amdgcn_exp2f((float)(m - top) * LOG2E) : 0.0;
    m_out = top;
    s_out = wave_sum_d(s);
}

template <int DT, int OT, int FORM>
__device__ __forceinline__ void logits_row(const RowArgs& a, uint32_t row_of_launch, uint32_t slice, const LogitsLaunch& q) {
    __shared__ SliceBias sb;
    __shared__ Sums sh;
    __shared__ uint32_t wave_count[16];
    uint32_t* bits = reinterpret_cast<uint32_t*>(dyn_lds);
    const uint32_t lo = slice * q.per_slice, hi = min(q.vocab, lo + q.per_slice);
    const uint32_t row = (uint32_t)a.row;   // of the output
    void* out = static_cast<char*>(q.out) + (size_t)row * q.stride * (OT == LILY_F32 ? 4u : 2u);
    if (a.n_bias != 0u) {
        list_biases(a, lo, hi, sb, bits, wave_count);
    }
    LogSum lse = {0.0f, 0.0f};
    auto write = [&](uint32_t id, const float (&v)[GROUP]) {
        if (FORM == FORM_ADJUSTED || FORM == FORM_ADJUSTED_SUM) {
            store_group<OT>(out, id, v);
        } else {
            float p[GROUP];
#pragma unroll
            for (int j = 0; j < GROUP; ++j) {
                p[j] = lse.logprob(v[j]);
            }
            store_group<OT>(out, id, p);
        }
    };
    auto write_one = [&](uint32_t id, float v) {
        store_one<OT>(out, id, FORM == FORM_ADJUSTED || FORM == FORM_ADJUSTED_SUM ? v : lse.logprob(v));
    };
    if constexpr (FORM == FORM_ADJUSTED) {
        pass_over<DT>(a, lo, hi, &sb, bits, write, write_one);
        return;
    } else {
        double m, s;
        if constexpr (FORM != FORM_LOGPROBS) {
            RowSum acc;
            acc.init();
            pass_over<DT>(
                a, lo, hi, &sb, bits,
                [&](uint32_t id, const float (&v)[GROUP]) {
                    const float top = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
                    const float ref = acc.raise(top);
#pragma unroll
                    for (int j = 0; j < GROUP; ++j) {
                        acc.add(v[j], ref);
                    }
                    if (FORM == FORM_ADJUSTED_SUM) {
                        write(id, v);
                    }
                },
                [&](uint32_t id, float v) {
                    acc.add(v, acc.raise(v));
                    if (FORM == FORM_ADJUSTED_SUM) {
                        write_one(id, v);
                    }
                });
            merge_threads(acc, sh, m, s);
            if constexpr (FORM != FORM_BOTH) {
                if (FORM == FORM_SUM || q.slices > 1u) {
                    const size_t first = (size_t)row_of_launch * q.slices;
                    if (threadIdx.x == 0u) {
                        handed_store(q.part, (first + slice) * 2, m);
                        handed_store(q.part, (first + slice) * 2 + 1, s);
                    }
                    if (FORM == FORM_SUM || !last_to_arrive(q.ticket + row_of_launch, q.slices, sh.last, q.relaxed != 0u)) {
                        return;
                    }
                    merge_slices(q.part, first, q.slices, m, s);
                }
            }
        } else {
            merge_slices(q.part, (size_t)row_of_launch * q.slices, q.slices, m, s);
        }
        lse = log_sum(m, s);
        if (q.lse != nullptr && threadIdx.x == 0u && (FORM != FORM_LOGPROBS || slice == 0u)) {
            q.lse[row] = lse.whole();
        }
        if constexpr (FORM == FORM_LOGPROBS || FORM == FORM_BOTH) {
            pass_over<DT>(a, lo, hi, &sb, bits, write, write_one);
        }
    }
}

__device__ __forceinline__ RowArgs row_of(const LILY_CONST RowArgs* p) {
    RowArgs a;
    __builtin_memcpy(&a, (const RowArgs*)p, sizeof a);
    return a;
}

template <int DT, int OT, int FORM>
__global__ void __launch_bounds__(FORM == FORM_BOTH ? 1024 : 256) k_logits_rows_table(const RowArgs* table, LogitsLaunch q) {
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
    const dim3 grid(rows * q.slices);
    const size_t lds = (size_t)q.bias_bits * 4u;
    if constexpr (FORM == FORM_BOTH) {
        hipLaunchKernelGGL((k_logits_rows_table<DT, OT, FORM>), grid, dim3(1024), lds, stream, table, q);
    } else if (few != nullptr) {
        hipLaunchKernelGGL((k_logits_rows_inline<DT, OT, FORM>), grid, dim3(256), lds, stream, *few, q);
    } else {
        hipLaunchKernelGGL((k_logits_rows_table<DT, OT, FORM>), grid, dim3(256), lds, stream, table, q);
    }
    return hipGetLastError();
}

template <int DT, int OT>
hipError_t launch_typed(hipStream_t stream, const RowArgs* table, const InlineRows* few, uint32_t rows, LogitsLaunch& q,
                        bool logprobs, bool both) {
    if (!logprobs) {
        return q.lse == nullptr ? launch_form<DT, OT, FORM_ADJUSTED>(stream, table, few, rows, q)
                                : launch_form<DT, OT, FORM_ADJUSTED_SUM>(stream, table, few, rows, q);
    }
    if (both) {
        return launch_form<DT, OT, FORM_BOTH>(stream, table, few, rows, q);
    }
    const hipError_t e = launch_form<DT, OT, FORM_SUM>(stream, table, few, rows, q);
    return e != hipSuccess ? e : launch_form<DT, OT, FORM_LOGPROBS>(stream, table, few, rows, q);
}

}  // namespace

hipError_t launch_logits_rows(hipStream_t stream, int dtype, uint32_t rows, uint32_t vocab, const RowArgs* table,
                              const InlineRows* few, const LogitsRows& w) {
    LogitsLaunch q = {};
    q.out = w.out;
    q.stride = w.stride;
    q.lse = w.lse;
    q.part = w.part;
    q.ticket = w.ticket;
    q.vocab = vocab;
    // A launch takes as many rows as the workspace has sums for.
    for (uint32_t first = 0; first < rows; first += w.max_rows) {
        const uint32_t n = min(rows - first, w.max_rows);
        const bool both = w.logprobs && few == nullptr && n >= LOGITS_ROWS_WHOLE && !(w.biased && vocab > LOGITS_SLICE_MAX);
        uint32_t slices = 1;
        if (!both) {
            slices = min((LOGITS_GROUPS + n - 1u) / n, (vocab + LOGITS_SLICE_MIN - 1u) / LOGITS_SLICE_MIN);
            slices = max(1u, min(slices, MAX_SLICES));
        }
        if (w.biased) {
            slices = max(slices, (vocab + LOGITS_SLICE_MAX - 1u) / LOGITS_SLICE_MAX);
        }
        q.per_slice = ((vocab + slices - 1u) / slices + 31u) / 32u * 32u;
        q.slices = (vocab + q.per_slice - 1u) / q.per_slice;
        q.bias_bits = w.biased ? q.per_slice / 32u : 0u;
        q.relaxed = w.handover == 2u || (w.handover == 0u && n * q.slices > RELAXED_FROM) ? 1u : 0u;
        const RowArgs* part = table != nullptr ? table + first : nullptr;
        hipError_t e;
        if (dtype == LILY_BF16) {
            e = w.out_dtype == LILY_BF16 ? launch_typed<LILY_BF16, LILY_BF16>(stream, part, few, n, q, w.logprobs, both)
                                         : launch_typed<LILY_BF16, LILY_F32>(stream, part, few, n, q, w.logprobs, both);
        } else {
            e = w.out_dtype == LILY_BF16 ? launch_typed<LILY_F32, LILY_BF16>(stream, part, few, n, q, w.logprobs, both)
                                         : launch_typed<LILY_F32, LILY_F32>(stream, part, few, n, q, w.logprobs, both);
        }
        if (e != hipSuccess) {
            return e;
        }
    }
    return hipSuccess;
}

}  // namespace lily
