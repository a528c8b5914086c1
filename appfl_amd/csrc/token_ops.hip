// token_ops.hip -- operators on a language model's (or classifier's) answers, for federations that
// exchange answers instead of weights: scoring a row of logits (log probability of the given token,
// entropy, most probable tokens), merging K clients' top lists into one teacher, and distilling from
// such lists (loss and gradient).  Softmax statistics are fp32 with the running maximum subtracted
// first; merged probabilities are fp64 (their order decides which tokens are kept).

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <math.h>
#include <stdint.h>

#include "../../include/appfl_amd.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWave = 64;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kInf = __builtin_inff();

using u16 = unsigned short;

// ---- element types ------------------------------------------------------------------------------
template <int DT> struct Elem;
template <> struct Elem<FA_LOGITS_F32> {
    using Raw = float;
    static __device__ __forceinline__ float widen(float v) { return v; }
    static __device__ __forceinline__ float narrow(float v) { return v; }
};
template <> struct Elem<FA_LOGITS_BF16> {
    using Raw = u16;
    static __device__ __forceinline__ float widen(u16 v) { return __uint_as_float(static_cast<unsigned>(v) << 16); }
    static __device__ __forceinline__ u16 narrow(float v) {      // to nearest, ties to even
        return __builtin_bit_cast(u16, static_cast<__bf16>(v));
    }
};
template <> struct Elem<FA_LOGITS_F16> {
    using Raw = u16;
    static __device__ __forceinline__ float widen(u16 v) { return static_cast<float>(__builtin_bit_cast(_Float16, v)); }
    static __device__ __forceinline__ u16 narrow(float v) {
        return __builtin_bit_cast(u16, static_cast<_Float16>(v));
    }
};

struct Rows {            // a [outer, inner, vocab] view with unit stride along the vocabulary
    int64_t inner, stride_outer, stride_inner;
    __device__ __forceinline__ int64_t offset(int64_t row) const {
        return (row / inner) * stride_outer + (row % inner) * stride_inner;
    }
};

// ---- softmax statistics: m = max x, s = sum exp((x - m) / tau), e = sum exp((x - m) / tau) (x - m) / tau
struct Stat {
    float m, s, e;
};

__device__ __forceinline__ Stat stat_empty() { return {-kInf, 0.0f, 0.0f}; }

// exp2 of the hardware: below 2^-126 it returns 0, which is nothing beside the largest term's 1
__device__ __forceinline__ float exp2_hw(float v) { return __builtin_amdgcn_exp2f(v); }

// Two parts of a row.  A part without a finite logit has s = 0 and adds nothing; a NaN stays a NaN.
__device__ __forceinline__ Stat stat_join(const Stat a, const Stat b, float scale2) {
    Stat r;
    r.m = fmaxf(a.m, b.m);
    const float ref = r.m == -kInf ? 0.0f : r.m;
    const float da = (a.m - ref) * scale2, db = (b.m - ref) * scale2;     // log2 units
    const float fa = exp2_hw(da), fb = exp2_hw(db);
    // a part too far below (its distance may be -inf) or without a finite logit adds nothing
    const float ea = a.s == 0.0f || fa == 0.0f ? 0.0f : fa * (a.e + a.s * da);
    const float eb = b.s == 0.0f || fb == 0.0f ? 0.0f : fb * (b.e + b.s * db);
    r.s = a.s * fa + b.s * fb;
    r.e = ea + eb;
    return r;
}

__device__ __forceinline__ Stat stat_wave(Stat v, float scale2) {
    for (int d = kWave / 2; d > 0; d >>= 1) {
        Stat o;
        o.m = __shfl_xor(v.m, d);
        o.s = __shfl_xor(v.s, d);
        o.e = __shfl_xor(v.e, d);
        v = stat_join(v, o, scale2);
    }
    return v;
}

template <int THREADS>
__device__ __forceinline__ Stat stat_block(Stat v, float scale2, Stat* lds) {
    v = stat_wave(v, scale2);
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    Stat r = lds[0];
    for (int i = 1; i < THREADS / kWave; ++i) r = stat_join(r, lds[i], scale2);
    __syncthreads();
    return r;
}

// e is kept in log2 units: entropy = log s - e ln 2 / s
constexpr float kLn2 = 0.69314718055994530942f;

template <int DT>
__device__ __forceinline__ Stat row_stat(const typename Elem<DT>::Raw* x, int vocab, float scale2, Stat* lds) {
    Stat st = stat_empty();
    for (int i = threadIdx.x; i < vocab; i += kThreads) {
        const float v = Elem<DT>::widen(x[i]);
        const Stat one = {v, v == -kInf ? 0.0f : (v != v ? v : 1.0f), 0.0f};
        st = stat_join(st, one, scale2);
    }
    return stat_block<kThreads>(st, scale2, lds);
}

// ---- order of logits: by value, ties to the lowest index, NaN first; -0 and +0 are equal ----------
__device__ __forceinline__ uint64_t order_key(float v, unsigned index) {
    const unsigned b = __float_as_uint(v + 0.0f);
    unsigned o = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
    if (v != v) o = 0xfffffffeu;
    return (static_cast<uint64_t>(o) << 32) | (0xffffffffu - index);
}

__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
    for (int d = kWave / 2; d > 0; d >>= 1) {
        const uint64_t o = __shfl_xor(static_cast<unsigned long long>(v), d);
        v = o > v ? o : v;
    }
    return v;
}

__device__ __forceinline__ uint64_t block_max_u64(uint64_t v, uint64_t* lds) {
    v = wave_max_u64(v);
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    uint64_t r = lds[0];
    for (int i = 1; i < kThreads / kWave; ++i) r = lds[i] > r ? lds[i] : r;
    __syncthreads();
    return r;
}

struct ScoreArgs {
    const void* x;
    Rows rows;
    int vocab, top;
    const int64_t* targets;
    int64_t ignore_index;
    float *logprob, *entropy, *lse, *top_logprobs;
    int32_t* top_ids;
};

template <int DT>
__global__ __launch_bounds__(kThreads) void token_scores_kernel(const ScoreArgs a) {
    using E = Elem<DT>;
    __shared__ Stat lds[kThreads / kWave];
    __shared__ uint64_t best[kThreads / kWave];
    const int64_t row = blockIdx.x;
    const typename E::Raw* x = static_cast<const typename E::Raw*>(a.x) + a.rows.offset(row);
    const Stat st = row_stat<DT>(x, a.vocab, kLog2e, lds);
    const float log_s = logf(st.s);
    if (threadIdx.x == 0) {
        a.lse[row] = st.m + log_s;
        a.entropy[row] = st.s == 0.0f ? 0.0f : log_s - st.e * kLn2 / st.s;
        if (a.targets) {
            const int64_t t = a.targets[row];
            float lp = 0.0f;
            if (t != a.ignore_index) {
                lp = __builtin_nanf("");
                if (t >= 0 && t < a.vocab) {
                    const float v = E::widen(x[t]);
                    lp = v == -kInf && !(st.s != st.s) ? -kInf : (v - st.m) - log_s;
                }
            }
            a.logprob[row] = lp;
        }
    }
    uint64_t prev = ~0ull;
    for (int j = 0; j < a.top; ++j) {
        uint64_t mine = 0;
        for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
            const uint64_t key = order_key(E::widen(x[i]), i);
            if (key < prev && key > mine) mine = key;
        }
        prev = block_max_u64(mine, best);
        if (threadIdx.x == 0) {
            const unsigned id = 0xffffffffu - static_cast<unsigned>(prev);
            const float v = E::widen(x[id]);
            a.top_ids[row * a.top + j] = static_cast<int32_t>(id);
            a.top_logprobs[row * a.top + j] = v == -kInf && !(st.s != st.s) ? -kInf : (v - st.m) - log_s;
        }
    }
}

// ---- distillation ---------------------------------------------------------------------------------
struct TeacherArgs {
    const int32_t* ids;
    const float* lp;
    int64_t id_stride, lp_stride;
    int k;
    float inv_tau, tau;
    const float* row_weight;
};

struct DistillArgs {
    const void* x;
    Rows rows;
    int vocab;
    TeacherArgs t;
    float* loss;
    float* stat;                 // (m, log s) per row
    const float* stat_in;
    const float* row_grad;
    void* grad;
    Rows grad_rows;
};

// One row's teacher, one entry per thread: t = softmax over the entries of lp / tau.
struct Entry {
    int id;          // -1: no entry
    float t, log_t;
    bool empty;      // the row has no entry with a probability
    bool bad;        // an entry names a token outside the vocabulary
};

__device__ __forceinline__ float block_max_f(float v, float* lds) {
    for (int d = kWave / 2; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    float r = lds[0];
    for (int i = 1; i < kThreads / kWave; ++i) r = fmaxf(r, lds[i]);
    __syncthreads();
    return r;
}

__device__ __forceinline__ float block_sum_f(float v, float* lds) {
    for (int d = kWave / 2; d > 0; d >>= 1) v += __shfl_xor(v, d);
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    float r = lds[0];
    for (int i = 1; i < kThreads / kWave; ++i) r += lds[i];
    __syncthreads();
    return r;
}

__device__ __forceinline__ Entry teacher_entry(const TeacherArgs& t, int64_t row, int vocab, float* lds) {
    Entry e = {-1, 0.0f, 0.0f, false, false};
    float lp = -kInf;
    if (static_cast<int>(threadIdx.x) < t.k) {
        e.id = t.ids[row * t.id_stride + threadIdx.x];
        if (e.id >= 0) lp = t.lp[row * t.lp_stride + threadIdx.x];
    }
    const bool bad = e.id >= vocab;
    const float nan = block_sum_f(lp != lp || bad ? 1.0f : 0.0f, lds);
    const float peak = block_max_f(lp, lds);
    e.empty = peak == -kInf && nan == 0.0f;
    e.bad = nan != 0.0f || peak == kInf;
    const float d = e.empty || lp == -kInf ? -kInf : (lp - peak) * t.inv_tau;
    const float u = exp2_hw(d * kLog2e);
    const float z = block_sum_f(u, lds);
    e.t = e.empty ? 0.0f : u / z;
    e.log_t = d - logf(z);
    return e;
}

template <int DT>
__device__ __forceinline__ void row_loss(const DistillArgs& a, int64_t row, const Entry& e, float xv, const Stat& st,
                                         float weight, float* lds) {
    const float log_s = logf(st.s);
    float term = 0.0f;
    if (e.t > 0.0f) {
        const float log_q = xv == -kInf ? -kInf : (xv - st.m) * a.t.inv_tau - log_s;
        term = e.t * (e.log_t - log_q);
    }
    float loss = block_sum_f(term, lds) * (a.t.tau * a.t.tau) * weight;
    if (e.bad || st.s != st.s) loss = __builtin_nanf("");
    if (threadIdx.x == 0) a.loss[row] = loss;
}

template <int DT>
__device__ __forceinline__ void row_grad(const DistillArgs& a, int64_t row, const typename Elem<DT>::Raw* x,
                                         const Entry& e, float xv, float m, float log_s, float c, float* vals,
                                         int* ids) {
    using E = Elem<DT>;
    typename E::Raw* g = static_cast<typename E::Raw*>(a.grad) + a.grad_rows.offset(row);
    const float ref = m == -kInf ? 0.0f : m;
    const float shift = log_s == -kInf ? 0.0f : log_s * kLog2e;
    const float scale2 = a.t.inv_tau * kLog2e;
    for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
        const float q = exp2_hw((E::widen(x[i]) - ref) * scale2 - shift);
        g[i] = E::narrow(c * q);
    }
    ids[threadIdx.x] = e.id;
    vals[threadIdx.x] = e.t;
    __syncthreads();
    if (e.id >= 0 && e.id < a.vocab) {
        bool first = true;
        float t = 0.0f;
        for (int j = 0; j < a.t.k; ++j)
            if (ids[j] == e.id) {
                t += vals[j];
                if (j < static_cast<int>(threadIdx.x)) first = false;
            }
        const float q = exp2_hw((xv - ref) * scale2 - shift);
        if (first) g[e.id] = E::narrow(c * (q - t));
    }
}

template <int DT>
__device__ __forceinline__ void fill_grad(const DistillArgs& a, int64_t row, float v) {
    typename Elem<DT>::Raw* g = static_cast<typename Elem<DT>::Raw*>(a.grad) + a.grad_rows.offset(row);
    for (int i = threadIdx.x; i < a.vocab; i += kThreads) g[i] = Elem<DT>::narrow(v);
}

template <int DT, bool LOSS, bool GRAD>
__global__ __launch_bounds__(kThreads) void distill_kernel(const DistillArgs a) {
    using E = Elem<DT>;
    __shared__ Stat lds[kThreads / kWave];
    __shared__ float red[kThreads / kWave];
    __shared__ float vals[kThreads];
    __shared__ int ids[kThreads];
    const int64_t row = blockIdx.x;
    const typename E::Raw* x = static_cast<const typename E::Raw*>(a.x) + a.rows.offset(row);
    const float weight = a.t.row_weight ? a.t.row_weight[row] : 1.0f;
    const Entry e = teacher_entry(a.t, row, a.vocab, red);
    const float c = GRAD ? weight * a.t.tau * (a.row_grad ? a.row_grad[row] : 1.0f) : 0.0f;
    if (weight == 0.0f || e.empty) {
        if (LOSS && threadIdx.x == 0) {
            a.loss[row] = 0.0f;
            if (a.stat) a.stat[2 * row] = a.stat[2 * row + 1] = 0.0f;
        }
        if (GRAD) fill_grad<DT>(a, row, 0.0f);
        return;
    }
    const float xv = e.id >= 0 && e.id < a.vocab ? E::widen(x[e.id]) : -kInf;
    float m, log_s;
    if (LOSS) {
        const Stat st = row_stat<DT>(x, a.vocab, a.t.inv_tau * kLog2e, lds);
        row_loss<DT>(a, row, e, xv, st, weight, red);
        m = st.m;
        log_s = logf(st.s);
        if (a.stat && threadIdx.x == 0) {
            a.stat[2 * row] = m;
            a.stat[2 * row + 1] = log_s;
        }
    } else {
        m = a.stat_in[2 * row];
        log_s = a.stat_in[2 * row + 1];
    }
    if (GRAD) {
        if (c == 0.0f || e.bad) fill_grad<DT>(a, row, e.bad ? __builtin_nanf("") : 0.0f);
        else row_grad<DT>(a, row, x, e, xv, m, log_s, c, vals, ids);
    }
}

// ---- merging the clients' lists -------------------------------------------------------------------
struct MergeArgs {
    const int32_t* ids;
    const float* lp;
    int64_t id_client, id_row, lp_client, lp_row;
    const float* unit;
    int64_t unit_client, unit_row;
    int K, k, top, n2;           // n2: K * k rounded up to a power of two
    int32_t* out_ids;
    float* out_lp;
    double w[FA_MERGE_CLIENTS];
};

__global__ __launch_bounds__(kThreads) void merge_tops_kernel(const MergeArgs a) {
    extern __shared__ uint64_t dyn[];
    __shared__ int answered[FA_MERGE_CLIENTS];
    __shared__ uint64_t red[kThreads / kWave];
    uint64_t* key = dyn;                                   // (id, position), position in client order
    double* p = reinterpret_cast<double*>(dyn + a.n2);     // by position
    const int64_t row = blockIdx.x;
    const int n = a.K * a.k;
    for (int c = threadIdx.x; c < FA_MERGE_CLIENTS; c += kThreads) answered[c] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < a.n2; i += kThreads) {
        uint64_t kk = ~0ull;
        double v = -1.0;
        if (i < n) {
            const int c = i / a.k, j = i - c * a.k;
            const float u = a.unit ? a.unit[c * a.unit_client + row * a.unit_row] : 1.0f;
            const double share = a.w[c] * static_cast<double>(u);
            const int id = a.ids[c * a.id_client + row * a.id_row + j];
            if (id >= 0 && share > 0.0) {
                v = share * exp(static_cast<double>(a.lp[c * a.lp_client + row * a.lp_row + j]));
                if (v != v) v = __builtin_nan("");
                kk = (static_cast<uint64_t>(static_cast<unsigned>(id)) << 32) | static_cast<unsigned>(i);
                answered[c] = 1;
            }
        }
        key[i] = kk;
        p[i] = v;
    }
    for (int size = 2; size <= a.n2; size <<= 1)
        for (int d = size >> 1; d > 0; d >>= 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < a.n2 / 2; i += kThreads) {
                const int lo = 2 * i - (i & (d - 1)), hi = lo + d;
                const bool up = (lo & size) == 0;
                const uint64_t x = key[lo], y = key[hi];
                if ((x > y) == up) {
                    key[lo] = y;
                    key[hi] = x;
                }
            }
        }
    __syncthreads();
    double total = 0.0;
    for (int c = 0; c < a.K; ++c)
        if (answered[c]) total += a.w[c] * static_cast<double>(a.unit ? a.unit[c * a.unit_client + row * a.unit_row] : 1.0f);
    for (int i = threadIdx.x; i < a.n2; i += kThreads) {
        if (key[i] == ~0ull) continue;
        const unsigned id = static_cast<unsigned>(key[i] >> 32);
        if (i && static_cast<unsigned>(key[i - 1] >> 32) == id) continue;
        double s = 0.0;                                    // a run's slots belong to its first entry
        for (int j = i; j < a.n2 && static_cast<unsigned>(key[j] >> 32) == id; ++j) {
            const unsigned pos = static_cast<unsigned>(key[j]);
            s += p[pos];
            p[pos] = -1.0;
        }
        p[static_cast<unsigned>(key[i])] = s;
    }
    __syncthreads();
    for (int t = 0; t < a.top; ++t) {
        // largest value, then (among equals) the first place in the order of ids
        int64_t best = -1;
        int at = 0;
        for (int i = threadIdx.x; i < a.n2; i += kThreads) {
            if (key[i] == ~0ull) continue;
            const double v = p[static_cast<unsigned>(key[i])];
            const int64_t b = v != v ? 0x7ff8000000000000ll : __double_as_longlong(v);
            if (b > best) {
                best = b;
                at = i;
            }
        }
        const uint64_t v1 = best < 0 ? 0 : static_cast<uint64_t>(best) + 1;
        uint64_t top = wave_max_u64(v1);
        if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = top;
        __syncthreads();
        top = red[0];
        for (int i = 1; i < kThreads / kWave; ++i) top = red[i] > top ? red[i] : top;
        __syncthreads();
        uint64_t place = v1 == top && top ? ~static_cast<uint64_t>(at) : 0;
        place = wave_max_u64(place);
        if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = place;
        __syncthreads();
        place = red[0];
        for (int i = 1; i < kThreads / kWave; ++i) place = red[i] > place ? red[i] : place;
        if (threadIdx.x == 0) {
            int32_t id = -1;
            float lp = -kInf;
            if (top) {
                const unsigned i = static_cast<unsigned>(~place);
                const unsigned pos = static_cast<unsigned>(key[i]);
                id = static_cast<int32_t>(key[i] >> 32);
                lp = static_cast<float>(log(p[pos] / total));
                p[pos] = -1.0;
            }
            a.out_ids[row * a.top + t] = id;
            a.out_lp[row * a.top + t] = lp;
        }
        __syncthreads();
    }
}

// ---- host side ------------------------------------------------------------------------------------
int hip_code(hipError_t e) { return e == hipSuccess ? FA_OK : FA_ERR_HIP - static_cast<int>(e); }

int elem_size(int dtype) { return dtype == FA_LOGITS_F32 ? 4 : 2; }

bool aligned_to(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

int check_logits(const fa_logits* x) {
    if (!x || x->vocab <= 0 || x->outer < 0 || x->inner < 0) return FA_ERR_INVALID;
    if (x->dtype != FA_LOGITS_F32 && x->dtype != FA_LOGITS_BF16 && x->dtype != FA_LOGITS_F16) return FA_ERR_INVALID;
    if (x->stride_outer < 0 || x->stride_inner < 0) return FA_ERR_INVALID;
    if (x->inner && x->outer > INT32_MAX / x->inner) return FA_ERR_TOO_LARGE;
    if (x->outer * x->inner && !x->data) return FA_ERR_INVALID;
    if (!aligned_to(x->data, elem_size(x->dtype))) return FA_ERR_ALIGN;
    return FA_OK;
}

int check_teacher(const fa_teacher* t, int64_t rows) {
    if (!t || t->k < 1 || t->k > FA_TOP_MAX) return FA_ERR_INVALID;
    if (rows && (!t->ids || !t->logprobs)) return FA_ERR_INVALID;
    if (t->id_stride < 0 || t->lp_stride < 0) return FA_ERR_INVALID;
    if (!(t->temperature > 0.0) || !(t->temperature <= 1e30) || !(t->temperature >= 1e-30)) return FA_ERR_INVALID;
    return FA_OK;
}

Rows rows_of(const fa_logits* x) { return {x->inner, x->stride_outer, x->stride_inner}; }

DistillArgs distill_args(const fa_logits* x, const fa_teacher* t) {
    DistillArgs a = {};
    a.x = x->data;
    a.rows = rows_of(x);
    a.vocab = x->vocab;
    a.t = {t->ids, t->logprobs, t->id_stride, t->lp_stride, t->k, static_cast<float>(1.0 / t->temperature),
           static_cast<float>(t->temperature), t->row_weight};
    return a;
}

template <bool LOSS, bool GRAD>
int launch_distill(const fa_logits* x, const DistillArgs& a, hipStream_t st) {
    const unsigned rows = static_cast<unsigned>(x->outer * x->inner);
    switch (x->dtype) {
        case FA_LOGITS_F32:
            hipLaunchKernelGGL((distill_kernel<FA_LOGITS_F32, LOSS, GRAD>), dim3(rows), dim3(kThreads), 0, st, a);
            break;
        case FA_LOGITS_BF16:
            hipLaunchKernelGGL((distill_kernel<FA_LOGITS_BF16, LOSS, GRAD>), dim3(rows), dim3(kThreads), 0, st, a);
            break;
        default:
            hipLaunchKernelGGL((distill_kernel<FA_LOGITS_F16, LOSS, GRAD>), dim3(rows), dim3(kThreads), 0, st, a);
    }
    return hip_code(hipGetLastError());
}

hipStream_t as_stream(fa_stream_t s) { return reinterpret_cast<hipStream_t>(s); }

}  // namespace

extern "C" {

int fa_token_workspace(const fa_logits* x, int top, size_t* bytes) {
    const int rc = check_logits(x);
    if (rc != FA_OK) return rc;
    if (!bytes || top < 0 || top > FA_TOP_MAX) return FA_ERR_INVALID;
    *bytes = 0;
    return FA_OK;
}

int fa_token_scores(const fa_logits* x, const int64_t* targets, int64_t ignore_index, int top, float* logprob,
                    float* entropy, float* lse, int32_t* top_ids, float* top_logprobs, void* ws, fa_stream_t stream) {
    const int rc = check_logits(x);
    if (rc != FA_OK) return rc;
    if (top < 0 || top > FA_TOP_MAX || top > x->vocab) return FA_ERR_INVALID;
    const int64_t rows = x->outer * x->inner;
    if (rows == 0) return FA_OK;
    if (!entropy || !lse || (targets && !logprob) || (top && (!top_ids || !top_logprobs))) return FA_ERR_INVALID;
    (void)ws;
    const ScoreArgs a = {x->data, rows_of(x), x->vocab, top, targets, ignore_index, logprob, entropy, lse,
                         top_logprobs, top_ids};
    const dim3 grid(static_cast<unsigned>(rows));
    switch (x->dtype) {
        case FA_LOGITS_F32:
            hipLaunchKernelGGL(token_scores_kernel<FA_LOGITS_F32>, grid, dim3(kThreads), 0, as_stream(stream), a);
            break;
        case FA_LOGITS_BF16:
            hipLaunchKernelGGL(token_scores_kernel<FA_LOGITS_BF16>, grid, dim3(kThreads), 0, as_stream(stream), a);
            break;
        default:
            hipLaunchKernelGGL(token_scores_kernel<FA_LOGITS_F16>, grid, dim3(kThreads), 0, as_stream(stream), a);
    }
    return hip_code(hipGetLastError());
}

int fa_distill_loss(const fa_logits* x, const fa_teacher* t, float* loss, float* stat, void* ws, fa_stream_t stream) {
    int rc = check_logits(x);
    if (rc == FA_OK) rc = check_teacher(t, x->outer * x->inner);
    if (rc != FA_OK) return rc;
    if (x->outer * x->inner == 0) return FA_OK;
    if (!loss || !stat) return FA_ERR_INVALID;
    (void)ws;
    DistillArgs a = distill_args(x, t);
    a.loss = loss;
    a.stat = stat;
    return launch_distill<true, false>(x, a, as_stream(stream));
}

int fa_distill_grad(const fa_logits* x, const fa_teacher* t, const float* stat, const float* row_grad, void* grad,
                    int64_t grad_stride_outer, int64_t grad_stride_inner, fa_stream_t stream) {
    int rc = check_logits(x);
    if (rc == FA_OK) rc = check_teacher(t, x->outer * x->inner);
    if (rc != FA_OK) return rc;
    if (x->outer * x->inner == 0) return FA_OK;
    if (!stat || !grad || grad_stride_outer < 0 || grad_stride_inner < 0) return FA_ERR_INVALID;
    if (!aligned_to(grad, elem_size(x->dtype))) return FA_ERR_ALIGN;
    DistillArgs a = distill_args(x, t);
    a.stat_in = stat;
    a.row_grad = row_grad;
    a.grad = grad;
    a.grad_rows = {x->inner, grad_stride_outer, grad_stride_inner};
    return launch_distill<false, true>(x, a, as_stream(stream));
}

int fa_distill_loss_grad(const fa_logits* x, const fa_teacher* t, float* loss, void* grad, int64_t grad_stride_outer,
                         int64_t grad_stride_inner, void* ws, fa_stream_t stream) {
    int rc = check_logits(x);
    if (rc == FA_OK) rc = check_teacher(t, x->outer * x->inner);
    if (rc != FA_OK) return rc;
    if (x->outer * x->inner == 0) return FA_OK;
    if (!loss || !grad || grad_stride_outer < 0 || grad_stride_inner < 0) return FA_ERR_INVALID;
    if (!aligned_to(grad, elem_size(x->dtype))) return FA_ERR_ALIGN;
    (void)ws;
    DistillArgs a = distill_args(x, t);
    a.loss = loss;
    a.grad = grad;
    a.grad_rows = {x->inner, grad_stride_outer, grad_stride_inner};
    return launch_distill<true, true>(x, a, as_stream(stream));
}

int fa_merge_tops(const fa_tops* in, const double* w, int K, int64_t rows, int top, int32_t* out_ids,
                  float* out_logprobs, fa_stream_t stream) {
    if (!in || !w || K < 1 || K > FA_MERGE_CLIENTS || rows < 0 || in->k < 1 || in->k > FA_TOP_MAX) return FA_ERR_INVALID;
    if (static_cast<int64_t>(K) * in->k > FA_MERGE_ENTRIES || rows > INT32_MAX) return FA_ERR_TOO_LARGE;
    if (top < 1 || top > K * in->k) return FA_ERR_INVALID;
    if (in->id_client < 0 || in->id_row < 0 || in->lp_client < 0 || in->lp_row < 0 || in->unit_client < 0 ||
        in->unit_row < 0)
        return FA_ERR_INVALID;
    for (int c = 0; c < K; ++c)
        if (!(w[c] >= 0.0) || !(w[c] < HUGE_VAL)) return FA_ERR_INVALID;
    if (rows == 0) return FA_OK;
    if (!in->ids || !in->logprobs || !out_ids || !out_logprobs) return FA_ERR_INVALID;
    MergeArgs a = {};
    a.ids = in->ids;
    a.lp = in->logprobs;
    a.id_client = in->id_client;
    a.id_row = in->id_row;
    a.lp_client = in->lp_client;
    a.lp_row = in->lp_row;
    a.unit = in->token_weight;
    a.unit_client = in->unit_client;
    a.unit_row = in->unit_row;
    a.K = K;
    a.k = in->k;
    a.top = top;
    a.n2 = 1;
    while (a.n2 < K * in->k) a.n2 *= 2;
    a.out_ids = out_ids;
    a.out_lp = out_logprobs;
    for (int c = 0; c < K; ++c) a.w[c] = w[c];
    const unsigned lds = static_cast<unsigned>(a.n2) * 16;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(merge_tops_kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, FA_MERGE_ENTRIES * 16);
    if (e != hipSuccess) return hip_code(e);
    hipLaunchKernelGGL(merge_tops_kernel, dim3(static_cast<unsigned>(rows)), dim3(kThreads), lds, as_stream(stream), a);
    return hip_code(hipGetLastError());
}

}  // extern "C"
