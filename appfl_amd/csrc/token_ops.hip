// token_ops.hip -- operators on a language model's (or classifier's) answers, for federations that
// exchange answers instead of weights: scoring a row of logits (log probability of the given token,
// entropy, most probable tokens), merging K clients' top lists into one teacher, and distilling from
// such lists (loss and gradient).
//
// Softmax sums are fp32 (below), lists are ranked by whole keys, merged probabilities are fp64 terms
// added as 64-bit whole numbers (their order decides which tokens are kept).  Nothing is rounded to 16
// bits but a gradient's elements, once.  A block takes a row, and few long rows of a gradient, or of loss
// and gradient in one call, are cut in parts (launch_grad, launch_step; the latter with a workspace of the
// call's own).  Blocks of one launch share nothing and no float is added atomically, so results are the
// same in every run.
//
// What bounds them (one MI355X): scores and the gradient alone move 5.0-6.9 TB/s of their bytes (8192 x
// 128000 bf16: lists of 8 351 us, sums alone 322; a gradient 855 us), loss and gradient in one call
// 4.5-4.9 TB/s counting the logits once (855-925 us); merges are bound by instructions and LDS latency.

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <math.h>
#include <stdint.h>

#include "../../include/appfl_amd.h"

namespace {

constexpr int kWave = 64;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
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
    __device__ __forceinline__ int64_t offset(int64_t row) const {       // rows and inner are below 2^31
        const unsigned r = static_cast<unsigned>(row), n = static_cast<unsigned>(inner), o = r / n;
        return o * stride_outer + (r - o * n) * stride_inner;
    }
};

template <int N>
__device__ __forceinline__ float max_of(const float (&v)[N]) {
    float m = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, v[i]);
    return m;
}

// 16 bytes of a row, and the rest of it: `head` elements before the first 16-byte boundary, `nvec`
// vectors, `tail` elements behind the last one.
struct Span {
    int head, nvec, tail;
};

template <int DT>
struct Vec {
    using Raw = typename Elem<DT>::Raw;
    static constexpr int N = 16 / sizeof(Raw);
    // what fills the lanes past the end of a row
    static constexpr unsigned kFill = DT == FA_LOGITS_F32 ? 0xff800000u : DT == FA_LOGITS_BF16 ? 0xff80ff80u : 0xfc00fc00u;

    static __device__ __forceinline__ Span span(const Raw* x, int vocab) {
        const unsigned off = static_cast<unsigned>(reinterpret_cast<uintptr_t>(x)) % 16 / sizeof(Raw);
        Span s;
        s.head = off ? N - static_cast<int>(off) : 0;
        if (s.head > vocab) s.head = vocab;
        s.nvec = (vocab - s.head) / N;
        s.tail = vocab - s.head - s.nvec * N;
        return s;
    }
    static __device__ __forceinline__ uint4 fill() { return {kFill, kFill, kFill, kFill}; }
    static __device__ __forceinline__ void widen(const uint4& r, float (&v)[N]) {
        const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == FA_LOGITS_F32) {
                v[i] = __uint_as_float(w[i]);
            } else if constexpr (DT == FA_LOGITS_BF16) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            } else {
                v[2 * i] = Elem<DT>::widen(static_cast<u16>(w[i]));
                v[2 * i + 1] = Elem<DT>::widen(static_cast<u16>(w[i] >> 16));
            }
        }
    }
    // The largest element; for float16 by pairs, so that the conversion is left to the multiply-add.
    static __device__ __forceinline__ float peak(const uint4& r, const float (&v)[N]) {
        if constexpr (DT == FA_LOGITS_F16) {
            typedef _Float16 h2 __attribute__((ext_vector_type(2)));
            const h2 m = __builtin_elementwise_max(
                __builtin_elementwise_max(__builtin_bit_cast(h2, r.x), __builtin_bit_cast(h2, r.y)),
                __builtin_elementwise_max(__builtin_bit_cast(h2, r.z), __builtin_bit_cast(h2, r.w)));
            const _Float16 lo = m.x, hi = m.y;
            return fmaxf(static_cast<float>(lo), static_cast<float>(hi));
        } else {
            return max_of(v);
        }
    }
    // The same for a value that was widened before: costs less than the registers to keep it.
    static __device__ __forceinline__ void widen_again(uint4 r, float (&v)[N]) {
        asm volatile("" : "+v"(r.x), "+v"(r.y), "+v"(r.z), "+v"(r.w));
        widen(r, v);
    }
    static __device__ __forceinline__ uint4 narrow(const float (&v)[N]) {
        unsigned w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == FA_LOGITS_F32)
                w[i] = __float_as_uint(v[i]);
            else
                w[i] = Elem<DT>::narrow(v[2 * i]) | static_cast<unsigned>(Elem<DT>::narrow(v[2 * i + 1])) << 16;
        }
        return {w[0], w[1], w[2], w[3]};
    }
};

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// A row that is read once: past the caches.
__device__ __forceinline__ uint4 load_once(const uint4* p) {
    const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
    return {v.x, v.y, v.z, v.w};
}

__device__ __forceinline__ void store_once(uint4* p, const uint4& r) {
    const u32x4 v = {r.x, r.y, r.z, r.w};
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(p));
}

// ---- softmax statistics ---------------------------------------------------------------------------
// With k = log2(e) / T every term is 2^(x k - R), R a whole number near the largest x k: the
// multiply-add rounds once, relative to its small result, rescaling by a power of two is exact, and
// the rounding of k is a change of T by 2^-25 that all of a row's terms share.
//   s = sum 2^(x k - R),   e = sum 2^(x k - R) (x k - R)   (entropy = (log2 s - e / s) / k)
// R is raised only when a value passes it by more than 2^kSlack: terms are then at most that large,
// which fp32 does not mind.
// R stays within +-kFar, so a distance is finite.  From |x k| = 2^24 on R is a multiple of 2 and more:
// where all of a lane's values (or of a row's) lie that far out, behind a mask of -1e10 or on a row of
// padding, its terms are 2^r, r up to half of R's step, and s or e may be inf.  Beside an ordinary
// value such a lane's sums are dropped (acc_raise).  A row that keeps them holds |r| <= 64 below
// |x k| = 2^31 (x = 1.5e9 at T = 1); a sum outside 2^+-80, a row beyond +-kFar (the type's lowest value,
// infinities) and a NaN make acc_good refuse, and the row is taken again by slow_stat, which subtracts
// the maximum before it scales.
constexpr float kFar = 1e38f;

struct Acc {
    float R, s, e;
};

__device__ __forceinline__ Acc acc_empty() { return {-kFar, 0.0f, 0.0f}; }

// exp2 of the hardware: below 2^-126 it returns 0, which is nothing beside the largest term
__device__ __forceinline__ float exp2_hw(float v) { return __builtin_amdgcn_exp2f(v); }

// Sums below 2^-126 of the new reference are dropped whole: scaled, an infinite one would be a NaN.  A
// NaN stays; a lane with a logit of +inf holds R = kFar, above which nothing is raised.
template <bool ENT>
__device__ __forceinline__ void acc_raise(Acc& a, float R) {
    const float d = a.R - R, f = exp2_hw(d);
    const bool gone = f == 0.0f && a.s == a.s;
    if (ENT) a.e = gone ? 0.0f : f * (a.e + a.s * d);
    a.s = gone ? 0.0f : a.s * f;
    a.R = R;
}

template <bool ENT>
__device__ __forceinline__ void acc_one(Acc& a, float v, float k) {
    const float y = fmaf(v, k, -a.R);
    const float t = exp2_hw(y);
    a.s += t;
    if (ENT) a.e = fmaf(t, fmaxf(y, -200.0f), a.e);       // 0 * -inf; a NaN stays in t
}

constexpr float kSlack = 8.0f;

// N terms whose largest is `top`
template <bool ENT, int N>
__device__ __forceinline__ void acc_add(Acc& a, const float (&v)[N], float top, float k) {
    const float y = top * k;
    if (__any(y > a.R + kSlack)) acc_raise<ENT>(a, fmaxf(a.R, fminf(rintf(y), kFar)));
#pragma unroll
    for (int i = 0; i < N; ++i) acc_one<ENT>(a, v[i], k);
}

template <bool ENT>
__device__ __forceinline__ Acc acc_join(Acc a, Acc b) {
    const bool up = a.R >= b.R;                    // never NaN
    const Acc hi = up ? a : b;
    Acc lo = up ? b : a;
    acc_raise<ENT>(lo, hi.R);
    return {hi.R, hi.s + lo.s, hi.e + lo.e};
}

template <bool ENT>
__device__ __forceinline__ Acc acc_wave(Acc v) {
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) {
        Acc o;
        o.R = __shfl_xor(v.R, d);
        o.s = __shfl_xor(v.s, d);
        o.e = ENT ? __shfl_xor(v.e, d) : 0.0f;
        v = acc_join<ENT>(v, o);
    }
    return v;
}

// Ends with every thread holding the row's sums; one barrier, `lds` is not used again in the row.
template <bool ENT, int THREADS>
__device__ __forceinline__ Acc acc_block(Acc v, Acc* lds) {
    v = acc_wave<ENT>(v);
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    if constexpr (THREADS / kWave > 4) {           // the waves' sums in lanes, joined as lanes are
        Acc r = lds[threadIdx.x % (THREADS / kWave)];
#pragma unroll
        for (int d = THREADS / kWave / 2; d > 0; d >>= 1) {
            Acc o;
            o.R = __shfl_xor(r.R, d);
            o.s = __shfl_xor(r.s, d);
            o.e = ENT ? __shfl_xor(r.e, d) : 0.0f;
            r = acc_join<ENT>(r, o);
        }
        return r;
    } else {
        Acc r = lds[0];
#pragma unroll
        for (int i = 1; i < THREADS / kWave; ++i) r = acc_join<ENT>(r, lds[i]);
        return r;
    }
}

// What a row's softmax is afterwards.  slow: in terms of m and log s (natural, of (x - m) / T).
struct RowStat {
    float R, s, m, log_s, entropy;
    bool slow;
};

template <int THREADS>
__device__ float block_max_f(float v, float* lds) {
    for (int d = kWave / 2; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    __syncthreads();
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    float r = lds[0];
    for (int i = 1; i < THREADS / kWave; ++i) r = fmaxf(r, lds[i]);
    return r;
}

template <int THREADS>
__device__ float block_sum_f(float v, float* lds) {
    for (int d = kWave / 2; d > 0; d >>= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    float r = lds[0];
    for (int i = 1; i < THREADS / kWave; ++i) r += lds[i];
    return r;
}

// Rows the fast sums cannot hold: two plain passes.  A row of nothing but -inf has s = 0.
template <int DT, int THREADS>
__device__ __attribute__((noinline)) RowStat slow_stat(const typename Elem<DT>::Raw* x, int vocab, float inv_tau, float* lds) {
    float m = -kInf;
    for (int i = threadIdx.x; i < vocab; i += THREADS) m = fmaxf(m, Elem<DT>::widen(x[i]));
    m = block_max_f<THREADS>(m, lds);
    const float ref = m == -kInf ? 0.0f : m;
    float s = 0.0f, e = 0.0f;
    for (int i = threadIdx.x; i < vocab; i += THREADS) {
        const float d = (Elem<DT>::widen(x[i]) - ref) * inv_tau, t = exp2_hw(d * kLog2e);
        s += t;
        if (t != 0.0f) e += t * d;
    }
    s = block_sum_f<THREADS>(s, lds);
    e = block_sum_f<THREADS>(e, lds);
    RowStat r = {0.0f, s, m, logf(s), 0.0f, true};
    r.entropy = s == 0.0f ? 0.0f : r.log_s - e / s;
    return r;
}

// Within 2^+-80 s, its reciprocal and a gradient's factor over it keep all of their bits.
__device__ __forceinline__ bool acc_good(const Acc& a) { return a.s > 0x1p-80f && a.s < 0x1p80f && fabsf(a.e) < kInf; }

struct Scale {               // k = fl(log2(e) / T), 1 / k, 1 / T
    float k, inv_k, inv_tau;
};

// ---- order of logits: by value, ties to the lowest index, NaN first; -0 and +0 are equal ----------
__device__ __forceinline__ uint64_t order_key(float v, unsigned index) {
    const unsigned b = __float_as_uint(v + 0.0f);
    unsigned o = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
    if (v != v) o = 0xfffffffeu;
    return (static_cast<uint64_t>(o) << 32) | (0xffffffffu - index);
}

__device__ __forceinline__ unsigned key_index(uint64_t key) { return 0xffffffffu - static_cast<unsigned>(key); }

__device__ __forceinline__ float key_value(uint64_t key) {       // not for a NaN's key
    const unsigned o = static_cast<unsigned>(key >> 32);
    return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}

// ---- the top entries of a row ---------------------------------------------------------------------
// One pass.  The row is read in chunks of adjacent elements.  From the first chunk every group of
// threads contributes its largest value; the top-th largest of those is a bound that at least `top`
// elements reach, and the elements that reach it become candidates, in a buffer of their wave.  From
// then on only elements above the floor -- a value that `top` elements before them reach -- are
// candidates (an equal one has a higher index), found by comparing the largest of a vector's elements.
// The floor is raised when 4, 8, 16, ... chunks have been read (2, 4, 8, ... cost 3 % more at
// 2048 x 50261) and at the end: with W waves, to the least of the waves' ceil(top / W)-th largest
// candidates.  Candidates below it are dropped; in a row in no particular order about
// top * (1 + ln(n / chunk)) elements ever become candidates.  The last ones are ranked against each other.
// A row that brings more candidates than fit (an ascending one) or holds a NaN is taken again by
// slow_top, whose steps bring at most 8 * top: 2048 x 50261 bf16, top 32: 55 us, ascending 1.6 ms.
template <int THREADS>
struct TopLds {
    static constexpr int kWaves = THREADS / kWave;
    // groups for the first chunk's bound: twice the largest `top`, so that the bound is near it.  A lone
    // wave's lanes make two each, of their even and their odd vectors.
    static constexpr int kGroups = THREADS == kWave ? 128 : 256;
    static constexpr int kSplit = THREADS == kWave ? 2 : 1;
    static constexpr int kRoom = kWaves == 16 ? 192 : 512;
    static constexpr int kFlat = kWaves > 4 ? 512 : 0;
    uint64_t cand[kWaves * kRoom];
    uint64_t flat[kFlat + 1];
    uint64_t list[kGroups];
    unsigned bound[kGroups];
    int held[kWaves];
    float floor[kWaves];
    unsigned limit, limit_group, tie, count;
    uint64_t reach;
    static_assert(kWaves * kRoom >= (kGroups < THREADS ? kGroups : THREADS) * 8, "a step of slow_top");
};

__device__ __forceinline__ unsigned order_of(float v) { return static_cast<unsigned>(order_key(v, 0) >> 32); }

__device__ __forceinline__ unsigned wave_max_u(unsigned v) {
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) {
        const unsigned o = __shfl_xor(v, d);
        v = o > v ? o : v;
    }
    return v;
}

// A value T that at least `want` (>= 1) of the wave's N values a lane reach, 0 if fewer are above 0.
// Either no more than want + want / 8 reach it, or it is the want-th largest (`exact`, and equal ones
// are why more reach it).  The search by halves takes about six counts instead of the fifteen that
// the want-th largest itself would.
template <int N>
__device__ __forceinline__ unsigned wave_nth(const unsigned (&v)[N], int want, bool& exact) {
    auto count = [&](unsigned t) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) c += __popcll(__ballot(v[i] >= t));
        return c;
    };
    exact = false;
    int reach = count(1);
    if (reach < want) return 0;
    unsigned top = v[0], low = ~0u;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        top = v[i] > top ? v[i] : top;
        low = v[i] && v[i] < low ? v[i] : low;
    }
    unsigned lo = ~wave_max_u(~low), hi = wave_max_u(top);       // all above 0 reach lo
    hi = hi == ~0u ? hi : hi + 1;                                // none reaches hi
    const int most = want + want / 8;
    while (reach > most && hi - lo > 1) {
        const unsigned mid = lo + (hi - lo) / 2;
        const int c = count(mid);
        if (c >= want) {
            lo = mid;
            reach = c;
        } else {
            hi = mid;
        }
    }
    exact = reach > most;
    return lo;
}

__device__ __forceinline__ int lanes_below(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi(static_cast<unsigned>(mask >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<unsigned>(mask), 0));
}

template <int THREADS>
struct TopState {
    uint64_t* mine;          // the wave's candidates
    int held;                // how many were found (more than kRoom: some are lost)
    float floor;
    __device__ __forceinline__ void add(bool hit, uint64_t key) {
        const uint64_t m = __ballot(hit);
        if (!m) return;
        const int at = held + lanes_below(m);
        if (hit && at < TopLds<THREADS>::kRoom) mine[at] = key;
        held += __popcll(m);
    }
};

// A better floor; drops what is below it.  False if candidates were lost.  Two barriers.
template <int THREADS>
__device__ __forceinline__ bool top_raise(TopLds<THREADS>& l, TopState<THREADS>& t, int top) {
    using L = TopLds<THREADS>;
    constexpr int kRegs = L::kRoom / kWave;
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const int have = t.held < L::kRoom ? t.held : L::kRoom;
    unsigned v[kRegs];
#pragma unroll
    for (int i = 0; i < kRegs; ++i) v[i] = lane + i * kWave < have ? static_cast<unsigned>(t.mine[lane + i * kWave] >> 32) : 0;
    const int want = (top + L::kWaves - 1) / L::kWaves;
    bool exact;
    unsigned nth;
    if (have <= kWave) {
        const unsigned few[1] = {v[0]};
        nth = wave_nth(few, want, exact);
    } else if (have <= 2 * kWave) {
        const unsigned few[2] = {v[0], v[1]};
        nth = wave_nth(few, want, exact);
    } else {
        nth = wave_nth(v, want, exact);
    }
    if (lane == 0) {
        l.held[wave] = t.held;
        l.floor[wave] = nth ? key_value(static_cast<uint64_t>(nth) << 32) : -kInf;
    }
    __syncthreads();
    float floor = l.floor[0];
    bool fits = l.held[0] <= L::kRoom;
#pragma unroll
    for (int w = 1; w < L::kWaves; ++w) {
        floor = fminf(floor, l.floor[w]);
        fits = fits && l.held[w] <= L::kRoom;
    }
    t.floor = fmaxf(t.floor, floor);
    const unsigned least = order_of(t.floor);
    int kept = 0;
#pragma unroll
    for (int i = 0; i < kRegs; ++i) {
        if (i * kWave >= have) continue;
        const uint64_t m = __ballot(v[i] >= least && v[i]);
        const uint64_t key = lane + i * kWave < have ? t.mine[lane + i * kWave] : 0;
        if (m >> lane & 1) t.mine[kept + lanes_below(m)] = key;
        kept += __popcll(m);
    }
    t.held = kept;
    __syncthreads();
    return fits;
}

// How many of n keys are above `key`; kStep reads are on their way at once, so that the keys are padded
// with zeros, which are below every key, to a multiple of it.
constexpr int kStep = 8;

__device__ __forceinline__ int count_above(const uint64_t* o, int n, uint64_t key) {
    int above = 0;
    for (int j = 0; j < n; j += kStep) {
        uint64_t other[kStep];
#pragma unroll
        for (int q = 0; q < kStep; ++q) other[q] = o[j + q];
#pragma unroll
        for (int q = 0; q < kStep; ++q) above += other[q] > key;
    }
    return above;
}

// The candidates in order into l.list.  All threads; one barrier before (two with many waves), one after.
template <int THREADS>
__device__ __forceinline__ bool top_rank(TopLds<THREADS>& l, TopState<THREADS>& t, int top) {
    using L = TopLds<THREADS>;
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    if (lane == 0) l.held[wave] = t.held;
    if (lane < kStep && t.held + lane < (t.held + kStep - 1) / kStep * kStep && t.held + lane < L::kRoom) t.mine[t.held + lane] = 0;
    __syncthreads();
    bool fits = true;
    int total = 0, before = 0;
#pragma unroll
    for (int w = 0; w < L::kWaves; ++w) {
        const int n = l.held[w];
        fits = fits && n <= L::kRoom;
        before += w < wave ? n : 0;
        total += n;
    }
    if (L::kFlat && fits && total <= L::kFlat - kStep) {         // many waves with few candidates each: side by side
        if (lane < t.held) l.flat[before + lane] = t.mine[lane];
        for (int i = lane + kWave; i < t.held; i += kWave) l.flat[before + i] = t.mine[i];
        if (threadIdx.x < kStep) l.flat[total + threadIdx.x] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < total; i += THREADS) {
            const uint64_t key = l.flat[i];
            const int rank = count_above(l.flat, total, key);
            if (rank < top) l.list[rank] = key;
        }
    } else if (fits) {
        for (int i = lane; i < t.held; i += kWave) {
            const uint64_t key = t.mine[i];
            int rank = 0;
            for (int w = 0; w < L::kWaves; ++w) rank += count_above(l.cand + w * L::kRoom, l.held[w], key);
            if (rank < top) l.list[rank] = key;
        }
    }
    __syncthreads();
    return fits;
}

// The first chunk's bound.  `best`: the largest element of the caller's groups (or of the group of kShare
// neighbours it is in) as order_of, 0: none.  Afterwards l.limit is the bound (0: fewer than `top` groups
// have an element) and l.limit_group the last group whose equal elements are needed (all: INT32_MAX).
// Group h of a thread is h * kWave + thread, or thread / kShare.
template <int THREADS>
__device__ __forceinline__ void top_bound(TopLds<THREADS>& l, const unsigned (&best)[TopLds<THREADS>::kSplit], int top) {
    using L = TopLds<THREADS>;
    constexpr int kShare = THREADS * L::kSplit / L::kGroups, kRegs = L::kGroups / kWave;
    const int tid = threadIdx.x;
    if (tid % kShare == 0) {
#pragma unroll
        for (int h = 0; h < L::kSplit; ++h) l.bound[h * kWave + tid / kShare] = best[h];
    }
    __syncthreads();
    if (tid < kWave) {
        unsigned v[kRegs];
#pragma unroll
        for (int i = 0; i < kRegs; ++i) v[i] = l.bound[i * kWave + tid];
        bool exact;
        const unsigned nth = wave_nth(v, top, exact);
        int group = INT32_MAX;
        if (exact) {                                             // more are equal than needed
            int need = top;
#pragma unroll
            for (int i = 0; i < kRegs; ++i) need -= __popcll(__ballot(v[i] > nth));
#pragma unroll
            for (int i = 0; i < kRegs; ++i) {
                const uint64_t m = __ballot(v[i] == nth);
                const int c = __popcll(m);
                if (group == INT32_MAX && need <= c)
                    group = i * kWave + __ffsll(__ballot((m >> tid & 1) && lanes_below(m) == need - 1)) - 1;
                need -= c;
            }
        }
        if (tid == 0) {
            l.limit = nth;
            l.limit_group = group;
            l.tie = 0;
        }
    }
    __syncthreads();
}

// Steps of 8 elements a thread, 256 threads at most; exact for every row, NaN included.
template <int DT, int THREADS>
__device__ __attribute__((noinline)) void slow_top(const typename Elem<DT>::Raw* x, int vocab, int top, TopLds<THREADS>& l) {
    using L = TopLds<THREADS>;
    constexpr int kTakers = L::kGroups < THREADS ? L::kGroups : THREADS, kElements = kTakers * 8;
    const int tid = threadIdx.x;
    int have = 0;
    uint64_t low = 0;                                            // the list's last key once it is full
    for (int j = tid; j < L::kGroups; j += THREADS) l.list[j] = 0;
    for (int base = 0; base < vocab; base += kElements) {
        __syncthreads();
        if (tid == 0) {
            l.count = 0;
            l.reach = 0;
        }
        uint64_t best = 0;
        uint64_t keys[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = base + tid * 8 + j;
            const bool in = tid < kTakers && i < vocab;
            keys[j] = in ? order_key(Elem<DT>::widen(x[i]), i) : 0;
            if (keys[j] <= low) keys[j] = 0;
            best = keys[j] > best ? keys[j] : best;
        }
        // keys are all different, so at most 8 * top elements reach the top-th of the threads' best
        if (tid < kTakers) l.cand[tid] = best;
        __syncthreads();
        if (tid < kTakers && best && count_above(l.cand, kTakers, best) == top - 1) l.reach = best;
        __syncthreads();
        const uint64_t reach = l.reach;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (keys[j] && keys[j] >= reach) l.cand[atomicAdd(&l.count, 1u)] = keys[j];
        __syncthreads();
        const int n = static_cast<int>(l.count), total = have + n;
        if (tid < kStep && n + tid < L::kWaves * L::kRoom) l.cand[n + tid] = 0;
        __syncthreads();
        constexpr int kOwn = (kElements + L::kGroups + THREADS - 1) / THREADS;
        uint64_t own[kOwn];
        int rank[kOwn];
#pragma unroll
        for (int e = 0; e < kOwn; ++e) {
            const int i = tid + e * THREADS;
            own[e] = 0;
            rank[e] = top;
            if (i >= total) continue;
            own[e] = i < have ? l.list[i] : l.cand[i - have];
            rank[e] = (i < have ? i : count_above(l.list, have, own[e])) + count_above(l.cand, n, own[e]);
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kOwn; ++e)
            if (rank[e] < top) l.list[rank[e]] = own[e];
        __syncthreads();
        have = total < top ? total : top;
        if (have == top) low = l.list[top - 1];
    }
    __syncthreads();
}

struct ScoreArgs {
    const void* x;
    Rows rows;
    int vocab, top;
    const int64_t* targets;
    int64_t ignore_index;
    float *logprob, *entropy, *lse, *top_logprobs;
    int32_t* top_ids;
    Scale scale;
    int64_t row0;                // of the launch's first block
};

__device__ __forceinline__ float log_prob(const RowStat& st, const Scale& sc, float v, float lse) {
    if (st.slow) return v == -kInf && !(st.s != st.s) ? -kInf : (v - st.m) - st.log_s;
    const float y = fmaf(v, sc.k, -st.R) - st.log_s;             // log_s: log2 here
    return fabsf(y) < 1e30f ? y * sc.inv_k : v - lse;
}

// One block per row: a few vectors of 16 bytes per thread and chunk, the next chunk's loads in flight
// while one is summed.  Blocks of 256 threads take two: four need more than their 64 registers (fp32
// 4096 x 128000, top 8: 314 us with two, 343 with four; 2048 x 50261 bf16, top 32: 55 and 57).
constexpr int scores_vectors(int threads) { return threads == 256 ? 2 : 4; }

// Blocks of 256 threads: eight fit a CU by their LDS (19.6 KiB), 64 registers a thread.
constexpr int scores_waves(int threads, bool top) { return !top ? 1 : threads == 1024 ? 4 : threads == 256 ? 8 : 6; }

template <int DT, int THREADS, bool TOP>
__global__ __launch_bounds__(THREADS, scores_waves(THREADS, TOP)) void token_scores_kernel(const ScoreArgs a) {
    using E = Elem<DT>;
    using V = Vec<DT>;
    using L = TopLds<THREADS>;
    constexpr int kU = scores_vectors(THREADS);
    __shared__ Acc lds[THREADS / kWave];
    __shared__ float red[THREADS / kWave];
    __shared__ L l;
    const int64_t row = a.row0 + blockIdx.x;
    const typename E::Raw* x = static_cast<const typename E::Raw*>(a.x) + a.rows.offset(row);
    const Span sp = V::span(x, a.vocab);
    const uint4* body = reinterpret_cast<const uint4*>(x + sp.head);
    const int tid = threadIdx.x;
    const float k = a.scale.k;
    Acc acc = acc_empty();
    TopState<THREADS> t = {l.cand + (tid / kWave) * L::kRoom, 0, -kInf};

    uint4 cur[kU], next[kU];
    auto fetch = [&](int base) {
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int i = base + u * THREADS + tid;
            next[u] = i < sp.nvec ? load_once(body + i) : V::fill();
        }
    };
    fetch(0);
    // the row's ends, an element a thread: the head belongs to the first chunk, the tail behind the last
    const float head = tid < sp.head ? E::widen(x[tid]) : -kInf;
    const float tail = tid < sp.tail ? E::widen(x[a.vocab - sp.tail + tid]) : -kInf;
#pragma unroll
    for (int u = 0; u < kU; ++u) cur[u] = next[u];
    if (kU * THREADS < sp.nvec) fetch(kU * THREADS);
    // the target's logit, long before it is wanted
    int64_t want = a.ignore_index;
    float given = 0.0f;
    if (tid == 0 && a.targets) {
        want = a.targets[row];
        if (want >= 0 && want < a.vocab) given = E::widen(x[want]);
    }
    {
        const float v[2] = {head, tail};
        acc_add<true>(acc, v, fmaxf(head, tail), k);
    }
    float most[L::kSplit];
    most[0] = head;
#pragma unroll
    for (int h = 1; h < L::kSplit; ++h) most[h] = -kInf;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
        float v[V::N];
        V::widen(cur[u], v);
        const float peak = V::peak(cur[u], v);
        most[u % L::kSplit] = fmaxf(most[u % L::kSplit], peak);
        acc_add<true>(acc, v, peak, k);
    }
    if (TOP) {
        constexpr int kShare = THREADS * L::kSplit / L::kGroups;
        unsigned best[L::kSplit];
#pragma unroll
        for (int h = 0; h < L::kSplit; ++h) {
            best[h] = (h == 0 && tid < sp.head) || h * THREADS + tid < sp.nvec ? order_of(most[h]) : 0;
            for (int d = 1; d < kShare; d <<= 1) {
                const unsigned o = __shfl_xor(best[h], d);
                best[h] = o > best[h] ? o : best[h];
            }
        }
        top_bound(l, best, a.top);
        const unsigned limit = l.limit, last = l.limit_group;
        const float lim = limit ? key_value(static_cast<uint64_t>(limit) << 32) : -kInf;
        int tie = INT32_MAX;
        if (last != INT32_MAX) {
            // groups up to `last` at the bound's value: the lowest index of each has to be let in
#pragma unroll
            for (int h = 0; h < L::kSplit; ++h) {
                if (best[h] != limit || static_cast<unsigned>(h * kWave + tid / kShare) > last) continue;
                int at = h == 0 && tid < sp.head && head == lim ? tid : INT32_MAX;
#pragma unroll
                for (int u = h; u < kU; u += L::kSplit) {
                    float v[V::N];
                    V::widen_again(cur[u], v);
#pragma unroll
                    for (int i = 0; i < V::N; ++i)
                        if (at == INT32_MAX && u * THREADS + tid < sp.nvec && v[i] == lim)
                            at = sp.head + (u * THREADS + tid) * V::N + i;
                }
                for (int d = 1; d < kShare; d <<= 1) {
                    const int o = __shfl_xor(at, d);
                    at = o < at ? o : at;
                }
                atomicMax(&l.tie, static_cast<unsigned>(at));
            }
            __syncthreads();
            tie = static_cast<int>(l.tie);
        }
        t.add(tid < sp.head && (head > lim || (head == lim && tid <= tie)), order_key(head, tid));
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            float v[V::N];
            V::widen_again(cur[u], v);
            const bool in = u * THREADS + tid < sp.nvec;
            if (!__any(in && max_of(v) >= lim)) continue;
#pragma unroll
            for (int i = 0; i < V::N; ++i) {
                const int at = sp.head + (u * THREADS + tid) * V::N + i;
                t.add(in && (v[i] > lim || (v[i] == lim && at <= tie)), order_key(v[i], at));
            }
        }
        t.floor = lim;           // `top` elements reach it; -inf without a bound, and there is no further chunk
    }
    bool fits = true;
    int chunk = 1, due = 4;                                      // chunks read when the floor is raised next
    for (int base = kU * THREADS; base < sp.nvec; ++chunk) {
#pragma unroll
        for (int u = 0; u < kU; ++u) cur[u] = next[u];
        const int first = base;
        base += kU * THREADS;
        if (base < sp.nvec) fetch(base);
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            float v[V::N];
            V::widen(cur[u], v);
            const float peak = V::peak(cur[u], v);
            acc_add<true>(acc, v, peak, k);
            if (TOP && __any(peak > t.floor)) {
#pragma unroll
                for (int i = 0; i < V::N; ++i)
                    t.add(v[i] > t.floor, order_key(v[i], sp.head + (first + u * THREADS + tid) * V::N + i));
            }
        }
        if (TOP && chunk + 1 == due && base < sp.nvec) {
            fits = top_raise(l, t, a.top) && fits;
            due *= 2;
        }
    }
    if (TOP) {
        // without a bound every element is a candidate
        t.add(tid < sp.tail && (l.limit == 0 || tail > t.floor), order_key(tail, a.vocab - sp.tail + tid));
        if (chunk > 1) fits = top_raise(l, t, a.top) && fits;
        fits = top_rank(l, t, a.top) && fits;
    }
    acc = acc_block<true, THREADS>(acc, lds);
    RowStat st = {acc.R, acc.s, 0.0f, log2f(acc.s), 0.0f, false};
    st.entropy = (st.log_s - acc.e / acc.s) * a.scale.inv_k;
    float lse = static_cast<float>((static_cast<double>(st.R) + st.log_s) * static_cast<double>(a.scale.inv_k));
    if (!acc_good(acc)) {
        st = slow_stat<DT, THREADS>(x, a.vocab, a.scale.inv_tau, red);
        lse = st.m + st.log_s;
        fits = fits && st.s == st.s;         // lists do not depend on the sums, but the comparisons above pass a NaN by
    }
    if (TOP && !fits) slow_top<DT, THREADS>(x, a.vocab, a.top, l);
    if (tid == 0) {
        a.lse[row] = lse;
        a.entropy[row] = st.entropy;
        if (a.targets) {
            float lp = 0.0f;
            if (want != a.ignore_index)
                lp = want >= 0 && want < a.vocab ? log_prob(st, a.scale, given, lse) : __builtin_nanf("");
            a.logprob[row] = lp;
        }
    }
    if (TOP) {
        for (int j = tid; j < a.top; j += THREADS) {
            const uint64_t key = l.list[j];
            const float v = static_cast<unsigned>(key >> 32) == 0xfffffffeu ? __builtin_nanf("") : key_value(key);
            a.top_ids[row * a.top + j] = static_cast<int32_t>(key_index(key));
            a.top_logprobs[row * a.top + j] = log_prob(st, a.scale, v, lse);
        }
    }
}

// ---- distillation ---------------------------------------------------------------------------------
struct TeacherArgs {
    const int32_t* ids;
    const float* lp;
    int64_t id_stride, lp_stride;
    int k;
    float tau;
    const float* row_weight;
};

struct DistillArgs {
    const void* x;
    Rows rows;
    int vocab;
    TeacherArgs t;
    Scale scale;
    float* loss;
    float* stat;                 // FA_DISTILL_STAT floats per row: R, s, m, log s; R is NaN for a slow row
    float* partial;              // FA_DISTILL_WS_FLOATS for the sums of rows' parts, or NULL
    const float* stat_in;
    const float* row_grad;
    void* grad;
    Rows grad_rows;
    int64_t row0;                // of the launch's first block
};

// One row's teacher, made by the first wave alone: entries j = lane + 64 i.
constexpr int kPer = FA_TOP_MAX / kWave;

struct TeacherLds {
    int id[FA_TOP_MAX];          // -1: nothing to write (absent, or an earlier entry has the same id)
    float t[FA_TOP_MAX];         // probability, of all entries of the same id together
    float x[FA_TOP_MAX];         // the student's logit
    int empty, bad;
};

struct Teacher {
    int id[kPer];
    float lp[kPer], t[kPer], log_t[kPer], x[kPer];
};

__device__ __forceinline__ float wave_max_f(float v) {
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}

__device__ __forceinline__ float wave_sum_f(float v) {
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// In three steps, so that a kernel can put its own loads between them.
__device__ __forceinline__ void teacher_fetch(const TeacherArgs& a, int64_t row, Teacher& r) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int j = threadIdx.x + kWave * i;
        r.id[i] = -1;
        r.lp[i] = -kInf;
        if (j < a.k) {
            r.id[i] = a.ids[row * a.id_stride + j];
            r.lp[i] = a.lp[row * a.lp_stride + j];
        }
    }
}

template <int DT>
__device__ __forceinline__ void teacher_gather(const typename Elem<DT>::Raw* x, int vocab, Teacher& r) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        r.x[i] = -kInf;
        if (r.id[i] >= 0 && r.id[i] < vocab) r.x[i] = Elem<DT>::widen(x[r.id[i]]);
    }
}

__device__ __forceinline__ void teacher_make(Teacher& r, int vocab, float inv_tau, TeacherLds& l) {
    const int lane = threadIdx.x;
    bool outside = false, broken = false;
    float peak = -kInf;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        if (r.id[i] < 0) r.lp[i] = -kInf;
        outside = outside || r.id[i] >= vocab;
        broken = broken || r.lp[i] != r.lp[i];
        peak = fmaxf(peak, r.lp[i]);
    }
    broken = __any(broken);
    peak = wave_max_f(peak);
    const bool empty = !broken && peak == -kInf;                 // whatever its ids
    const bool bad = broken || __any(outside) || peak == kInf;
    float z = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        r.log_t[i] = r.lp[i] == -kInf ? -kInf : (r.lp[i] - peak) * inv_tau;
        r.t[i] = exp2_hw(r.log_t[i] * kLog2e);
        z += r.t[i];
    }
    z = wave_sum_f(z);
    const float log_z = logf(z), inv_z = 1.0f / z;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int j = lane + kWave * i;
        r.log_t[i] -= log_z;
        r.t[i] = empty ? 0.0f : r.t[i] * inv_z;
        l.id[j] = r.id[i] < vocab ? r.id[i] : -1;
        l.t[j] = r.t[i];
        l.x[j] = r.x[i];
    }
    if (lane == 0) {
        l.empty = empty;
        l.bad = bad;
    }
}

// Entries that name one token: the first takes their probabilities together (the gradient's term).
__device__ __forceinline__ void teacher_unite(int k, TeacherLds& l) {
    float sum[kPer];
    int id[kPer];
    __builtin_amdgcn_wave_barrier();
    __threadfence_block();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int j = threadIdx.x + kWave * i;
        sum[i] = 0.0f;
        id[i] = -1;
        if (j < k && l.id[j] >= 0) {
            id[i] = l.id[j];
            for (int o = 0; o < k; ++o)
                if (l.id[o] == l.id[j]) {
                    sum[i] += l.t[o];
                    if (o < j) id[i] = -1;
                }
        }
    }
    __builtin_amdgcn_wave_barrier();
    __threadfence_block();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int j = threadIdx.x + kWave * i;
        if (j < k) {
            l.id[j] = id[i];
            l.t[j] = sum[i];
        }
    }
}

// The loss, by the first wave.  Where the teacher wants what a mask has taken out, log q is x / T to all its
// bits; T^2 t x / T is then added as T (t x / 4) * 4, since x / T, and the sum of all t x, may be beyond fp32.
__device__ __forceinline__ float row_loss(const DistillArgs& a, const Teacher& e, const RowStat& st, float weight, bool bad) {
    float sum = 0.0f, far = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        if (!(e.t[i] > 0.0f)) continue;
        const bool none = e.x[i] == -kInf;
        float log_q, apart;
        if (st.slow) {
            apart = none ? -kInf : 0.25f * e.x[i] - 0.25f * st.m;
            log_q = none ? -kInf : (e.x[i] - st.m) * a.scale.inv_tau - st.log_s;
        } else {
            const float y = fmaf(e.x[i], a.scale.k, -st.R) - st.log_s;
            apart = 0.25f * e.x[i];
            log_q = y * kLn2;
        }
        if (log_q < -1e30f) far -= e.t[i] * apart;
        else sum += e.t[i] * (e.log_t[i] - log_q);
    }
    sum = wave_sum_f(sum) * (a.t.tau * a.t.tau) * weight;
    if (__any(far != 0.0f)) sum += wave_sum_f(far) * (a.t.tau * weight) * 4.0f;
    return bad || st.s != st.s ? __builtin_nanf("") : sum;
}

// c * q of one element
struct Softmax {
    float k, R, cs;              // 2^(x k - R) * cs
    float m, c2;                 // slow: 2^((x - m) k' - c2) * c
    float c;
    bool slow;
    __device__ __forceinline__ float operator()(float v) const {
        if (slow) return exp2_hw((v - m) * k - c2) * c;
        return exp2_hw(fmaf(v, k, -R)) * cs;
    }
};

__device__ __forceinline__ Softmax softmax_of(const RowStat& st, const Scale& sc, float c) {
    Softmax f;
    f.slow = st.slow;
    f.k = st.slow ? sc.inv_tau * kLog2e : sc.k;
    f.R = st.R;
    f.cs = c / st.s;
    f.m = st.m == -kInf ? 0.0f : st.m;
    f.c2 = st.log_s == -kInf ? 0.0f : st.log_s * kLog2e;
    f.c = c;
    return f;
}

constexpr int kU = 4;      // vectors a thread has on their way

// Vectors [lo, hi) of a row's part; the head goes with the first part, the tail with the last.
struct Part {
    int lo, hi;
};

__device__ __forceinline__ Part part_of(const Span& sp, int part, int parts) {
    return {static_cast<int>(static_cast<int64_t>(sp.nvec) * part / parts),
            static_cast<int>(static_cast<int64_t>(sp.nvec) * (part + 1) / parts)};
}

// Writes f(element) over a part of a row; reads by 16 bytes, writes so where the gradient's row has
// the same alignment.
// LAST: the elements are read past the caches.
template <int DT, int THREADS, bool LAST, class F>
__device__ __forceinline__ void map_row(const typename Elem<DT>::Raw* x, typename Elem<DT>::Raw* g, int vocab, int part,
                                        int parts, F f) {
    using E = Elem<DT>;
    using V = Vec<DT>;
    const Span sp = V::span(x, vocab);
    const int tid = threadIdx.x;
    if (part == 0 && tid < sp.head) g[tid] = E::narrow(f(E::widen(x[tid])));
    if (part == parts - 1 && tid < sp.tail) {
        const int i = vocab - sp.tail + tid;
        g[i] = E::narrow(f(E::widen(x[i])));
    }
    const bool same = reinterpret_cast<uintptr_t>(x) % 16 == reinterpret_cast<uintptr_t>(g) % 16;
    const uint4* body = reinterpret_cast<const uint4*>(x + sp.head);
    const int lo = part_of(sp, part, parts).lo, hi = part_of(sp, part, parts).hi;
    for (int base = lo; base < hi; base += kU * THREADS) {
        uint4 r[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int i = base + u * THREADS + tid;
            if (i < hi) r[u] = LAST ? load_once(body + i) : body[i];
        }
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int i = base + u * THREADS + tid;
            if (i >= hi) continue;
            float v[V::N];
            V::widen(r[u], v);
#pragma unroll
            for (int j = 0; j < V::N; ++j) v[j] = f(v[j]);
            if (same) {
                store_once(reinterpret_cast<uint4*>(g + sp.head) + i, V::narrow(v));
            } else {
#pragma unroll
                for (int j = 0; j < V::N; ++j) g[sp.head + i * V::N + j] = E::narrow(v[j]);
            }
        }
    }
}

// All of the block's stores have arrived before any thread goes on: the next store to one of their
// addresses, by another wave, is the one that stays.
__device__ __forceinline__ void stores_done() {
    __builtin_amdgcn_s_waitcnt(0x0f70);            // vmcnt(0) alone
    __syncthreads();
}

// The teacher's tokens, after the row's (or part's) other elements have been written: c (q - t).
template <int DT>
__device__ __forceinline__ void fix_row(typename Elem<DT>::Raw* g, const TeacherLds& l, int k, int lo, int hi, const Softmax& f) {
    for (int j = threadIdx.x; j < k; j += kWave) {
        const int id = l.id[j];
        if (id >= lo && id < hi) g[id] = Elem<DT>::narrow(f(l.x[j]) - f.c * l.t[j]);
    }
}

template <int DT, int THREADS>
__device__ __forceinline__ Acc sum_row(const typename Elem<DT>::Raw* x, int vocab, float k, int part, int parts) {
    using E = Elem<DT>;
    using V = Vec<DT>;
    const Span sp = V::span(x, vocab);
    const int tid = threadIdx.x;
    const int lo = part_of(sp, part, parts).lo, hi = part_of(sp, part, parts).hi;
    const uint4* body = reinterpret_cast<const uint4*>(x + sp.head);
    Acc acc = acc_empty();
    uint4 next[kU];
    auto fetch = [&](int base) {
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int i = base + u * THREADS + tid;
            next[u] = i < hi ? body[i] : V::fill();
        }
    };
    fetch(lo);
    if (part == 0 && tid < sp.head) {
        const float v[1] = {E::widen(x[tid])};
        acc_add<false>(acc, v, v[0], k);
    }
    if (part == parts - 1 && tid < sp.tail) {
        const float v[1] = {E::widen(x[vocab - sp.tail + tid])};
        acc_add<false>(acc, v, v[0], k);
    }
    for (int base = lo; base < hi;) {
        uint4 cur[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) cur[u] = next[u];
        base += kU * THREADS;
        if (base < hi) fetch(base);
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            float v[V::N];
            V::widen(cur[u], v);
            acc_add<false>(acc, v, V::peak(cur[u], v), k);
        }
    }
    return acc;
}

// The sums of a row's parts, for few long rows (launch_step): (R, s) of part p of a row at
// partial[2 * (row * parts + p)].
template <int DT, int THREADS>
__global__ __launch_bounds__(THREADS) void distill_parts_kernel(const DistillArgs a) {
    __shared__ Acc lds[THREADS / kWave];
    const int64_t row = a.row0 + blockIdx.x;
    const typename Elem<DT>::Raw* x = static_cast<const typename Elem<DT>::Raw*>(a.x) + a.rows.offset(row);
    const Acc acc = acc_block<false, THREADS>(sum_row<DT, THREADS>(x, a.vocab, a.scale.k, blockIdx.y, gridDim.y), lds);
    if (threadIdx.x == 0) {
        float* o = a.partial + 2 * (row * gridDim.y + blockIdx.y);
        o[0] = acc.R;
        o[1] = acc.s;
    }
}

// LOSS alone: the sums of a row.  GRAD alone: from the sums of an earlier call; a row may be cut in
// parts (blockIdx.y).  Both, in parts: from the sums of distill_parts_kernel.  Both, whole: the row is
// read twice, the second time from the memory-side cache as long as the rows under way fit there (see
// launch_step).
template <int DT, int THREADS, bool LOSS, bool GRAD, bool LAST>
__global__ __launch_bounds__(THREADS) void distill_kernel(const DistillArgs a) {
    using E = Elem<DT>;
    __shared__ Acc lds[THREADS / kWave];
    __shared__ float red[THREADS / kWave];
    __shared__ TeacherLds l;
    const int64_t row = a.row0 + blockIdx.x;
    const int part = blockIdx.y, parts = gridDim.y;              // LOSS alone: one part
    const typename E::Raw* x = static_cast<const typename E::Raw*>(a.x) + a.rows.offset(row);
    const float weight = a.t.row_weight ? a.t.row_weight[row] : 1.0f;
    const float c = GRAD ? weight * a.t.tau * (a.row_grad ? a.row_grad[row] : 1.0f) : 0.0f;
    const bool first_wave = threadIdx.x < kWave;
    Teacher e;
    if (first_wave) {
        teacher_fetch(a.t, row, e);
        teacher_gather<DT>(x, a.vocab, e);
        teacher_make(e, a.vocab, a.scale.inv_tau, l);
        if (GRAD) teacher_unite(a.t.k, l);
    }
    RowStat st;
    bool off = weight == 0.0f;                                   // nothing of the row's logits counts
    if (LOSS) {
        Acc acc = acc_empty();
        if (GRAD && parts > 1) {                                 // every wave joins them all; at most 64
            const int p = threadIdx.x % kWave;
            const float* o = a.partial + 2 * (row * parts + (p < parts ? p : 0));
            if (p < parts) acc = {o[0], o[1], 0.0f};
            acc = acc_wave<false>(acc);
            __syncthreads();
        } else {
            if (!off) acc = sum_row<DT, THREADS>(x, a.vocab, a.scale.k, 0, 1);
            acc = acc_block<false, THREADS>(acc, lds);
        }
        off = off || l.empty;
        st = {acc.R, acc.s, 0.0f, log2f(acc.s), 0.0f, false};
        if (!off && !acc_good(acc)) st = slow_stat<DT, THREADS>(x, a.vocab, a.scale.inv_tau, red);
        if (first_wave && part == 0) {
            const float loss = off ? 0.0f : row_loss(a, e, st, weight, l.bad);
            if (threadIdx.x == 0) {
                a.loss[row] = loss;
                if (a.stat) {
                    float* o = a.stat + FA_DISTILL_STAT * row;
                    o[0] = st.slow ? __builtin_nanf("") : st.R;
                    o[1] = st.s;
                    o[2] = st.m;
                    o[3] = st.log_s;
                }
            }
        }
    } else {
        const float* o = a.stat_in + FA_DISTILL_STAT * row;
        st = {o[0], o[1], o[2], o[3], 0.0f, o[0] != o[0]};
        __syncthreads();
        off = off || l.empty;
    }
    if (!GRAD) return;
    typename E::Raw* g = static_cast<typename E::Raw*>(a.grad) + a.grad_rows.offset(row);
    if (off || c == 0.0f || l.bad) {
        const float v = !off && l.bad ? __builtin_nanf("") : 0.0f;
        map_row<DT, THREADS, LAST>(x, g, a.vocab, part, parts, [v](float) { return v; });
        return;
    }
    const Softmax f = softmax_of(st, a.scale, c);
    map_row<DT, THREADS, LAST>(x, g, a.vocab, part, parts, f);
    stores_done();
    if (first_wave) {
        const Span sp = Vec<DT>::span(x, a.vocab);
        const int lo = part == 0 ? 0 : sp.head + part_of(sp, part, parts).lo * Vec<DT>::N;
        const int hi = part == parts - 1 ? a.vocab : sp.head + part_of(sp, part, parts).hi * Vec<DT>::N;
        fix_row<DT>(g, l, a.t.k, lo, hi, f);
    }
}

// Loss and gradient of a row that stays in its block's registers between the sums and the gradient:
// read once, written once.  NV vectors of 16 bytes a thread.
template <int DT, int THREADS, int NV>
__global__ __launch_bounds__(THREADS) void distill_step_kernel(const DistillArgs a) {
    using E = Elem<DT>;
    using V = Vec<DT>;
    __shared__ Acc lds[THREADS / kWave];
    __shared__ float red[THREADS / kWave];
    __shared__ TeacherLds l;
    const int64_t row = a.row0 + blockIdx.x;
    const typename E::Raw* x = static_cast<const typename E::Raw*>(a.x) + a.rows.offset(row);
    typename E::Raw* g = static_cast<typename E::Raw*>(a.grad) + a.grad_rows.offset(row);
    const float weight = a.t.row_weight ? a.t.row_weight[row] : 1.0f;
    const float c = weight * a.t.tau;
    const bool first_wave = threadIdx.x < kWave;
    const int tid = threadIdx.x;
    const Span sp = V::span(x, a.vocab);
    const uint4* body = reinterpret_cast<const uint4*>(x + sp.head);
    const float k = a.scale.k;
    Teacher e;
    if (first_wave) teacher_fetch(a.t, row, e);
    uint4 r[NV];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        const int i = u * THREADS + tid;
        r[u] = i < sp.nvec ? load_once(body + i) : V::fill();
    }
    const bool has_head = tid < sp.head, has_tail = tid < sp.tail;
    const int tail_at = a.vocab - sp.tail + tid;
    const float head = has_head ? E::widen(x[tid]) : -kInf, tail = has_tail ? E::widen(x[tail_at]) : -kInf;
    if (first_wave) teacher_gather<DT>(x, a.vocab, e);
    Acc acc = acc_empty();
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        float v[V::N];
        V::widen(r[u], v);
        acc_add<false>(acc, v, V::peak(r[u], v), k);
    }
    {
        const float v[2] = {head, tail};
        acc_add<false>(acc, v, fmaxf(head, tail), k);
    }
    if (first_wave) {
        teacher_make(e, a.vocab, a.scale.inv_tau, l);
        teacher_unite(a.t.k, l);
    }
    acc = acc_block<false, THREADS>(acc, lds);
    const bool off = weight == 0.0f || l.empty;
    RowStat st = {acc.R, acc.s, 0.0f, log2f(acc.s), 0.0f, false};
    if (!off && !acc_good(acc)) st = slow_stat<DT, THREADS>(x, a.vocab, a.scale.inv_tau, red);
    if (first_wave) {
        const float loss = off ? 0.0f : row_loss(a, e, st, weight, l.bad);
        if (tid == 0) a.loss[row] = loss;
    }
    const bool flat = off || c == 0.0f || l.bad;                 // one value for the whole row
    const float level = !off && l.bad ? __builtin_nanf("") : 0.0f;
    const Softmax f = softmax_of(st, a.scale, c);
    const bool same = reinterpret_cast<uintptr_t>(x) % 16 == reinterpret_cast<uintptr_t>(g) % 16;
    uint4* out = reinterpret_cast<uint4*>(g + sp.head);
    if (has_head) g[tid] = E::narrow(flat ? level : f(head));
    if (has_tail) g[tail_at] = E::narrow(flat ? level : f(tail));
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        const int i = u * THREADS + tid;
        if (i >= sp.nvec) continue;
        float v[V::N];
        V::widen_again(r[u], v);
        if (flat) {
#pragma unroll
            for (int j = 0; j < V::N; ++j) v[j] = level;
        } else {
#pragma unroll
            for (int j = 0; j < V::N; ++j) v[j] = f(v[j]);
        }
        if (same) {
            store_once(out + i, V::narrow(v));
        } else {
#pragma unroll
            for (int j = 0; j < V::N; ++j) g[sp.head + i * V::N + j] = E::narrow(v[j]);
        }
    }
    if (flat) return;
    stores_done();
    if (first_wave) fix_row<DT>(g, l, a.t.k, 0, a.vocab, f);
}

// ---- merging the clients' lists -------------------------------------------------------------------
// One block per row, every entry in a register of its thread.  Entries are grouped by a hash table in
// LDS.  A group's probabilities are added as whole numbers, scaled by the power of two that puts the
// group's largest below 2^51: whole numbers add up to the same sum in any order, and a sum is off by
// no more than 2^-51 of the largest term per entry (fp64 additions: 2^-53 of the sum each).  A term
// may be rounded up to 2^51, and 2^13 of those are 2^64: that sum alone comes out as 0, which a
// group's is not otherwise, its largest term being 2^50 at least (or subnormal).  The groups' values
// are then ranked, ties to the lowest id.
// A table takes kFull different tokens, and those that are on their way when it fills; a row with more
// is merged in rounds, each of which takes the tokens that got into the table and ranks them together
// with the best of the rounds before.
struct MergeArgs {
    const int32_t* ids;
    const float* lp;
    int64_t id_client, id_row, lp_client, lp_row;
    const float* unit;
    int64_t unit_client, unit_row;
    int K, k, top;
    int64_t row0;                // of the launch's first block
    int near;                    // both lists have one client stride, K of which stay below 2^30 elements
    uint64_t per_k;              // 2^32 / k, rounded up: i / k for i * k < 2^32
    int32_t* out_ids;
    float* out_lp;
    double w[FA_MERGE_CLIENTS];
};

__device__ __forceinline__ bool before(uint64_t ka, unsigned ia, uint64_t kb, unsigned ib) {
    return ka > kb || (ka == kb && ia < ib);
}

constexpr unsigned kFree = ~0u;
constexpr unsigned kExpInf = 2047;

// ROUNDS: rows may hold more different tokens than the table takes; else at most SLOTS / 2.
template <int SLOTS, bool ROUNDS>
struct MergeLds {
    static constexpr int kFull = SLOTS * 3 / 4;
    static constexpr int kList = ROUNDS ? FA_TOP_MAX : 0;
    static constexpr int kAll = SLOTS + kList + 8;
    static_assert(!ROUNDS || SLOTS / 2 >= FA_TOP_MAX, "the ranked values");
    double share[FA_MERGE_CLIENTS];
    unsigned answered[FA_MERGE_CLIENTS];
    unsigned token[kAll];                          // by slot: id, ~0: free.  Later by group: id
    uint64_t sum[kAll];                            // by slot: sum.  Later by group: the value's bits
    union {
        unsigned peak[SLOTS];                      // exponent of the group's largest term
        uint64_t best[SLOTS / 2];                  // after the last round: the ranked values
    };
    u16 slot[ROUNDS ? SLOTS : SLOTS / 2];          // by group, in the order of their coming
    uint64_t list_key[kList + 1];                  // the best of the rounds before
    unsigned list_id[kList + 1];
    unsigned count, open, left, bound;
    double total;
};

// The slot of `id` (< 2^31), or -1 with `at` the free slot met first, kFree in a full table.
template <int SLOTS, bool ROUNDS>
__device__ __forceinline__ int find_slot(const MergeLds<SLOTS, ROUNDS>& l, unsigned id, unsigned& at) {
    for (int n = 0; n < SLOTS; ++n) {
        const unsigned t = __hip_atomic_load(&l.token[at], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        if (t == id) return static_cast<int>(at);
        if (t == kFree) return -1;
        at = (at + 1) & (SLOTS - 1);
    }
    at = kFree;
    return -1;
}

template <int SLOTS>
__device__ __forceinline__ unsigned hash_of(unsigned id) {
    return (id * 0x9e3779b1u) >> (32 - __builtin_ctz(SLOTS));
}

// The slot of `id`, put into the table if need be; -1: no room.
template <int SLOTS, bool ROUNDS>
__device__ __forceinline__ int take_slot(MergeLds<SLOTS, ROUNDS>& l, unsigned id, unsigned at) {
    for (;;) {
        const int s = find_slot(l, id, at);
        if (s >= 0) return s;
        if (at == kFree) return -1;
        if (ROUNDS && __hip_atomic_load(&l.count, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) >=
                          MergeLds<SLOTS, ROUNDS>::kFull)
            return -1;
        if (atomicCAS(&l.token[at], kFree, id) == kFree) {
            l.slot[atomicAdd(&l.count, 1u)] = static_cast<u16>(at);
            return static_cast<int>(at);
        }                                          // taken meanwhile, perhaps by this very token: look again
    }
}

__device__ __forceinline__ unsigned exponent_of(double p) { return static_cast<unsigned>(__double2hiint(p)) >> 20 & 2047u; }

// Waves a SIMD holds, so that the compiler keeps to their registers: as many as LDS lets in.
constexpr int merge_waves(int threads, int per) { return per >= 8 ? 4 : threads == 256 ? (per == 4 ? 5 : 8) : 6; }

// e^v of an fp32 value in fp64: 2^n times the Taylor series of e^r, |r| <= ln 2 / 2, whose first
// omitted term is below 2^-57; ln 2 in two parts keeps r exact to fp64.  About half the
// instructions of the library's, which has to take any fp64 argument.
__device__ __forceinline__ double exp_of(float v) {
    const double x = static_cast<double>(fminf(fmaxf(v, -1000.0f), 1000.0f));       // beyond: 0 and inf; NaN see below
    const double n = rint(x * 1.4426950408889634);
    const double r = fma(n, -2.3190468138462996e-17, fma(n, -0.6931471805599453, x));   // ln 2 in two parts
    double e = 1.0 / 6227020800.0;                                                  // 1 / 13!
    e = fma(e, r, 1.0 / 479001600.0);
    e = fma(e, r, 1.0 / 39916800.0);
    e = fma(e, r, 1.0 / 3628800.0);
    e = fma(e, r, 1.0 / 362880.0);
    e = fma(e, r, 1.0 / 40320.0);
    e = fma(e, r, 1.0 / 5040.0);
    e = fma(e, r, 1.0 / 720.0);
    e = fma(e, r, 1.0 / 120.0);
    e = fma(e, r, 1.0 / 24.0);
    e = fma(e, r, 1.0 / 6.0);
    e = fma(e, r, 0.5);
    e = fma(e, r, 1.0);
    e = fma(e, r, 1.0);
    return v != v ? __builtin_nan("") : ldexp(e, static_cast<int>(n));
}

// PER entries per thread
template <int THREADS, int PER, int SLOTS, bool ROUNDS>
__global__ __launch_bounds__(THREADS, merge_waves(THREADS, PER)) void merge_tops_kernel(const MergeArgs a) {
    using L = MergeLds<SLOTS, ROUNDS>;
    constexpr int kGroupsPer = (SLOTS + THREADS - 1) / THREADS;
    __shared__ L l;
    const int64_t row = a.row0 + blockIdx.x;
    const int tid = threadIdx.x;
    const int n = a.K * a.k;
    // entry e of a thread is i = tid + e * THREADS = (client, place) = (i / k, i % k)
    const int c0 = static_cast<int>((static_cast<uint64_t>(tid) * a.per_k) >> 32);
    const int dc = static_cast<int>((static_cast<uint64_t>(THREADS) * a.per_k) >> 32), dj = THREADS - dc * a.k;
    unsigned id[PER];
    float lp[PER];
    {
        int j = tid - c0 * a.k;
        if (a.near) {                              // one 32-bit offset serves both lists
            const int32_t* ip = a.ids + row * a.id_row;
            const float* lpp = a.lp + row * a.lp_row;
            const unsigned client = static_cast<unsigned>(a.id_client), step = dc * client + dj, wrapped = client - a.k;
            unsigned off = c0 * client + j;
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const bool in = tid + e * THREADS < n;
                id[e] = in ? static_cast<unsigned>(ip[off]) : kFree;
                lp[e] = in ? lpp[off] : 0.0f;
                j += dj;
                const bool wrap = j >= a.k;
                j -= wrap ? a.k : 0;
                off += step + (wrap ? wrapped : 0);
            }
        } else {
            const int32_t* ip = a.ids + row * a.id_row + c0 * a.id_client + j;
            const float* lpp = a.lp + row * a.lp_row + c0 * a.lp_client + j;
            const int64_t id_step = dc * a.id_client + dj, id_wrap = a.id_client - a.k;
            const int64_t lp_step = dc * a.lp_client + dj, lp_wrap = a.lp_client - a.k;
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const bool in = tid + e * THREADS < n;
                id[e] = in ? static_cast<unsigned>(*ip) : kFree;
                lp[e] = in ? *lpp : 0.0f;
                j += dj;
                const bool wrap = j >= a.k;
                j -= wrap ? a.k : 0;
                ip += id_step + (wrap ? id_wrap : 0);
                lpp += lp_step + (wrap ? lp_wrap : 0);
            }
        }
    }
    for (int c = tid; c < a.K; c += THREADS) {
        l.share[c] = a.w[c] * static_cast<double>(a.unit ? a.unit[c * a.unit_client + row * a.unit_row] : 1.0f);
        l.answered[c] = 0;
    }
    for (int i = tid; i < SLOTS; i += THREADS) {
        l.token[i] = kFree;
        l.peak[i] = 0;
        l.sum[i] = 0;
    }
    if (tid == 0) l.count = l.open = 0;

    __syncthreads();
    // at[e]: the entry's id while it waits for a slot, kSlot + its slot, kFree: absent or done
    constexpr unsigned kSlot = 1u << 31;
    unsigned (&at)[PER] = id;
    double p[PER];
    {
        int c = c0, j = tid - c0 * a.k;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            double share = 0.0;
            if (static_cast<int>(at[e]) >= 0) share = l.share[c];      // entries past the end are absent
            p[e] = share * exp_of(lp[e]);
            if (share > 0.0) l.answered[c] = 1;
            else at[e] = kFree;
            j += dj;
            const bool wrap = j >= a.k;
            j -= wrap ? a.k : 0;
            c += dc + (wrap ? 1 : 0);
        }
    }
    int kept = 0;
    for (bool more = true; more;) {
        // tokens into the table: the first entries bring most of them, the others mostly find theirs
        // at the first look, and those looks are on their way together
        bool waiting = false;
        unsigned seen[PER];
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            if (e == 1) {
#pragma unroll
                for (int o = 1; o < PER; ++o)
                    seen[o] = __hip_atomic_load(&l.token[hash_of<SLOTS>(at[o])], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            }
            if (static_cast<int>(at[e]) < 0) continue;
            const unsigned first = hash_of<SLOTS>(at[e]);
            const int s = e && seen[e] == at[e] ? static_cast<int>(first) : take_slot(l, at[e], first);
            if (s >= 0) {
                at[e] = kSlot + s;
                atomicMax(&l.peak[s], exponent_of(p[e]));
            } else {
                waiting = true;
            }
        }
        if (ROUNDS && waiting) l.open = 1;
        __syncthreads();
        more = ROUNDS && l.open != 0;
        const int groups = static_cast<int>(l.count);
        if (more) {
            // entries that found no room: their token may have come in through another entry
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                if (static_cast<int>(at[e]) < 0) continue;
                unsigned look = hash_of<SLOTS>(at[e]);
                const int s = find_slot(l, at[e], look);
                if (s < 0) continue;
                at[e] = kSlot + s;
                atomicMax(&l.peak[s], exponent_of(p[e]));
            }
            __syncthreads();
        }
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            if (static_cast<int>(at[e]) >= 0 || at[e] == kFree) continue;
            const unsigned s = at[e] - kSlot, x = l.peak[s];
            unsigned long long q;
            if (x == kExpInf) {                    // counts of NaN and of infinities
                q = p[e] != p[e] ? 1ull << 32 : p[e] > 1.7976931348623157e308 ? 1ull : 0ull;
            } else {
                // 2^51 above the peak's binade; adding 2^52 leaves the whole number in the low bits
                const double scaled = ldexp(p[e], 51 + 1022 - static_cast<int>(x ? x : 1));
                q = static_cast<unsigned long long>(__double_as_longlong(scaled + 4503599627370496.0)) & 0xfffffffffffffull;
            }
            atomicAdd(reinterpret_cast<unsigned long long*>(&l.sum[s]), q);
            at[e] = kFree;
        }
        __syncthreads();
        // the groups' values, moved together; behind them the list so far
        uint64_t key[kGroupsPer];
        unsigned name[kGroupsPer];
#pragma unroll
        for (int e = 0; e < kGroupsPer; ++e) {
            const int g = tid + e * THREADS;
            key[e] = 0;
            name[e] = kFree;
            if (g < groups) {
                const int s = l.slot[g];
                const unsigned x = l.peak[s];
                const uint64_t sum = l.sum[s];
                name[e] = l.token[s];
                const double whole = x && !sum ? 0x1p64 : static_cast<double>(sum);
                const double v = x == kExpInf ? (sum >> 32 ? __builtin_nan("") : __builtin_inf())
                                              : ldexp(whole, static_cast<int>(x ? x : 1) - 1022 - 51);
                key[e] = v != v ? 0x7ff8000000000000ull : static_cast<uint64_t>(__double_as_longlong(v));
            }
        }
        __syncthreads();
        // of many, only what reaches a bound that `top` of the threads' best reach
        unsigned least = 0;
        if (groups > 96 && groups >= 2 * a.top && a.top < THREADS / 2) {
            unsigned best = 0;
#pragma unroll
            for (int e = 0; e < kGroupsPer; ++e) {
                const unsigned hi = name[e] != kFree ? static_cast<unsigned>(key[e] >> 32) + 1 : 0;
                best = hi > best ? hi : best;
            }
            l.peak[tid] = best;
            __syncthreads();
            if (tid < kWave) {
                unsigned v[THREADS / kWave];
#pragma unroll
                for (int i = 0; i < THREADS / kWave; ++i) v[i] = l.peak[i * kWave + tid];
                bool exact;
                const unsigned nth = wave_nth(v, a.top, exact);
                if (tid == 0) l.bound = nth;
            }
            if (tid == 0) l.left = 0;
            __syncthreads();
            least = l.bound;
        }
        int total = groups;
        if (least) {
#pragma unroll
            for (int e = 0; e < kGroupsPer; ++e) {
                const bool in = name[e] != kFree && static_cast<unsigned>(key[e] >> 32) + 1 >= least;
                const uint64_t m = __ballot(in);
                unsigned base = 0;
                if (m && tid % kWave == 0) base = atomicAdd(&l.left, static_cast<unsigned>(__popcll(m)));
                base = __builtin_amdgcn_readfirstlane(base);
                if (in) {
                    l.sum[base + lanes_below(m)] = key[e];
                    l.token[base + lanes_below(m)] = name[e];
                }
            }
            __syncthreads();
            total = static_cast<int>(l.left);
        } else {
#pragma unroll
            for (int e = 0; e < kGroupsPer; ++e) {
                const int g = tid + e * THREADS;
                if (g < groups) {
                    l.sum[g] = key[e];
                    l.token[g] = name[e];
                }
            }
        }
        if (ROUNDS)
            for (int j = tid; j < kept; j += THREADS) {
                l.sum[total + j] = l.list_key[j];
                l.token[total + j] = l.list_id[j];
            }
        total += kept;
        if (tid < 8) {                             // ranks below everything
            l.sum[total + tid] = 0;
            l.token[total + tid] = kFree;
        }
        __syncthreads();
        kept = total < a.top ? total : a.top;
        // ranks: `share` neighbouring threads count for one value
        int share = 1;
        while (share < 16 && total * share * 2 <= THREADS) share *= 2;
        for (int g0 = 0; g0 < total; g0 += THREADS / share) {
            const int g = g0 + tid / share, part = tid % share;
            const uint64_t mine = l.sum[g < total ? g : total];
            const unsigned me = l.token[g < total ? g : total];
            int rank = 0;
            for (int o = part * 8; o < total; o += share * 8) {
                uint64_t k8[8];
                unsigned i8[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    k8[q] = l.sum[o + q];
                    i8[q] = l.token[o + q];
                }
#pragma unroll
                for (int q = 0; q < 8; ++q) rank += before(k8[q], i8[q], mine, me);
            }
            for (int d = 1; d < share; d *= 2) rank += __shfl_xor(rank, d);
            if (part || g >= total || rank >= a.top) continue;
            if (more) {
                l.list_key[rank] = mine;
                l.list_id[rank] = me;
            } else {
                a.out_ids[row * a.top + rank] = static_cast<int32_t>(me);
                l.best[rank] = mine;
            }
        }
        if (more) {
            __syncthreads();
            for (int i = tid; i < SLOTS; i += THREADS) {
                l.token[i] = kFree;
                l.peak[i] = 0;
                l.sum[i] = 0;
            }
            if (tid == 0) l.count = l.open = 0;
            __syncthreads();
        }
    }
    if (tid < kWave) {
        double t = 0.0;
        for (int c = tid; c < a.K; c += kWave)
            if (l.answered[c]) t += l.share[c];
        for (int d = kWave / 2; d > 0; d >>= 1) t += __shfl_xor(t, d);
        if (tid == 0) l.total = t;
    }
    __syncthreads();
    const double total = l.total;
    for (int j = tid; j < a.top; j += THREADS) {
        float out = -kInf;
        if (j < kept)
            out = static_cast<float>(log(__longlong_as_double(static_cast<long long>(l.best[j])) / total));
        else
            a.out_ids[row * a.top + j] = -1;
        a.out_lp[row * a.top + j] = out;
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
    if (x->vocab > FA_VOCAB_MAX || (x->inner && x->outer > INT32_MAX / x->inner)) return FA_ERR_TOO_LARGE;
    if (x->outer * x->inner && !x->data) return FA_ERR_INVALID;
    if (!aligned_to(x->data, elem_size(x->dtype))) return FA_ERR_ALIGN;
    return FA_OK;
}

int check_teacher(const fa_teacher* t, int64_t rows) {
    if (!t || t->k < 1 || t->k > FA_TOP_MAX) return FA_ERR_INVALID;
    if (rows && (!t->ids || !t->logprobs)) return FA_ERR_INVALID;
    if (t->id_stride < 0 || t->lp_stride < 0) return FA_ERR_INVALID;
    if (!(t->temperature >= 1e-3) || !(t->temperature <= 1e3)) return FA_ERR_INVALID;
    return FA_OK;
}

Rows rows_of(const fa_logits* x) { return {x->inner, x->stride_outer, x->stride_inner}; }

Scale scale_of(double temperature) {
    Scale s;
    s.k = static_cast<float>(1.44269504088896340736 / temperature);
    s.inv_k = static_cast<float>(1.0 / static_cast<double>(s.k));
    s.inv_tau = static_cast<float>(1.0 / temperature);
    return s;
}

DistillArgs distill_args(const fa_logits* x, const fa_teacher* t) {
    DistillArgs a = {};
    a.x = x->data;
    a.rows = rows_of(x);
    a.vocab = x->vocab;
    a.t = {t->ids, t->logprobs, t->id_stride, t->lp_stride, t->k, static_cast<float>(t->temperature), t->row_weight};
    a.scale = scale_of(t->temperature);
    return a;
}

// Few long rows: one block of 1024 threads each; else 256.
bool wide_blocks(int64_t rows, int vocab) { return rows < 512 && vocab >= 8192; }

constexpr int64_t kMemoryCache = 256ll << 20;      // the last-level cache of the memory side

int64_t row_bytes(const fa_logits* x) { return static_cast<int64_t>(x->vocab) * elem_size(x->dtype); }

// A launch counts its threads in 32 bits: 2^21 rows of up to 1024 threads at a time.
constexpr int64_t kRowsPerLaunch = 1 << 21;

template <class Args, class Launch>
void for_rows(int64_t rows, Args a, Launch launch) {
    for (a.row0 = 0; a.row0 < rows; a.row0 += kRowsPerLaunch) {
        const int64_t left = rows - a.row0;
        launch(static_cast<unsigned>(left < kRowsPerLaunch ? left : kRowsPerLaunch), a);
    }
}

template <int DT, int THREADS, bool LOSS, bool GRAD, bool LAST>
void launch_distill_t(int64_t rows, int parts, const DistillArgs& args, hipStream_t st) {
    for_rows(rows, args, [&](unsigned n, const DistillArgs& a) {
        hipLaunchKernelGGL((distill_kernel<DT, THREADS, LOSS, GRAD, LAST>), dim3(n, static_cast<unsigned>(parts)),
                           dim3(THREADS), 0, st, a);
    });
}

template <int DT>
void launch_loss(const fa_logits* x, const DistillArgs& a, hipStream_t st) {
    const int64_t rows = x->outer * x->inner;
    if (x->vocab <= 4096) launch_distill_t<DT, 64, true, false, false>(rows, 1, a, st);
    else if (wide_blocks(rows, x->vocab)) launch_distill_t<DT, 1024, true, false, false>(rows, 1, a, st);
    else launch_distill_t<DT, 256, true, false, false>(rows, 1, a, st);
}

// A gradient alone has nothing to sum, so that a row may be cut when there are few.
template <int DT>
void launch_grad(const fa_logits* x, const DistillArgs& a, hipStream_t st) {
    const int64_t rows = x->outer * x->inner;
    int parts = 1;
    while (parts < 64 && rows * parts < 2048 && x->vocab / parts >= 8192) parts *= 2;
    if (x->vocab <= 4096) launch_distill_t<DT, 64, false, true, false>(rows, 1, a, st);
    else launch_distill_t<DT, 256, false, true, false>(rows, parts, a, st);
}

template <int DT, int NV>
void launch_step_t(int64_t rows, const DistillArgs& args, hipStream_t st) {
    for_rows(rows, args, [&](unsigned n, const DistillArgs& a) {
        hipLaunchKernelGGL((distill_step_kernel<DT, kWave, NV>), dim3(n), dim3(kWave), 0, st, a);
    });
}

template <int DT>
void launch_step(const fa_logits* x, const DistillArgs& a, hipStream_t st) {
    const int64_t rows = x->outer * x->inner;
    const int nvec = x->vocab / Vec<DT>::N;
    if (nvec <= kWave * 4) return launch_step_t<DT, 4>(rows, a, st);
    if (nvec <= kWave * 8) return launch_step_t<DT, 8>(rows, a, st);
    // Few long rows fill the chip only in parts, at the price of a second launch: 1 x 128000 bf16 13.4 us
    // in parts, 21.7 whole; 128 x 128000 bf16 22.4 and 25.5; 4 x 1000000 fp32 17 and 199.  At 200 KB a
    // row the GPU gains as much as the launch costs the host (1 x 50261 fp32: 12.0 and 13.8, called one
    // by one 16.0 and 13.7).  Not where the gradient goes over the logits: a block reads the teacher's
    // tokens in other parts, whose blocks may have written them.
    if (a.partial && a.grad != a.x && rows <= FA_DISTILL_WS_ROWS && row_bytes(x) >= FA_DISTILL_WS_BYTES) {
        int parts = 2;
        while (parts < kWave && rows * parts * 2 <= FA_DISTILL_WS_FLOATS / 2 && nvec / (parts * 2) >= 1024) parts *= 2;
        hipLaunchKernelGGL((distill_parts_kernel<DT, 256>), dim3(static_cast<unsigned>(rows), parts), dim3(256), 0, st, a);
        return launch_distill_t<DT, 256, true, true, false>(rows, parts, a, st);
    }
    const bool last = rows * row_bytes(x) > kMemoryCache;
    if (wide_blocks(rows, x->vocab) || row_bytes(x) > (128 << 10)) {
        if (last) launch_distill_t<DT, 1024, true, true, true>(rows, 1, a, st);
        else launch_distill_t<DT, 1024, true, true, false>(rows, 1, a, st);
    } else {
        if (last) launch_distill_t<DT, 256, true, true, true>(rows, 1, a, st);
        else launch_distill_t<DT, 256, true, true, false>(rows, 1, a, st);
    }
}

template <int DT, int THREADS>
void launch_scores_t(const fa_logits* x, const ScoreArgs& args, hipStream_t st) {
    for_rows(x->outer * x->inner, args, [&](unsigned n, const ScoreArgs& a) {
        if (a.top)
            hipLaunchKernelGGL((token_scores_kernel<DT, THREADS, true>), dim3(n), dim3(THREADS), 0, st, a);
        else
            hipLaunchKernelGGL((token_scores_kernel<DT, THREADS, false>), dim3(n), dim3(THREADS), 0, st, a);
    });
}

template <int DT>
void launch_scores(const fa_logits* x, const ScoreArgs& a, hipStream_t st) {
    // a short row is one wave's: no barriers (8192 x 1000 fp32, top 64: 27 us, 44 with 256 threads)
    if (x->vocab <= 4096 && a.top <= kWave)
        launch_scores_t<DT, kWave>(x, a, st);
    else if (wide_blocks(x->outer * x->inner, x->vocab))
        launch_scores_t<DT, 1024>(x, a, st);
    else
        launch_scores_t<DT, 256>(x, a, st);
}

hipStream_t as_stream(fa_stream_t s) { return reinterpret_cast<hipStream_t>(s); }

template <int THREADS, int PER, int SLOTS, bool ROUNDS>
void launch_merge_t(const MergeArgs& args, int64_t rows, hipStream_t st) {
    for_rows(rows, args, [&](unsigned n, const MergeArgs& a) {
        hipLaunchKernelGGL((merge_tops_kernel<THREADS, PER, SLOTS, ROUNDS>), dim3(n), dim3(THREADS), 0, st, a);
    });
}

// Threads for at most 16 entries each; a table that holds every token of a short list at once.
int launch_merge(const MergeArgs& a, int64_t rows, hipStream_t st) {
    const int n = a.K * a.k;
    if (n <= 64) launch_merge_t<64, 1, 128, false>(a, rows, st);
    else if (n <= 128) launch_merge_t<64, 2, 256, false>(a, rows, st);
    else if (n <= 256) launch_merge_t<128, 2, 512, false>(a, rows, st);
    else if (n <= 512) launch_merge_t<256, 2, 1024, false>(a, rows, st);
    else if (n <= 1024) launch_merge_t<256, 4, 1024, true>(a, rows, st);
    else if (n <= 2048) launch_merge_t<512, 4, 1024, true>(a, rows, st);
    else if (n <= 4096) launch_merge_t<512, 8, 1024, true>(a, rows, st);
    else launch_merge_t<512, 16, 1024, true>(a, rows, st);
    return hip_code(hipGetLastError());
}

}  // namespace

extern "C" {

int fa_token_scores(const fa_logits* x, const int64_t* targets, int64_t ignore_index, int top, float* logprob,
                    float* entropy, float* lse, int32_t* top_ids, float* top_logprobs, fa_stream_t stream) {
    const int rc = check_logits(x);
    if (rc != FA_OK) return rc;
    if (top < 0 || top > FA_SCORES_TOP_MAX || top > x->vocab) return FA_ERR_INVALID;
    const int64_t rows = x->outer * x->inner;
    if (rows == 0) return FA_OK;
    if (!entropy || !lse || (targets && !logprob) || (top && (!top_ids || !top_logprobs))) return FA_ERR_INVALID;
    const ScoreArgs a = {x->data, rows_of(x), x->vocab, top, targets, ignore_index, logprob, entropy, lse,
                         top_logprobs, top_ids, scale_of(1.0), 0};
    switch (x->dtype) {
        case FA_LOGITS_F32: launch_scores<FA_LOGITS_F32>(x, a, as_stream(stream)); break;
        case FA_LOGITS_BF16: launch_scores<FA_LOGITS_BF16>(x, a, as_stream(stream)); break;
        default: launch_scores<FA_LOGITS_F16>(x, a, as_stream(stream));
    }
    return hip_code(hipGetLastError());
}

int fa_distill_loss(const fa_logits* x, const fa_teacher* t, float* loss, float* stat, fa_stream_t stream) {
    int rc = check_logits(x);
    if (rc == FA_OK) rc = check_teacher(t, x->outer * x->inner);
    if (rc != FA_OK) return rc;
    if (x->outer * x->inner == 0) return FA_OK;
    if (!loss || !stat) return FA_ERR_INVALID;
    DistillArgs a = distill_args(x, t);
    a.loss = loss;
    a.stat = stat;
    switch (x->dtype) {
        case FA_LOGITS_F32: launch_loss<FA_LOGITS_F32>(x, a, as_stream(stream)); break;
        case FA_LOGITS_BF16: launch_loss<FA_LOGITS_BF16>(x, a, as_stream(stream)); break;
        default: launch_loss<FA_LOGITS_F16>(x, a, as_stream(stream));
    }
    return hip_code(hipGetLastError());
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
    switch (x->dtype) {
        case FA_LOGITS_F32: launch_grad<FA_LOGITS_F32>(x, a, as_stream(stream)); break;
        case FA_LOGITS_BF16: launch_grad<FA_LOGITS_BF16>(x, a, as_stream(stream)); break;
        default: launch_grad<FA_LOGITS_F16>(x, a, as_stream(stream));
    }
    return hip_code(hipGetLastError());
}

int fa_distill_loss_grad(const fa_logits* x, const fa_teacher* t, float* loss, void* grad, int64_t grad_stride_outer,
                         int64_t grad_stride_inner, float* ws, fa_stream_t stream) {
    int rc = check_logits(x);
    if (rc == FA_OK) rc = check_teacher(t, x->outer * x->inner);
    if (rc != FA_OK) return rc;
    if (x->outer * x->inner == 0) return FA_OK;
    if (!loss || !grad || grad_stride_outer < 0 || grad_stride_inner < 0) return FA_ERR_INVALID;
    if (!aligned_to(grad, elem_size(x->dtype)) || !aligned_to(ws, sizeof(float))) return FA_ERR_ALIGN;
    DistillArgs a = distill_args(x, t);
    a.loss = loss;
    a.partial = ws;
    a.grad = grad;
    a.grad_rows = {x->inner, grad_stride_outer, grad_stride_inner};
    switch (x->dtype) {
        case FA_LOGITS_F32: launch_step<FA_LOGITS_F32>(x, a, as_stream(stream)); break;
        case FA_LOGITS_BF16: launch_step<FA_LOGITS_BF16>(x, a, as_stream(stream)); break;
        default: launch_step<FA_LOGITS_F16>(x, a, as_stream(stream));
    }
    return hip_code(hipGetLastError());
}

int fa_merge_tops(const fa_tops* in, const double* w, int K, int64_t rows, int top, int32_t* out_ids,
                  float* out_logprobs, fa_stream_t stream) {
    if (!in || !w || K < 1 || K > FA_MERGE_CLIENTS || rows < 0 || in->k < 1 || in->k > FA_TOP_MAX) return FA_ERR_INVALID;
    if (static_cast<int64_t>(K) * in->k > FA_MERGE_ENTRIES || rows > INT32_MAX) return FA_ERR_TOO_LARGE;
    if (top < 1 || top > K * in->k || top > FA_TOP_MAX) return FA_ERR_INVALID;
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
    a.near = in->id_client == in->lp_client && in->id_client < (1 << 30) / K;
    a.per_k = ((1ull << 32) + in->k - 1) / in->k;
    a.out_ids = out_ids;
    a.out_lp = out_logprobs;
    // Only the weights' ratios count: by a power of two (exact) the largest is put into [1/2, 1), so that
    // products and sums stay within fp64.  A weight that is nothing beside it still answers.
    double most = 0.0;
    for (int c = 0; c < K; ++c) most = w[c] > most ? w[c] : most;
    int power = 0;
    frexp(most, &power);
    for (int c = 0; c < K; ++c) {
        a.w[c] = ldexp(w[c], -power);
        if (w[c] > 0.0 && a.w[c] == 0.0) a.w[c] = 4.9406564584124654e-324;
    }
    return launch_merge(a, rows, as_stream(stream));
}

}  // extern "C"
