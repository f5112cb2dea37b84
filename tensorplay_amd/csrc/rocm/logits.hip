// gfx950 losses over the logits of a language model, behind tpr_token_logprob(),
// its backward, tpr_policy_loss() and tpr_preference_loss().
//
// A row x of V logits enters through two numbers, its largest logit m and
// log s = log sum exp((x - m) / T):
//   logp = (x_t - m) / T - log s,     softmax_v = exp((x_v - m) / T) / s.
// One pass over a row gives both (the running maximum and sum of a softmax); the
// backward pass reads the row once more and writes its gradient.
//
// Where one token is all but certain, s is 1 plus a rest that 32 bits would round
// away, and logp is minus that rest: so the element that sets the maximum is counted (n),
// with the equal ones that arrive with it, and only the others summed (r).  Equal ones
// that arrive later are summed, which costs no digits: s - 1 is then 1 and more.  What is
// kept of a row is m and s - 1 = n - 1 + r; log s = log1p(s - 1) has the rest's digits, and
// 1 - softmax at the target, the gradient's largest element, is -expm1(logp).
//
// Costs: a row is read once for its statistics (memory-bound from a few hundred rows on:
// [4096, 151936] bfloat16 211 us, 5.9 TB/s; [2048, 50261] float16 38 us, 5.4 TB/s), read
// and written for its gradient (408 us, 6.1 TB/s; 64 us, 6.5 TB/s), or read and written
// once for both
// (k_policy_rows).  A 2 GiB copy by torch moves 4.9 TB/s on this card, a fill writes 6.9.
//
// exp((x - m) / T) is 2^(x k - m k), k = log2(e) / T, one or two fused products.  k is
// split into k1, its 24 bits rounded down, and the rest k2 > 0: alone k1 would shift
// every exponent by up to 6e-8 of itself, 1e-6 of the sum where logits spread over 20.
// (k2 > 0: x = -inf then stays -inf.)

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>

#include "common.h"
#include "elem.h"
#include "ticket.h"

namespace tpr {
namespace {

constexpr int kLgBlock = 256;
constexpr float kLowest = -3.40282347e38f;  // the first maximum: finite, so that x - m never is NaN for x = -inf

// The state of a part of a row: maximum, how many elements equal it of those that were
// counted, and the sum of exp((x - m) / T) over the others.  Nothing seen but -inf: n = r = 0.
struct RowPart {
    float m, n;
    double r;
};

// m k1 beyond this is too coarse a reference for the exponents (its last bit 2^-4): they are
// then formed from x - m, which is what such magnitudes leave of any difference.
constexpr float kFar = 1048576.0f;

// log2(e) / T, whole and split
struct Scale {
    double k;
    float k1, k2;
};

__device__ __forceinline__ float ex2(float d) { return __builtin_amdgcn_exp2f(d); }

__device__ __forceinline__ RowPart merge(const RowPart& a, const RowPart& b, float k) {
    const float M = fmaxf(a.m, b.m);
    const float sa = ex2((a.m - M) * k), sb = ex2((b.m - M) * k);  // 1 for the larger
    RowPart c;
    c.m = M;
    c.n = (a.m == M ? a.n : 0.0f) + (b.m == M ? b.n : 0.0f);
    c.r = (a.m == M ? a.r : (a.n + a.r) * sa) + (b.m == M ? b.r : (b.n + b.r) * sb);
    return c;
}

// The parts of n neighbouring lanes, n a power of two up to the wave, in each of them
__device__ __forceinline__ RowPart merge_lanes(RowPart p, int n, float k) {
    for (int o = 1; o < n; o <<= 1) {
        const RowPart q{__shfl_xor(p.m, o, kWave), __shfl_xor(p.n, o, kWave), __shfl_xor(p.r, o, kWave)};
        p = merge(p, q, k);
    }
    return p;
}

struct RowStat {
    float m, rest;   // largest logit, s - 1 (NaN: the row is)
};

__device__ __forceinline__ RowStat finish(const RowPart& p) {
    const double rest = (double)(p.n - 1.0f) + p.r;
    RowStat s;
    s.m = p.m;
    // nothing above -inf (rest = -1), or +inf among them: NaN, as softmax has it
    s.rest = p.m == INFINITY || rest == -1.0 ? NAN : (float)rest;
    return s;
}

// log-probability of the logit xt
__device__ __forceinline__ double logp_of(float xt, const RowStat& s, double inv_t) {
    return ((double)xt - (double)s.m) * inv_t - log1p((double)s.rest);
}

// One wave's running state over elements that its lanes hold: m and mk = m k1 are the
// wave's, n and r each lane's.  While no lane sees an element above m, an element costs
// two fused products, an exponential and an addition; r is in 64 bits, one addition a
// batch.
struct WaveScan {
    float m = kLowest, n = 0.0f;
    float base = kLowest, mk = 0.0f;   // (x - base) k - mk is (x - m) k, in one of two forms
    bool far = true;                   // m k1 is past the range of the fused one
    double r = 0.0;

    // TOP: elements that equal m are counted: in the batch that has set m, and in every
    // batch while m is far
    template <int N, bool TOP>
    __device__ __forceinline__ void terms(const float (&v)[N], const Scale& k) {
        float s[4] = {};
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float d = TOP ? v[e] - base : v[e];
            const float t = ex2(fmaf(d, k.k2, fmaf(d, k.k1, -mk)));
            if constexpr (TOP) {
                n += v[e] == m ? 1.0f : 0.0f;
                s[e % 4] += v[e] == m ? 0.0f : t;
            } else {
                s[e % 4] += t;
            }
        }
        r += (double)((s[0] + s[1]) + (s[2] + s[3]));
    }

    // 2^(mk - m k): what the terms so far, relative to the rounded mk, have to be
    // multiplied by to be relative to m
    __device__ __forceinline__ float exact(const Scale& k) const {
        const float d = m - base;
        return ex2(-fmaf(d, k.k2, fmaf(d, k.k1, -mk)));
    }

    template <int N>
    __device__ __forceinline__ void add(const float (&v)[N], const Scale& k) {
        float cm = v[0];
#pragma unroll
        for (int e = 1; e < N; ++e) cm = fmaxf(cm, v[e]);
        if (__any(cm > m)) {
            // What is carried over becomes a term like those that follow, relative to the new
            // mk and not to m: part() takes the rounding of mk out of all of them at once.
            const float was = exact(k), d0 = m;
            m = wave_max_f(fmaxf(cm, m));
            far = !(fabsf(m * k.k1) < kFar);
            base = far ? m : 0.0f;
            mk = far ? 0.0f : m * k.k1;
            const float d = d0 - base, down = ex2(fmaf(d, k.k2, fmaf(d, k.k1, -mk)));
            r = fma(r, (double)(was * down), (double)(n * down));
            n = 0.0f;
            terms<N, true>(v, k);
        } else if (far) {
            terms<N, true>(v, k);
        } else {
            terms<N, false>(v, k);
        }
    }

    // the wave's part, in every lane
    __device__ __forceinline__ RowPart part(const Scale& k) const {
        RowPart p;
        p.m = m;
        p.n = wave_sum_f(n);
        p.r = wave_sum_d(r) * (double)exact(k);
        return p;
    }
};

struct LogitArgs {
    const void* x;
    const long long* target;
    long long rows, vocab, stride, ignore;
    long long chunk;   // elements of a row per workgroup, a multiple of 8
    int S;             // workgroups per row
    Scale k;
    double inv_t;
    const float* weight;  // rows of weight 0 are skipped (may be null)
    float* logp;
    double* logp64;    // the same unrounded, for the losses (may be null)
    RowStat* lse;
    RowPart* part;     // S > 1: [rows, S]
    unsigned* tickets; // S > 1: counters of the rows, or null: k_row_join joins the parts
};

// A row's target, read before the row: its logit is wanted at the end, when nothing
// else is under way to hide the read.
struct Target {
    long long t;
    bool skip, known;   // the row does not count; the target is in the vocabulary
    float x;
};

template <class T>
__device__ __forceinline__ Target target_of(const LogitArgs& a, long long row) {
    Target r;
    r.t = a.target[row];
    r.skip = r.t == a.ignore || (a.weight && a.weight[row] == 0.0f);
    r.known = r.t >= 0 && r.t < a.vocab;
    r.x = r.known && !r.skip ? (float)static_cast<const T*>(a.x)[row * a.stride + r.t] : 0.0f;
    return r;
}

__device__ __forceinline__ void put_row(const LogitArgs& a, long long row, const Target& t, RowStat s) {
    double lp = 0.0;
    if (t.skip) {
        s.m = s.rest = 0.0f;
    } else if (!t.known) {
        s.m = s.rest = NAN;
        lp = NAN;
    } else {
        lp = logp_of(t.x, s, a.inv_t);
    }
    a.lse[row] = s;
    a.logp[row] = (float)lp;
    if (a.logp64) a.logp64[row] = lp;
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr int kBufWord3 = 0x00020000;  // raw buffer resource, 32-bit data (gfx9 family)

// A workgroup's waves take `len` elements at x into their states: 16 elements a thread
// at a time, the next 16 on their way meanwhile (64 registers, so that a CU holds 32
// waves).
template <class T, int NT>
__device__ __forceinline__ void scan(WaveScan& w, const T* x, int len, const Scale& k) {
    using V = typename Vec16<T>::type;
    constexpr int VN = Vec16<T>::N, U = 16 / VN, kStep = NT * VN * U;
    const int tid = threadIdx.x, whole = len / VN * VN;
    const __amdgpu_buffer_rsrc_t in =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(x), (short)0, whole * (int)sizeof(T), kBufWord3);
    auto load = [&](u32x4 (&r)[U], int b) {   // past the end: 0, without a read
#pragma unroll
        for (int j = 0; j < U; ++j)
            r[j] = __builtin_amdgcn_raw_buffer_load_b128(in, (b + (j * NT + tid) * VN) * (int)sizeof(T), 0, 0);
    };
    auto take = [&](const u32x4 (&r)[U], int b) {
        if (b + kStep <= whole) {
            float v[U * VN];
#pragma unroll
            for (int j = 0; j < U; ++j)
#pragma unroll
                for (int e = 0; e < VN; ++e) v[j * VN + e] = (float)__builtin_bit_cast(V, r[j])[e];
            w.add(v, k);
        } else {
#pragma unroll
            for (int j = 0; j < U; ++j) {
                if (b + j * NT * VN >= whole) break;
                const bool on = b + (j * NT + tid) * VN < whole;
                float v[VN];
#pragma unroll
                for (int e = 0; e < VN; ++e) v[e] = on ? (float)__builtin_bit_cast(V, r[j])[e] : -INFINITY;
                w.add(v, k);
            }
        }
    };
    u32x4 p[U], q[U];
    load(p, 0);
    if (whole < len && tid < kWave) {   // the elements past the last whole vector
        const float v[1] = {whole + tid < len ? (float)x[whole + tid] : -INFINITY};
        w.add(v, k);
    }
    for (int b = 0; b < whole; b += 2 * kStep) {
        load(q, b + kStep);
        take(p, b);
        load(p, b + 2 * kStep);
        if (b + kStep < whole) take(q, b + kStep);
    }
}

// One workgroup per row (S == 1) or per chunk of a row, each reading it once.  A
// workgroup of 256 keeps eight rows on a CU, whose ends (joining lanes, a 64-bit
// logarithm, 2 us) overlap with the others' reads.
template <class T>
__global__ __launch_bounds__(kLgBlock) void k_row_stats(LogitArgs a) {
    __shared__ RowPart sh[kLgBlock / kWave];
    const long long row = blockIdx.x / a.S;
    const int chunk = blockIdx.x - row * a.S;
    const Target t = target_of<T>(a, row);
    const long long lo = chunk * a.chunk;
    const int len = t.skip ? 0 : (int)min(a.chunk, a.vocab - lo);
    WaveScan w;
    scan<T, kLgBlock>(w, static_cast<const T*>(a.x) + row * a.stride + lo, max(len, 0), a.k);
    RowPart p = w.part(a.k);
    if (__lane_id() == 0) sh[threadIdx.x / kWave] = p;
    __syncthreads();
    if (threadIdx.x >= kWave) return;
#pragma unroll
    for (int i = 1; i < kLgBlock / kWave; ++i) p = merge(p, sh[i], a.k.k1);
    if (a.S > 1) {   // one wave is left, whose lanes all hold the part
        RowPart* parts = a.part + row * a.S;
        if (!a.tickets) {
            if (__lane_id() == 0) parts[chunk] = p;
            return;
        }
        bool last = false;
        if (__lane_id() == 0) {
            publish_state(parts + chunk, p);
            last = last_of<false>(ticket_of(a.tickets, row), a.S, chunk);
        }
        if (!__any(last)) return;
        p = (int)__lane_id() < a.S ? fetch_state(parts + __lane_id()) : RowPart{kLowest, 0.0f, 0.0};
        p = merge_lanes(p, a.S, a.k.k1);
    }
    if (__lane_id() == 0) put_row(a, row, t, finish(p));
}

// Joins the S parts of each row: S lanes a row, S a power of two up to the wave.
template <class T>
__global__ __launch_bounds__(kLgBlock) void k_row_join(LogitArgs a) {
    const long long i = (long long)blockIdx.x * kLgBlock + threadIdx.x;
    const bool in = i < a.rows * a.S;
    const RowPart p = merge_lanes(in ? a.part[i] : RowPart{kLowest, 0.0f, 0.0}, a.S, a.k.k1);
    if (!in || i % a.S != 0) return;
    const long long row = i / a.S;
    put_row(a, row, target_of<T>(a, row), finish(p));
}

// ---- the logits' gradient -------------------------------------------------------
struct GradArgs {
    const void* x;
    const long long* target;
    const float* coef;
    const float* scale;
    const RowStat* lse;
    void* grad;
    long long vocab, stride, ignore;
    long long row0;
    int S;             // workgroups per row
    Scale k;
    double inv_t;
};

// -c / s exp((x - m) / T) for the elements of a row, c = coefficient / T; the target's is
// c (1 - softmax) = -c expm1(logp).  Half precision needs no k2: its own rounding is
// 2^-11 and more.
template <class T>
struct RowGrad {
    static constexpr bool kSplit = sizeof(T) == 4;
    float base, mk, c, cs;
    __device__ __forceinline__ RowGrad(const RowStat& s, float coef, const Scale& k) {
        const bool far = !(fabsf(s.m * k.k1) < kFar);
        base = far ? s.m : 0.0f;
        mk = far ? 0.0f : s.m * k.k1;
        c = coef;
        const float d = s.m - base, z = fmaf(d, k.k1, -mk);   // the rounding of mk, taken out again
        cs = (0.0f - c) / (1.0f + s.rest) * ex2(-(kSplit ? fmaf(d, k.k2, z) : z));
    }
    __device__ __forceinline__ float value(float x, const Scale& k) const {
        const float d = x - base, z = fmaf(d, k.k1, -mk);
        return cs * ex2(kSplit ? fmaf(d, k.k2, z) : z);
    }
    __device__ __forceinline__ float target(float x, const RowStat& s, double inv_t) const {
        return (float)(-(double)c * expm1(logp_of(x, s, inv_t)));
    }
};

// One workgroup per 1024 vectors of a row, read and written once: bound by memory.
// PASS: what passes the caches, 1 the stores, 2 the loads too.
template <class T, int PASS>
__global__ __launch_bounds__(kLgBlock) void k_logits_grad(GradArgs a) {
    constexpr int VN = Vec16<T>::N, U = 4;
    const long long row = a.row0 + blockIdx.x / a.S;
    const long long lo = (long long)(blockIdx.x % a.S) * (kLgBlock * VN * U);
    const long long t = a.target[row];
    const T* x = static_cast<const T*>(a.x) + row * a.stride + lo;
    T* g = static_cast<T*>(a.grad) + row * a.vocab + lo;
    const int len = (int)min((long long)kLgBlock * VN * U, a.vocab - lo);
    const float c = t == a.ignore ? 0.0f : a.coef[row];
    const RowStat s = a.lse[row];
    const RowGrad<T> f(s, (float)((double)(c * (a.scale ? a.scale[0] : 1.0f)) * a.inv_t), a.k);
    const int hit = t >= lo && t < lo + len ? (int)(t - lo) : -VN;   // the target's place in the chunk
#pragma unroll
    for (int j = 0; j < U; ++j) {
        const int at = (j * kLgBlock + threadIdx.x) * VN;
        if (at >= len) return;
        float v[VN];
        if (c == 0.0f) {
#pragma unroll
            for (int e = 0; e < VN; ++e) v[e] = 0.0f;
        } else {
            load_n<PASS == 2>(v, x + at, len - at, 0.0f);
#pragma unroll
            for (int e = 0; e < VN; ++e) v[e] = f.value(v[e], a.k);
            if (hit >= at && hit < at + VN) {
                const float z = f.target((float)x[hit], s, a.inv_t);
#pragma unroll
                for (int e = 0; e < VN; ++e) v[e] = hit - at == e ? z : v[e];
            }
        }
        store_n<PASS >= 1>(g + at, v, len - at);
    }
}

// ---- per-row part of the policy loss --------------------------------------------
struct PolicyTerms {
    double low, high, kl;   // bounds of the ratio, weight of the KL term
};
struct PolicyArgs {
    const long long* target;
    const double* logp;
    const float *old_logp, *advantage, *ref_logp, *weight;
    long long rows, ignore;
    PolicyTerms terms;
    float* coef;
    float* loss;
};

__device__ __forceinline__ double policy_weight(const PolicyArgs& a, long long i) {
    return a.target[i] == a.ignore ? 0.0 : a.weight ? (double)a.weight[i] : 1.0;
}

// dloss / dlp of a row of weight w / W, and the row's loss.  64 bits: the ratio may lie
// next to a border, and the KL estimate is a difference of near numbers.
__device__ __forceinline__ double policy_row(const PolicyTerms& a, float old_logp, float advantage, float ref_logp,
                                             double lp, double w, double& loss) {
    const double adv = advantage, r = exp(lp - (double)old_logp);
    const double s1 = r * adv, s2 = fmin(fmax(r, a.low), a.high) * adv;
    double l = s1 <= s2 ? -s1 : s1 > s2 ? -s2 : -s1 - s2;  // the last: NaN
    double c = s1 > s2 ? 0.0 : -s1;
    if (a.kl != 0.0) {
        const double d = (double)ref_logp - lp, e = expm1(d);
        l += a.kl * (e - d);
        c -= a.kl * e;
    }
    loss += w * l;
    return w * c;
}

// Sums over the rows' weights, and how many rows count: one workgroup's run of rows.
struct WeightPart {
    double w;
    long long live;
};

__device__ __forceinline__ WeightPart weight_part(const PolicyArgs& a, long long i) {
    const double w = i < a.rows ? policy_weight(a, i) : 0.0;
    return {w, w != 0.0};
}

template <int NT>
__device__ __forceinline__ WeightPart team_sum_w(WeightPart p, WeightPart* sh) {
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const WeightPart q = lane_xor(p, o);
        p = {p.w + q.w, p.live + q.live};
    }
    if (__lane_id() == 0) sh[threadIdx.x / kWave] = p;
    __syncthreads();
    p = sh[0];
#pragma unroll
    for (int i = 1; i < NT / kWave; ++i) p = {p.w + sh[i].w, p.live + sh[i].live};
    return p;
}

__global__ __launch_bounds__(kLgBlock) void k_weight_parts(PolicyArgs a, WeightPart* part, long long run) {
    __shared__ WeightPart sh[kLgBlock / kWave];
    const long long b = blockIdx.x * run, e = min(b + run, a.rows);
    WeightPart p{0.0, 0};
    for (long long i = b + threadIdx.x; i < e; i += kLgBlock) {
        const WeightPart q = weight_part(a, i);
        p = {p.w + q.w, p.live + q.live};
    }
    p = team_sum_w<kLgBlock>(p, sh);
    if (threadIdx.x == 0) part[blockIdx.x] = p;
}

// One workgroup (1024 rows and fewer): first the weights' sum, then each row.
constexpr int kOneBlock = 1024;
__global__ __launch_bounds__(kOneBlock) void k_policy(PolicyArgs a) {
    __shared__ double sh[2][kOneBlock / kWave];
    const long long i = threadIdx.x;
    const double w = i < a.rows ? policy_weight(a, i) : 0.0;
    const double total = fmax(team_sum_d<kOneBlock>(w, sh[0]), 1.0);
    double loss = 0.0;
    if (i < a.rows)
        a.coef[i] = w == 0.0 ? 0.0f : (float)policy_row(a.terms, a.old_logp[i], a.advantage[i],
                                                        a.terms.kl != 0.0 ? a.ref_logp[i] : 0.0f, a.logp[i], w / total, loss);
    loss = team_sum_d<kOneBlock>(loss, sh[1]);
    if (threadIdx.x == 0) a.loss[0] = (float)loss;
}

// More rows: a run for each workgroup, after k_weight_parts; the losses of the runs are
// added by k_loss_sum.  [4096] 17 us in one workgroup.
__global__ __launch_bounds__(kLgBlock) void k_policy_many(PolicyArgs a, const WeightPart* part, long long run,
                                                          double* losses) {
    __shared__ double sh[2][kLgBlock / kWave];
    static_assert(kLgBlock == 256, "a thread for each part");
    const double all = threadIdx.x < gridDim.x ? part[threadIdx.x].w : 0.0;
    const double total = fmax(team_sum_d<kLgBlock>(all, sh[0]), 1.0);
    const long long b = blockIdx.x * run, e = min(b + run, a.rows);
    double loss = 0.0;
    for (long long i = b + threadIdx.x; i < e; i += kLgBlock) {
        const double w = policy_weight(a, i);
        a.coef[i] = w == 0.0 ? 0.0f : (float)policy_row(a.terms, a.old_logp[i], a.advantage[i],
                                                        a.terms.kl != 0.0 ? a.ref_logp[i] : 0.0f, a.logp[i], w / total, loss);
    }
    loss = team_sum_d<kLgBlock>(loss, sh[1]);
    if (threadIdx.x == 0) losses[blockIdx.x] = loss;
}

// ---- policy loss and gradient in one pass ------------------------------------------
// A workgroup holds a row in registers from its load to its gradient's store, so
// logits are read once and gradients written once; it then walks on to the row
// gridDim.x further.  A row's vectors are taken into the running maximum and sum as
// they arrive, and the next row's loads are issued one by one as the stores free
// registers: exponentials run while memory does.  Loads and stores go through buffer
// resources, which drop what lies past the row (and, with no records, everything), so
// that no branch stands between them and each vector is waited for by itself.  Past
// the last whole vector a thread holds one element more.
//
// [4096, 151936] bfloat16, 90 % of the rows counting: 674 us as statistics, loss and
// gradient; 663 held in registers with a branch around each load, which makes every
// wait a wait for all; 520 so; 498 with rows dealt out evenly and nontemporal accesses
// (4.8 TB/s).  What is left is a CU's one row: 18 issue slots an element, two
// exponentials among them, are 20 of the 31 us that a row takes, and its reductions
// and 64-bit loss another 2.  Two readings of the row with the second from the last-level
// cache took 760 us, 512 threads of 38 vectors 564.
struct PolicyRowsArgs {
    LogitArgs a;
    PolicyArgs p;
    void* grad;
    // Where workgroups take several rows: max(sum of weights, 1), and the rows that count
    // followed by the others, so that each gets the same number of both wherever prompts
    // and padding lie.  Null: each workgroup sums the weights, rows as they come.
    const double* total;
    const int* order;
    double* part;          // a workgroup's loss
    unsigned* ticket;      // or null: k_loss_sum adds the parts
};

// Adds `n` parts of the loss in an order of their own, whichever threads add them
template <int NT, class F>
__device__ __forceinline__ void sum_loss(int n, float* loss, double* sh, F&& part) {
    double l = 0.0;
    for (int i = threadIdx.x; i < n; i += NT) l += part(i);
    l = team_sum_d<NT>(l, sh);
    if (threadIdx.x == 0) loss[0] = (float)l;
}

// The bits of -inf
template <class T>
constexpr uint32_t kNone = std::is_same<T, float>::value ? 0xFF800000u : std::is_same<T, f16_t>::value ? 0xFC00u : 0xFF80u;

// What a row's loss takes, read for kAhead of a workgroup's rows at once: a read of its
// own for each would stand in the way of the row that is on its way.
struct RowIn {
    int row, t;  // t -1: outside the vocabulary
    float w, old_logp, advantage, ref_logp, xt;
};
constexpr int kAhead = 64;

template <class T>
__device__ __forceinline__ RowIn row_in(const PolicyRowsArgs& q, long long k) {
    RowIn r{0, -1, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (k >= q.a.rows) return r;
    const int row = q.order ? q.order[k] : (int)k;
    r.row = row;
    const long long t = q.a.target[row];
    if (t == q.a.ignore) return r;
    r.w = q.p.weight ? q.p.weight[row] : 1.0f;
    if (r.w == 0.0f) return r;
    r.old_logp = q.p.old_logp[row];
    r.advantage = q.p.advantage[row];
    if (q.p.terms.kl != 0.0) r.ref_logp = q.p.ref_logp[row];
    if (t >= 0 && t < q.a.vocab) {
        r.t = (int)t;
        r.xt = (float)static_cast<const T*>(q.a.x)[(long long)row * q.a.stride + t];
    }
    return r;
}

// What a row's workgroup shares once its parts are joined
struct RowShare {
    RowStat s;
    float c, at_target;    // coefficient / T, the gradient at the target
    float logp;
    double loss;
};

// A call, so that the 64-bit functions' registers are not the row's
__attribute__((noinline)) __device__ RowShare row_result(PolicyTerms terms, RowIn in, RowStat s, double inv_t,
                                                         double total) {
    RowShare r;
    r.loss = 0.0;
    r.s = s;
    const double lp = in.t >= 0 ? logp_of(in.xt, s, inv_t) : NAN;
    if (in.t < 0) r.s.m = r.s.rest = NAN;
    const double c = policy_row(terms, in.old_logp, in.advantage, in.ref_logp, lp, (double)in.w / total, r.loss) * inv_t;
    r.c = (float)c;
    r.at_target = (float)(-c * expm1(lp));
    r.logp = (float)lp;
    return r;
}

// Joins the W waves' parts in wave 0, whose lanes all compute the row's loss, and
// hands the result to the workgroup.
template <int W>
__device__ __forceinline__ RowShare share_row(const PolicyRowsArgs& q, const RowPart& part, const RowIn& in, double total,
                                              RowPart* sh, RowShare* out) {
    const int wave = threadIdx.x / kWave, lane = __lane_id();
    if (lane == 0) sh[wave] = part;
    __syncthreads();
    if (wave == 0) {
        RowPart p = sh[lane % W];
#pragma unroll
        for (int o = 1; o < W; o <<= 1) p = merge(p, lane_xor(p, o), q.a.k.k1);
        const RowShare r = row_result(q.p.terms, in, finish(p), q.a.inv_t, total);
        if (lane == 0) *out = r;
    }
    __syncthreads();
    return *out;
}

template <int NT>
__device__ __forceinline__ double total_weight(const PolicyRowsArgs& q, double* sh) {
    if (q.total) return q.total[0];
    double w = 0.0;
    for (int i = threadIdx.x; i < (int)q.a.rows; i += NT) w += policy_weight(q.p, i);
    return fmax(team_sum_d<NT>(w, sh), 1.0);
}

template <class T, int NT, int NV, bool STREAM>
__global__ __launch_bounds__(NT, 4) void k_policy_rows(PolicyRowsArgs q) {
    using V = typename Vec16<T>::type;
    constexpr int kPolicy = STREAM ? 2 : 0;   // cache policy: nontemporal
    constexpr int VN = Vec16<T>::N, W = NT / kWave;
    __shared__ double shd[W];
    __shared__ RowPart shp[W];
    __shared__ RowShare shr;
    __shared__ RowIn shi[kAhead + 1];
    // The elements past the whole vectors, read with shi: [4096, 50261] bfloat16 218 us, 224
    // with each read by its thread a row ahead, which made its wave wait for all the row.
    __shared__ T tails[kAhead + 1][VN];
    const LogitArgs& a = q.a;
    const int tid = threadIdx.x;
    const int vocab = (int)a.vocab, whole = vocab / VN * VN;
    const bool tail = tid < vocab - whole;
    u32x4 x[NV];
    auto row_of = [&](long long row) { return static_cast<const T*>(a.x) + row * a.stride; };
    auto rsrc = [&](const T* p, bool on) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(p), (short)0, on ? whole * (int)sizeof(T) : 0, kBufWord3);
    };
    bool live;
    {   // a dropped store before each load: the counts of what is under way are then those of later rows
        const RowIn first = row_in<T>(q, blockIdx.x);
        live = first.w != 0.0f;
        const T* p = row_of(__builtin_amdgcn_readfirstlane(first.row));
        const __amdgpu_buffer_rsrc_t none = rsrc(p, false), in = rsrc(p, live);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            __builtin_amdgcn_raw_buffer_store_b128(u32x4{}, none, (j * NT + tid) * 16, 0, 0);
            x[j] = __builtin_amdgcn_raw_buffer_load_b128(in, (j * NT + tid) * 16, 0, kPolicy);
        }
    }
    const double total = total_weight<NT>(q, shd);
    double loss = 0.0;
    int ahead = 0;
    for (long long k = blockIdx.x; k < a.rows; k += gridDim.x, ahead = (ahead + 1) % kAhead) {
        if (ahead == 0) {
            __syncthreads();
            for (int i = tid; i <= kAhead; i += NT) {
                const RowIn in = row_in<T>(q, k + (long long)i * gridDim.x);
                shi[i] = in;
                if (whole < vocab && in.w != 0.0f) {
                    const T* p = row_of(in.row);
#pragma unroll
                    for (int e = 0; e < VN; ++e) tails[i][e] = p[min(whole + e, vocab - 1)];
                }
            }
            __syncthreads();
        }
        RowShare r{{0.0f, 0.0f}, 0.0f, 0.0f, 0.0f, 0.0};
        const RowIn& in_row = shi[ahead];
        const long long row = __builtin_amdgcn_readfirstlane(in_row.row);
        if (live) {
            WaveScan w;
            int first = tid * VN;
            asm volatile("" : "+v"(first));
#pragma unroll
            for (int j = 0; j < NV; j += 2) {
                float v[2 * VN];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (j + i == NV) {   // an odd count: the element past the vectors, alone
#pragma unroll
                        for (int e = 0; e < VN; ++e) v[i * VN + e] = e == 0 && tail ? (float)tails[ahead][tid] : -INFINITY;
                        continue;
                    }
                    u32x4& y = x[j + i];
                    if ((j + i + 1) * NT * VN > whole) {   // vectors past the row's end have been read as 0
                        const bool in = first + (j + i) * NT * VN < whole;
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[e] = in ? y[e] : sizeof(T) == 4 ? kNone<T> : kNone<T> << 16 | kNone<T>;
                    }
                    const V z = __builtin_bit_cast(V, y);
#pragma unroll
                    for (int e = 0; e < VN; ++e) v[i * VN + e] = (float)z[e];
                }
                w.add(v, a.k);
            }
            if (NV % 2 == 0) {
                const float v[1] = {tail ? (float)tails[ahead][tid] : -INFINITY};
                w.add(v, a.k);
            }
            // as they are: otherwise elements converted to float are kept for the gradient
#pragma unroll
            for (int j = 0; j < NV; ++j) asm volatile("" : "+v"(x[j]));
            r = share_row<W>(q, w.part(a.k), in_row, total, shp, &shr);
            loss += r.loss;
        }
        // a coefficient of 0 makes zeros of whatever the registers hold: the exponentials of
        // a row that has a coefficient are finite, and those of no row are of 0
        const RowGrad<T> f(r.s, r.c, a.k);
        const bool skip = !live;
        const int t = in_row.t;
        live = shi[ahead + 1].w != 0.0f;
        const T* np = row_of(__builtin_amdgcn_readfirstlane(shi[ahead + 1].row));
        T* g = static_cast<T*>(q.grad) + row * a.vocab;
        const __amdgpu_buffer_rsrc_t out = rsrc(g, true), in = rsrc(np, live);
        int off = tid * 16;
        asm volatile("" : "+v"(off));   // not 19 offsets kept over the loop
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const V z = __builtin_bit_cast(V, x[j]);
            V o;
#pragma unroll
            for (int e = 0; e < VN; ++e) o[e] = (T)f.value((float)z[e], a.k);
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), out, off + j * NT * 16, 0, kPolicy);
            x[j] = __builtin_amdgcn_raw_buffer_load_b128(in, off + j * NT * 16, 0, kPolicy);
        }
        if (tail) g[whole + tid] = (T)(skip ? 0.0f : f.value((float)tails[ahead][tid], a.k));
        // the target's element, again, by the thread that has written it
        if (t >= 0 && tid == (t < whole ? t / VN % NT : t - whole)) g[t] = (T)r.at_target;
        if (tid == 0) a.logp[row] = r.logp;
    }
    if (!q.ticket) {
        if (tid == 0) q.part[blockIdx.x] = loss;
        return;
    }
    __shared__ bool last_group;
    if (tid == 0) {
        publish_state(q.part + blockIdx.x, loss);
        last_group = last_of<true>(q.ticket, gridDim.x, blockIdx.x);
    }
    __syncthreads();
    if (last_group) sum_loss<NT>(gridDim.x, q.p.loss, shd, [&](int i) { return fetch_state(q.part + i); });
}

// The order of the rows, and max(sum of weights, 1): each workgroup places its run, a
// wave's rows at a time, after k_weight_parts, or up to kOwnParts rows after it has
// summed all weights itself (4096 rows: one launch of 9 us for two of 5 and 6).
constexpr long long kOwnParts = 8192;
__global__ __launch_bounds__(kLgBlock) void k_order(PolicyArgs a, const WeightPart* part, long long run, double* total,
                                                    int* order) {
    __shared__ WeightPart sh[2][kLgBlock / kWave];
    __shared__ int counts[2][kLgBlock / kWave];
    const int tid = threadIdx.x, wave = tid / kWave;
    const long long b = blockIdx.x * run, e = min(b + run, a.rows);
    WeightPart mine{0.0, 0}, front{0.0, 0};
    if (part) {
        if (tid < (int)gridDim.x) mine = part[tid];
        if (tid < (int)blockIdx.x) front = mine;
    } else {
        for (long long i = tid; i < a.rows; i += kLgBlock) {
            const WeightPart q = weight_part(a, i);
            mine = {mine.w + q.w, mine.live + q.live};
            if (i < b) front.live += q.live;
        }
    }
    const WeightPart all = team_sum_w<kLgBlock>(mine, sh[0]), before = team_sum_w<kLgBlock>(front, sh[1]);
    if (blockIdx.x == 0 && tid == 0) total[0] = fmax(all.w, 1.0);
    long long live = before.live, dead = all.live + b - before.live;
    int flip = 0;
    for (long long i = b + tid; i - tid < e; i += kLgBlock, flip ^= 1) {
        const bool in = i < e, on = in && policy_weight(a, i) != 0.0;
        const uint64_t ml = __ballot(on), md = __ballot(in && !on), below = (1ull << __lane_id()) - 1;
        if (__lane_id() == 0) counts[flip][wave] = __popcll(ml) | __popcll(md) << 16;
        __syncthreads();
        int l0 = 0, d0 = 0, l1 = 0, d1 = 0;
#pragma unroll
        for (int k = 0; k < kLgBlock / kWave; ++k) {
            const int c = counts[flip][k];
            if (k < wave) l0 += c & 0xFFFF, d0 += c >> 16;
            l1 += c & 0xFFFF, d1 += c >> 16;
        }
        if (on) order[live + l0 + __popcll(ml & below)] = (int)i;
        else if (in) order[dead + d0 + __popcll(md & below)] = (int)i;
        live += l1;
        dead += d1;
    }
}
// the loss from its parts, in a fixed order
__global__ __launch_bounds__(kLgBlock) void k_loss_sum(const double* part, int n, float* loss) {
    __shared__ double sh[kLgBlock / kWave];
    sum_loss<kLgBlock>(n, loss, sh, [&](int i) { return part[i]; });
}

// ---- preference loss over the rows' log-probabilities ------------------------------
struct PrefArgs {
    const double* logp;
    const long long* offsets;
    const float* ref;
    long long rows, pairs;
    double beta, eps;
    float *loss, *reward, *coef;
    double* sums;   // [2 pairs]: a sequence's sum, then its coefficient
};

// A sequence's rows, whatever its offsets are
struct Range {
    long long b, e;
};
__device__ __forceinline__ Range range_of(const PrefArgs& a, long long q) {
    return {min(max(a.offsets[q], 0LL), a.rows), min(a.offsets[q + 1], a.rows)};
}

// What one wave makes of sequence q, and one thread of pair i
__device__ __forceinline__ void pref_sum(const PrefArgs& a, long long q) {
    const Range r = range_of(a, q);
    double s = 0.0;
    for (long long i = r.b + __lane_id(); i < r.e; i += kWave) s += a.logp[i];
    s = wave_sum_d(s);
    if (__lane_id() == 0) a.sums[q] = s;
}
__device__ __forceinline__ double pref_pair(const PrefArgs& a, long long i) {
    const double rc = a.beta * (a.sums[i] - (double)a.ref[i]);
    const double rr = a.beta * (a.sums[i + a.pairs] - (double)a.ref[i + a.pairs]);
    a.reward[i] = (float)rc;
    a.reward[i + a.pairs] = (float)rr;
    const double h = rc - rr;
    // log(1 + e^-h) and log(1 + e^h), and their derivatives: each from e^-|h| without a
    // difference, so that a pair far apart keeps the digits of its e^-|h|
    const double u = exp(-fabs(h)), l = log1p(u);
    const double up = (h >= 0.0 ? 1.0 : u) / (1.0 + u), down = (h >= 0.0 ? u : 1.0) / (1.0 + u);
    const double c = a.beta / (double)a.pairs * (a.eps * up - (1.0 - a.eps) * down);
    a.sums[i] = c;
    a.sums[i + a.pairs] = -c;
    // h is infinite where a token of one answer has no probability: a share of 0 then has
    // no part of the loss
    return (a.eps < 1.0 ? (1.0 - a.eps) * (fmax(-h, 0.0) + l) : 0.0) + (a.eps > 0.0 ? a.eps * (fmax(h, 0.0) + l) : 0.0);
}
__device__ __forceinline__ void pref_coef(const PrefArgs& a, long long q) {
    const Range r = range_of(a, q);
    const float c = (float)a.sums[q];
    for (long long i = r.b + __lane_id(); i < r.e; i += kWave) a.coef[i] = c;
}
__device__ __forceinline__ void pref_pairs(const PrefArgs& a, double* sh) {
    double loss = 0.0;
    for (long long i = threadIdx.x; i < a.pairs; i += kOneBlock) loss += pref_pair(a, i);
    loss = team_sum_d<kOneBlock>(loss, sh);   // its barrier also orders the coefficients
    if (threadIdx.x == 0) a.loss[0] = (float)(loss / (double)a.pairs);
}

// One workgroup: a wave takes a sequence at a time, a thread a pair ([4091] tokens of 32
// sequences 7 us).
__global__ __launch_bounds__(kOneBlock) void k_preference(PrefArgs a) {
    __shared__ double sh[kOneBlock / kWave];
    const int wave = threadIdx.x / kWave;
    for (long long i = threadIdx.x; i < a.rows; i += kOneBlock) a.coef[i] = 0.0f;
    for (long long q = wave; q < 2 * a.pairs; q += kOneBlock / kWave) pref_sum(a, q);
    __syncthreads();
    pref_pairs(a, sh);
    for (long long q = wave; q < 2 * a.pairs; q += kOneBlock / kWave) pref_coef(a, q);
}

// Above kOneRows tokens or pairs: its three parts as launches of their own.
constexpr long long kOneRows = 16384;
__global__ __launch_bounds__(kLgBlock) void k_pref_sums(PrefArgs a) {
    const long long step = (long long)gridDim.x * kLgBlock, at = (long long)blockIdx.x * kLgBlock + threadIdx.x;
    for (long long i = at; i < a.rows; i += step) a.coef[i] = 0.0f;
    for (long long q = at / kWave; q < 2 * a.pairs; q += step / kWave) pref_sum(a, q);
}
__global__ __launch_bounds__(kOneBlock) void k_pref_pairs(PrefArgs a) {
    __shared__ double sh[kOneBlock / kWave];
    pref_pairs(a, sh);
}
__global__ __launch_bounds__(kLgBlock) void k_pref_coef(PrefArgs a) {
    const long long step = (long long)gridDim.x * kLgBlock, at = (long long)blockIdx.x * kLgBlock + threadIdx.x;
    for (long long q = at / kWave; q < 2 * a.pairs; q += step / kWave) pref_coef(a, q);
}

// ---- host ---------------------------------------------------------------------------
int check_logits(const tpr_logits_desc* d, const char* who) {
    if (!d) return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": null descriptor");
    if (!is_elem(d->dtype))
        return fail(TPR_ERR_UNSUPPORTED_DTYPE, std::string(who) + ": logits must be float32, float16 or bfloat16");
    if (d->rows < 0 || d->vocab < 0) return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": negative extent");
    if (d->rows > 0 && d->vocab == 0) return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": empty vocabulary");
    if (d->vocab >= (1LL << 28) || d->rows >= (1LL << 31))
        return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": 2^28 logits a row or 2^31 rows, or more");
    if (d->rows > 1 && d->row_stride < 0) return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": negative row stride");
    const double t = d->temperature;
    if (!(t >= 1e-20 && t <= 1e20))
        return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": temperature must be in [1e-20, 1e20]");
    return TPR_OK;
}

// Workgroups per row: one where there are more than 256 rows, or short ones, else a
// power of two that gives up to 512 in all, with 2048 elements each at least.  A row's
// last workgroup joins the parts, which costs 2 us: [512, 32000] bfloat16 takes 9.5 us
// whole and 11.4 in two parts, [256, 8000] 4.7 and 5.9, but [8, 32000] 6.5 in two
// parts and 5.4 in eight, [1, 151936] float32 6.5 in 16 and 5.9 in 64.
int row_split(const tpr_logits_desc* d) {
    long long s = 1;
    while (s < 64 && 2 * s * d->rows <= 512 && d->vocab >= std::max(16384LL, 2048 * 2 * s)) s *= 2;
    return (int)s;
}

size_t part_bytes(const tpr_logits_desc* d) {
    const int s = row_split(d);
    return s > 1 ? (size_t)d->rows * s * sizeof(RowPart) : 0;
}
Scale scale_of(double temperature) {
    Scale k;
    k.k = 1.44269504088896340736 / temperature;
    k.k1 = (float)k.k;
    if ((double)k.k1 >= k.k) k.k1 = std::nextafterf(k.k1, 0.0f);
    k.k2 = (float)(k.k - (double)k.k1);
    return k;
}

size_t align16(size_t n) { return (n + 15) & ~(size_t)15; }

LogitArgs logit_args(const tpr_logits_desc* d, const void* logits, const int64_t* target) {
    LogitArgs a{};
    a.x = logits;
    a.target = reinterpret_cast<const long long*>(target);
    a.rows = d->rows;
    a.vocab = d->vocab;
    a.stride = d->row_stride;
    a.ignore = d->ignore_index;
    a.k = scale_of(d->temperature);
    a.inv_t = 1.0 / d->temperature;
    return a;
}

int launch_stats(const tpr_logits_desc* d, const void* logits, const int64_t* target, const float* weight, float* logp,
                 double* logp64, float* lse, void* ws, hipStream_t st, const char* who) {
    if (d->rows == 0) return TPR_OK;
    LogitArgs a = logit_args(d, logits, target);
    a.S = row_split(d);
    a.chunk = ((d->vocab + a.S - 1) / a.S + 7) / 8 * 8;
    if (a.S > 1) a.tickets = stream_tickets(st);   // at most 256 rows
    a.weight = weight;
    a.logp = logp;
    a.logp64 = logp64;
    a.lse = reinterpret_cast<RowStat*>(lse);
    a.part = static_cast<RowPart*>(ws);
    // a launch's threads stay below 2^32: rows go in runs
    const long long most = kMaxThreads / kLgBlock;
    return with_elem(d->dtype, [&](auto t) -> int {
        using T = decltype(t);
        for (long long r0 = 0; r0 < d->rows; r0 += most / a.S) {
            LogitArgs b = a;
            b.rows = std::min(most / a.S, d->rows - r0);
            b.x = static_cast<const T*>(a.x) + r0 * a.stride;
            b.target = a.target + r0;
            b.weight = a.weight ? a.weight + r0 : nullptr;
            b.logp = a.logp + r0;
            b.logp64 = a.logp64 ? a.logp64 + r0 : nullptr;
            b.lse = a.lse + r0;
            hipLaunchKernelGGL(k_row_stats<T>, dim3((unsigned)(b.rows * b.S)), dim3(kLgBlock), 0, st, b);
            int rc = check_launch(who);
            if (rc != TPR_OK) return rc;
            if (b.S > 1 && !b.tickets) {  // only where all rows fit one launch
                const unsigned blocks = (unsigned)((b.rows * b.S + kLgBlock - 1) / kLgBlock);
                hipLaunchKernelGGL(k_row_join<T>, dim3(blocks), dim3(kLgBlock), 0, st, b);
                rc = check_launch(who);
                if (rc != TPR_OK) return rc;
            }
        }
        return TPR_OK;
    });
}

// Sizes of the logits from which the gradient's stores, and its loads too, pass the
// caches: dirty lines of a gradient are written back while the next logits are read,
// but a product that follows reads what the last-level cache (256 MB) holds of it.
// Log-probabilities and gradient over three sets of inputs in turn, without a product and
// with one by [V, 2048], stores through the caches -> past them: bfloat16 [512, 50264]
// (49 MiB) 30 -> 30, 356 -> 407 us; [1024, 50264] 63 -> 53, 543 -> 544; [512, 151936]
// (148 MiB) 95 -> 83, 681 -> 688; float16 [2048, 50261] (196 MiB) 132 -> 112, 691 -> 676;
// [768, 151936] 138 -> 115, 939 -> 933.  Stores -> loads too: bfloat16 [1024, 151936]
// (297 MiB) 153 -> 155, 1038 -> 1039; float16 [3500, 50261] (336 MiB) 203 -> 188, 1145 ->
// 1130; bfloat16 [1600, 151936] 253 -> 227, 1657 -> 1630.  The statistics' loads past the
// caches: [1600, 151936] 227 -> 239.
constexpr long long kPassStores = 160LL << 20, kPassLoads = 320LL << 20;

int launch_grad(const tpr_logits_desc* d, const float* coef, const float* scale, const void* logits,
                const int64_t* target, const float* lse, void* grad, hipStream_t st, const char* who) {
    if (d->rows == 0) return TPR_OK;
    GradArgs a{};
    a.x = logits;
    a.target = reinterpret_cast<const long long*>(target);
    a.coef = coef;
    a.scale = scale;
    a.lse = reinterpret_cast<const RowStat*>(lse);
    a.grad = grad;
    a.vocab = d->vocab;
    a.stride = d->row_stride;
    a.ignore = d->ignore_index;
    a.k = scale_of(d->temperature);
    a.inv_t = 1.0 / d->temperature;
    return with_elem(d->dtype, [&](auto t) -> int {
        using T = decltype(t);
        const long long per = (long long)kLgBlock * Vec16<T>::N * 4;
        a.S = (int)((d->vocab + per - 1) / per);
        const long long most = kMaxThreads / kLgBlock / a.S, bytes = d->rows * d->vocab * (long long)sizeof(T);
        for (long long r0 = 0; r0 < d->rows; r0 += most) {
            a.row0 = r0;
            const long long n = std::min(most, d->rows - r0);
            auto kernel = bytes < kPassStores ? k_logits_grad<T, 0> : bytes < kPassLoads ? k_logits_grad<T, 1>
                                                                                          : k_logits_grad<T, 2>;
            hipLaunchKernelGGL(kernel, dim3((unsigned)(n * a.S)), dim3(kLgBlock), 0, st, a);
            const int rc = check_launch(who);
            if (rc != TPR_OK) return rc;
        }
        return TPR_OK;
    });
}

// Runs of rows for what needs no logits: up to 256, of 512 rows at least.
struct WeightRuns {
    unsigned n;
    long long run;
};
WeightRuns weight_runs(int64_t rows) {
    const long long run = std::max<long long>(512, (rows + 255) / 256);
    return {(unsigned)((rows + run - 1) / run), run};
}

int launch_weight_parts(const PolicyArgs& a, const WeightRuns& r, WeightPart* part, hipStream_t st, const char* who) {
    hipLaunchKernelGGL(k_weight_parts, dim3(r.n), dim3(kLgBlock), 0, st, a, part, r.run);
    return check_launch(who);
}

// Rows that a workgroup's registers hold: threads, vectors a thread and workgroups per
// CU.  At most 76 registers of a thread are the row's, so 16 waves stay on a CU; longer
// rows (float32 above 77824 logits) take statistics and gradient apart.
struct HeldPlan {
    int nt, nv, per_cu;
};
HeldPlan held_plan(const tpr_logits_desc* d) {
    const long long vecs = d->vocab / (d->dtype == TPR_FLOAT32 ? 4 : 8);
    if (vecs <= 256 * 2) return {256, 2, 8};
    if (vecs <= 256 * 6) return {256, 6, 6};
    if (vecs <= 256 * 12) return {256, 12, 4};
    if (vecs <= 256 * 19) return {256, 19, 4};
    if (vecs <= 512 * 19) return {512, 19, 2};
    if (vecs <= 1024 * 19) return {1024, 19, 1};
    return {0, 0, 0};
}
constexpr int kMaxHeld = 8;               // workgroups per CU
// Logits from which loads and stores pass the caches.  As above, through -> past them:
// bfloat16 [1024, 50264] 61 -> 61 us, with a product 548 -> 535; float16 [2048, 50261]
// 124 -> 119, 700 -> 695; bfloat16 [4096, 32000] 128 -> 117, 579 -> 581; [4096, 151936]
// 516 -> 501, 2508 -> 2504.
constexpr long long kStreamBytes = kPassStores;

int launch_policy_rows(const tpr_logits_desc* d, const HeldPlan& h, PolicyRowsArgs q, double* total, int* order,
                       WeightPart* weights, hipStream_t st, const char* who) {
    const unsigned blocks = (unsigned)std::min(d->rows, (int64_t)device_info().cus * h.per_cu);
    if (d->rows > blocks) {
        q.total = total;
        q.order = order;
        const WeightRuns r = weight_runs(d->rows);
        if (d->rows <= kOwnParts) weights = nullptr;
        int rc = weights ? launch_weight_parts(q.p, r, weights, st, who) : TPR_OK;
        if (rc != TPR_OK) return rc;
        hipLaunchKernelGGL(k_order, dim3(r.n), dim3(kLgBlock), 0, st, q.p, weights, r.run, total, order);
        rc = check_launch(who);
        if (rc != TPR_OK) return rc;
    }
    const bool stream = d->rows * d->vocab * (d->dtype == TPR_FLOAT32 ? 4 : 2) >= kStreamBytes;
    q.ticket = stream_tickets(st);
    int rc = with_elem(d->dtype, [&](auto t) -> int {
        using T = decltype(t);
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(blocks), dim3(h.nt), 0, st, q);
            return check_launch(who);
        };
        if (h.nt == 1024) return go(stream ? k_policy_rows<T, 1024, 19, true> : k_policy_rows<T, 1024, 19, false>);
        if (h.nt == 512) return go(stream ? k_policy_rows<T, 512, 19, true> : k_policy_rows<T, 512, 19, false>);
        if (h.nv == 19) return go(stream ? k_policy_rows<T, 256, 19, true> : k_policy_rows<T, 256, 19, false>);
        if (h.nv == 12) return go(stream ? k_policy_rows<T, 256, 12, true> : k_policy_rows<T, 256, 12, false>);
        if (h.nv == 6) return go(stream ? k_policy_rows<T, 256, 6, true> : k_policy_rows<T, 256, 6, false>);
        return go(stream ? k_policy_rows<T, 256, 2, true> : k_policy_rows<T, 256, 2, false>);
    });
    if (rc != TPR_OK || q.ticket) return rc;
    hipLaunchKernelGGL(k_loss_sum, dim3(1), dim3(kLgBlock), 0, st, q.part, (int)blocks, q.p.loss);
    return check_launch(who);
}

}  // namespace
}  // namespace tpr

using namespace tpr;

extern "C" size_t tpr_token_logprob_workspace_bytes(const tpr_logits_desc* desc) {
    if (check_logits(desc, "tpr_token_logprob") != TPR_OK) return 0;
    return part_bytes(desc);
}

extern "C" int tpr_token_logprob(const tpr_logits_desc* desc, const void* logits, const int64_t* target, float* logp,
                                 float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "tpr_token_logprob";
    const int rc = check_logits(desc, who);
    if (rc != TPR_OK) return rc;
    if (desc->rows == 0) return TPR_OK;
    if (!logits || !target || !logp || !lse) return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": null pointer");
    const size_t need = part_bytes(desc);
    if (need && (!workspace || workspace_bytes < need))
        return fail(TPR_ERR_WORKSPACE, std::string(who) + ": workspace smaller than tpr_token_logprob_workspace_bytes");
    return launch_stats(desc, logits, target, nullptr, logp, nullptr, lse, workspace, static_cast<hipStream_t>(stream), who);
}

extern "C" int tpr_token_logprob_backward(const tpr_logits_desc* desc, const float* coef, const float* scale,
                                          const void* logits, const int64_t* target, const float* lse, void* grad,
                                          void* stream) {
    const char* who = "tpr_token_logprob_backward";
    const int rc = check_logits(desc, who);
    if (rc != TPR_OK) return rc;
    if (desc->rows == 0) return TPR_OK;
    if (!logits || !target || !coef || !lse || !grad) return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": null pointer");
    return launch_grad(desc, coef, scale, logits, target, lse, grad, static_cast<hipStream_t>(stream), who);
}

namespace {
// Policy workspace: the statistics' parts, the unrounded logp, lse and coef where the
// caller has none, the weights' sum and a part of the loss for each workgroup that holds
// rows, the weights' parts and the order of the rows.
struct PolicyWs {
    size_t logp, lse, coef, parts, weights, order, total;
};
PolicyWs policy_ws(const tpr_logits_desc* d) {
    PolicyWs w;
    w.logp = align16(part_bytes(d));
    w.lse = w.logp + align16((size_t)d->rows * 8);
    w.coef = w.lse + align16((size_t)d->rows * 8);
    w.parts = w.coef + align16((size_t)d->rows * 4);
    w.weights = w.parts + align16((size_t)(1 + (long long)device_info().cus * kMaxHeld) * 8);
    w.order = w.weights + 256 * sizeof(WeightPart);
    w.total = w.order + align16((size_t)d->rows * 4);
    return w;
}
}  // namespace

extern "C" size_t tpr_policy_loss_workspace_bytes(const tpr_logits_desc* desc) {
    if (check_logits(desc, "tpr_policy_loss") != TPR_OK) return 0;
    return policy_ws(desc).total;
}

extern "C" int tpr_policy_loss(const tpr_logits_desc* desc, const tpr_policy_desc* policy, const void* logits,
                               const int64_t* target, const float* old_logp, const float* advantage,
                               const float* ref_logp, const float* weight, float* loss, float* logp, float* lse,
                               float* coef, void* grad, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "tpr_policy_loss";
    int rc = check_logits(desc, who);
    if (rc != TPR_OK) return rc;
    if (!policy) return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": null descriptor");
    if (!(policy->clip_low >= 0.0 && policy->clip_low <= 1.0) || !(policy->clip_high >= 0.0))
        return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": clip_low must be in [0, 1] and clip_high not negative");
    if (!(std::isfinite(policy->kl_coef) && std::isfinite(policy->clip_high)))
        return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": kl_coef and clip_high must be finite");
    if (!loss) return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": null pointer");
    if (desc->rows > 0) {
        if (!logits || !target || !old_logp || !advantage || !logp || (!grad && (!lse || !coef)))
            return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": null pointer");
        if (!ref_logp && policy->kl_coef != 0.0)
            return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": a KL term needs ref_logp");
    }
    const PolicyWs w = policy_ws(desc);
    if (w.total && (!workspace || workspace_bytes < w.total))
        return fail(TPR_ERR_WORKSPACE, std::string(who) + ": workspace smaller than tpr_policy_loss_workspace_bytes");
    char* ws = static_cast<char*>(workspace);
    PolicyArgs a{};
    a.target = reinterpret_cast<const long long*>(target);
    a.old_logp = old_logp;
    a.advantage = advantage;
    a.ref_logp = ref_logp;
    a.weight = weight;
    a.rows = desc->rows;
    a.ignore = desc->ignore_index;
    a.terms = PolicyTerms{1.0 - policy->clip_low, 1.0 + policy->clip_high, policy->kl_coef};
    a.loss = loss;
    WeightPart* weights = reinterpret_cast<WeightPart*>(ws + w.weights);
    const HeldPlan held = held_plan(desc);
    if (grad && !lse && !coef && held.nt && desc->rows > 0) {
        PolicyRowsArgs q{};
        q.a = logit_args(desc, logits, target);
        q.a.logp = logp;
        q.p = a;
        q.grad = grad;
        q.part = reinterpret_cast<double*>(ws + w.parts) + 1;
        return launch_policy_rows(desc, held, q, q.part - 1, reinterpret_cast<int*>(ws + w.order), weights,
                                  static_cast<hipStream_t>(stream), who);
    }
    if (!lse) lse = reinterpret_cast<float*>(ws + w.lse);
    if (!coef) coef = reinterpret_cast<float*>(ws + w.coef);
    hipStream_t st = static_cast<hipStream_t>(stream);
    double* logp64 = reinterpret_cast<double*>(ws + w.logp);
    rc = launch_stats(desc, logits, target, weight, logp, logp64, lse, ws, st, who);
    if (rc != TPR_OK) return rc;
    a.logp = logp64;
    a.coef = coef;
    if (desc->rows <= kOneBlock) {
        hipLaunchKernelGGL(k_policy, dim3(1), dim3(kOneBlock), 0, st, a);
    } else {
        const WeightRuns r = weight_runs(desc->rows);
        rc = launch_weight_parts(a, r, weights, st, who);
        if (rc != TPR_OK) return rc;
        double* losses = reinterpret_cast<double*>(ws + w.parts);
        hipLaunchKernelGGL(k_policy_many, dim3(r.n), dim3(kLgBlock), 0, st, a, weights, r.run, losses);
        rc = check_launch(who);
        if (rc != TPR_OK) return rc;
        hipLaunchKernelGGL(k_loss_sum, dim3(1), dim3(kLgBlock), 0, st, losses, (int)r.n, loss);
    }
    rc = check_launch(who);
    if (rc != TPR_OK || !grad) return rc;
    return launch_grad(desc, coef, nullptr, logits, target, lse, grad, st, who);
}

extern "C" size_t tpr_preference_loss_workspace_bytes(const tpr_logits_desc* desc, int64_t pairs) {
    if (check_logits(desc, "tpr_preference_loss") != TPR_OK || pairs < 0) return 0;
    return align16(part_bytes(desc)) + align16((size_t)desc->rows * 8) + (size_t)pairs * 16;
}

extern "C" int tpr_preference_loss(const tpr_logits_desc* desc, int64_t pairs, double beta, double label_smoothing,
                                   const void* logits, const int64_t* target, const int64_t* offsets, const float* ref,
                                   float* loss, float* reward, float* logp, float* lse, float* coef, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    const char* who = "tpr_preference_loss";
    int rc = check_logits(desc, who);
    if (rc != TPR_OK) return rc;
    if (pairs < 1 || pairs >= (1LL << 30))
        return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": there must be a pair, and fewer than 2^30");
    if (!std::isfinite(beta)) return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": beta must be finite");
    if (!(label_smoothing >= 0.0 && label_smoothing <= 1.0))
        return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": label_smoothing must be in [0, 1]");
    if (!offsets || !ref || !loss || !reward || (desc->rows > 0 && (!logits || !target || !logp || !lse || !coef)))
        return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": null pointer");
    const size_t need = tpr_preference_loss_workspace_bytes(desc, pairs);
    if (!workspace || workspace_bytes < need)
        return fail(TPR_ERR_WORKSPACE, std::string(who) + ": workspace smaller than tpr_preference_loss_workspace_bytes");
    hipStream_t st = static_cast<hipStream_t>(stream);
    double* logp64 = reinterpret_cast<double*>(static_cast<char*>(workspace) + align16(part_bytes(desc)));
    rc = launch_stats(desc, logits, target, nullptr, logp, logp64, lse, workspace, st, who);
    if (rc != TPR_OK) return rc;
    PrefArgs a{};
    a.logp = logp64;
    a.offsets = reinterpret_cast<const long long*>(offsets);
    a.ref = ref;
    a.rows = desc->rows;
    a.pairs = pairs;
    a.beta = beta;
    a.eps = label_smoothing;
    a.loss = loss;
    a.reward = reward;
    a.coef = coef;
    a.sums = logp64 + (align16((size_t)desc->rows * 8) / 8);
    if (desc->rows <= kOneRows && pairs <= kOneRows) {
        hipLaunchKernelGGL(k_preference, dim3(1), dim3(kOneBlock), 0, st, a);
        return check_launch(who);
    }
    // a wave for each sequence, up to 32 a CU
    const unsigned blocks = (unsigned)std::min<long long>((2 * pairs + 3) / 4, (long long)device_info().cus * 8);
    hipLaunchKernelGGL(k_pref_sums, dim3(blocks), dim3(kLgBlock), 0, st, a);
    rc = check_launch(who);
    if (rc != TPR_OK) return rc;
    hipLaunchKernelGGL(k_pref_pairs, dim3(1), dim3(kOneBlock), 0, st, a);
    rc = check_launch(who);
    if (rc != TPR_OK) return rc;
    hipLaunchKernelGGL(k_pref_coef, dim3(blocks), dim3(kLgBlock), 0, st, a);
    return check_launch(who);
}
