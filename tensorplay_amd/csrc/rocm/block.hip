// gfx950 dropout and the end of a transformer block, behind tpr_dropout(),
// tpr_gated_norm() and tpr_gated_norm_backward().
//
// Dropout's mask is a function of (seed, offset, row, column) (philox.h): it is made
// again where it is needed, eight columns from one block of random bits.
//
// End of a block, along a row of n columns, with rms(v) = sqrt(mean(v^2) + eps):
//   nx = x / rms(x),  u = mask (nx w1),  out = a h + g u,  no = out / rms(out),  y = no w2.
// Backward, given dy and dout:
//   t = dy w2,   d = dout + (t - no mean(t no)) / rms(out),   dh = a d,
//   q = d g mask w1,   dx = (q - nx mean(q nx)) / rms(x),
//   dw2 = sum_rows dy no,   dw1 = sum_rows d g mask nx,   dg = sum_rows d u.
// A row is read once, held in registers over its reductions and written once.  The
// sums over rows are kept in registers while a workgroup walks its run of rows, and
// the runs' sums are added in a fixed order by a second launch.  All of it is bound by
// memory: at [16384, 4096] bfloat16 with a float32 residual the forward pass takes 144 us
// (5.6 TB/s), the backward 238 + 7 (4.9), dropout of [16384, 4096] 41 (6.5, of which the
// random bits' multiplications alone would take 30).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>

#include "common.h"
#include "elem.h"
#include "philox.h"

namespace tpr {
namespace {

constexpr int kBlk = 256;

// ---- dropout ----------------------------------------------------------------------
// q = n / d for 32-bit n by a multiplication (Granlund and Montgomery, "Division by
// invariant integers using multiplication", PLDI 1994).
struct FastDiv {
    uint32_t d, mul, shift;
    FastDiv() : FastDiv(1) {}
    explicit FastDiv(uint32_t den) : d(den) {
        shift = 0;
        while (shift < 32 && (1ull << shift) < den) ++shift;
        mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - den)) / den + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const {
        return (uint32_t)(((uint64_t)__umulhi(n, mul) + n) >> shift);
    }
};

struct DropoutArgs {
    const void* in;
    void* out;
    DropArgs d;
    FastDiv vecs;      // vectors of 8 columns in a row
    uint32_t total;    // vectors of this launch
    uint32_t row0;
    long long cols;
};

// PASS: the stores pass the caches, in half precision from kDropoutPass bytes on: two
// dropouts of [16384, 4096] bfloat16 one after the other 104 -> 89 us (6.0 TB/s), of
// [8192, 4096] 43 -> 47.  float32 stores two halves of 32 bytes a thread, which must
// meet in a cache: one dropout of [16384, 4096] 95 -> 107 us.
constexpr long long kDropoutPass = 128LL << 20;

template <class T, bool PASS>
__global__ __launch_bounds__(kBlk) void k_dropout(DropoutArgs a) {
    const uint32_t i = blockIdx.x * kBlk + threadIdx.x;
    if (i >= a.total) return;
    const uint32_t r = a.vecs.div(i), vec = i - r * a.vecs.d;
    const long long at = (long long)r * a.cols + (long long)vec * 8;
    const int left = (int)min(8LL, a.cols - (long long)vec * 8);
    float v[8];
    load_n(v, static_cast<const T*>(a.in) + at, left, 0.0f);
    const uint32_t keep = drop_keep(a.d, vec, a.row0 + r);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (keep >> e & 1) ? v[e] * a.d.up : 0.0f;
    store_n<PASS>(static_cast<T*>(a.out) + at, v, left);
}

// ---- end of a block -----------------------------------------------------------------
struct BlockArgs {
    const void *x, *h, *pre, *post, *gate;   // h: the residual stream before (forward) or out (backward)
    void *out, *y;
    float *rstd_post, *rstd_pre;
    int rows, cols;
    FastDiv group;       // rows of one gate
    float inv_cols, eps, scale;
    DropArgs d;
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr int kBufWord3 = 0x00020000;  // raw buffer resource, 32-bit data (gfx9 family)

// Eight elements as they lie in memory.
template <class T>
struct Raw8 {
    static constexpr int kParts = 8 * sizeof(T) / 16;
    u32x4 v[kParts];
    // as it is: otherwise the compiler keeps the elements converted to float from one
    // use to the next, in twice the registers
    __device__ __forceinline__ void settle() {
#pragma unroll
        for (int i = 0; i < kParts; ++i) asm volatile("" : "+v"(v[i]));
    }
    __device__ __forceinline__ float at(int i) const {
        constexpr int K = Vec16<T>::N;
        return (float)__builtin_bit_cast(typename Vec16<T>::type, v[i / K])[i % K];
    }
};

// A row of `cols` elements, taken in vectors of 8, 16 bytes a load, through a buffer
// resource, which reads 0 past the row and drops stores there: no branch stands between
// loads.  ODD (cols no multiple of 8): the row's last, partial 16 bytes are read as the
// 16 that end with the row, and shifted into place by fix() once they are used.  ODD 2:
// a row may be shorter than 16 bytes, which takes a branch with loads of its own; where
// rows are longer, it would only keep loads from passing it ([8192, 8191] bfloat16, float32
// residual: backward 364 us with it everywhere, 275 so).
template <class T, int ODD>
struct Row {
    static constexpr int K = Vec16<T>::N, kParts = Raw8<T>::kParts;
    T* p;
    int cols;
    __amdgpu_buffer_rsrc_t r;
    __device__ __forceinline__ Row(const void* base, long long row, int n, bool on = true) {
        p = const_cast<T*>(static_cast<const T*>(base)) + row * n;
        cols = on ? n : 0;
        r = __builtin_amdgcn_make_buffer_rsrc(p, (short)0, cols * (int)sizeof(T), kBufWord3);
    }
    // the partial part, or one that no thread has
    static __device__ __forceinline__ int partial(int n) { return n % K ? n / K : -1; }
    __device__ __forceinline__ Raw8<T> load(int vec) const {
        Raw8<T> o;
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
            const int part = vec * kParts + i;
            int off = part * 16;
            if (ODD) off = part == partial(cols) ? (cols - K) * (int)sizeof(T) : off;   // cols < K: out of range
            o.v[i] = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
        }
        return o;
    }
    __device__ __forceinline__ void fix(Raw8<T>& o, int vec) const {
        if constexpr (!ODD) return;
        if (ODD == 2 && cols < K) {   // a row that is all of a part
            using V = typename Vec16<T>::type;
            if (vec == 0) {
                V t;
#pragma unroll
                for (int e = 0; e < K; ++e) t[e] = e < cols ? p[e] : (T)0.0f;
                o.v[0] = __builtin_bit_cast(u32x4, t);
            }
            return;
        }
        const int s = K - cols % K;   // elements to drop in front
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
            const u32x4 v = o.v[i];
            u32x4 t = v;
            int words = s;
            if constexpr (sizeof(T) == 2) {
                if (s & 1)
                    t = u32x4{t[0] >> 16 | t[1] << 16, t[1] >> 16 | t[2] << 16, t[2] >> 16 | t[3] << 16, t[3] >> 16};
                words = s >> 1;
            }
            if (words & 1) t = u32x4{t[1], t[2], t[3], 0};
            if (words & 2) t = u32x4{t[2], t[3], 0, 0};
            const bool on = vec * kParts + i == partial(cols);
#pragma unroll
            for (int e = 0; e < 4; ++e) o.v[i][e] = on ? t[e] : v[e];
        }
    }
    __device__ __forceinline__ Raw8<T> get(int vec) const {
        Raw8<T> o = load(vec);
        fix(o, vec);
        return o;
    }
    __device__ __forceinline__ void store(int vec, const float (&v)[8]) const {
        using V = typename Vec16<T>::type;
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
            V t;
#pragma unroll
            for (int e = 0; e < K; ++e) t[e] = (T)v[i * K + e];
            const int part = vec * kParts + i;
            if (!ODD || part != partial(cols)) {
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, t), r, part * 16, 0, 0);
            } else {
#pragma unroll
                for (int e = 0; e < K - 1; ++e)
                    if (part * K + e < cols) p[part * K + e] = t[e];
            }
        }
    }
};

// The team of threads that takes a row: a wave, or the workgroup; and its lanes.
template <int NT>
struct Team {
    static constexpr int kThreads = NT < kBlk ? kBlk : NT, kTeams = kThreads / NT;
    static __device__ __forceinline__ int index() {
        return kTeams == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / NT);
    }
    static __device__ __forceinline__ int lane() { return threadIdx.x % NT; }
};

// NT threads a row, NV vectors of 8 columns a thread.  Everything that a row needs is
// under way before its first sum: [8, 4096] bfloat16 takes 3.7 us, 5.6 with the residual,
// the weights and the gate loaded where they are used.
template <class T, class R, int NT, int NV, int ODD>
__global__ __launch_bounds__(Team<NT>::kThreads) void k_block_fwd(BlockArgs a) {
    __shared__ float sh1[NT / kWave], sh2[NT / kWave];
    const int lane = Team<NT>::lane();
    const int row = blockIdx.x * Team<NT>::kTeams + Team<NT>::index();
    if (row >= a.rows) return;   // whole waves
    Raw8<T> x[NV], post[NV], gate[NV], pre[NV];
    Raw8<R> h[NV];
    {
        const Row<T, ODD> rx(a.x, row, a.cols), rpost(a.post, 0, a.cols, a.post), rpre(a.pre, 0, a.cols);
        const Row<T, ODD> rgate(a.gate, a.gate ? a.group.div(row) : 0, a.cols, a.gate);
        const Row<R, ODD> rh(a.h, row, a.cols);
#pragma unroll
        for (int j = 0; j < NV; ++j) x[j] = rx.load(j * NT + lane);
#pragma unroll
        for (int j = 0; j < NV; ++j) h[j] = rh.load(j * NT + lane);
#pragma unroll
        for (int j = 0; j < NV; ++j) post[j] = rpost.load(j * NT + lane);
#pragma unroll
        for (int j = 0; j < NV; ++j) gate[j] = rgate.load(j * NT + lane);
#pragma unroll
        for (int j = 0; j < NV; ++j) pre[j] = rpre.load(j * NT + lane);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int vec = j * NT + lane;
            rx.fix(x[j], vec);
            rh.fix(h[j], vec);
            if (a.post) rpost.fix(post[j], vec);
            if (a.gate) rgate.fix(gate[j], vec);
            rpre.fix(pre[j], vec);
        }
    }
    float rstd = 1.0f;
    if (a.post) {
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(x[j].at(e), x[j].at(e), ss);
        ss = team_sum_f<NT>(ss, sh1);
        rstd = 1.0f / sqrtf(fmaf(ss, a.inv_cols, a.eps));
        if (lane == 0) a.rstd_post[row] = rstd;
    }
    float u[NV][8];
    float ss = 0.0f;
    const Row<R, ODD> out(a.out, row, a.cols);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int vec = j * NT + lane;
#pragma unroll
        for (int e = 0; e < 8; ++e) u[j][e] = a.post ? x[j].at(e) * rstd * post[j].at(e) : x[j].at(e);
        if (a.d.below) {
            const uint32_t keep = drop_keep(a.d, vec, (uint32_t)row);
#pragma unroll
            for (int e = 0; e < 8; ++e) u[j][e] = (keep >> e & 1) ? u[j][e] * a.d.up : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            u[j][e] = a.gate ? fmaf(a.scale, h[j].at(e), u[j][e] * gate[j].at(e)) : fmaf(a.scale, h[j].at(e), u[j][e]);
            ss = fmaf(u[j][e], u[j][e], ss);
        }
        out.store(vec, u[j]);
    }
    ss = team_sum_f<NT>(ss, sh2);
    rstd = 1.0f / sqrtf(fmaf(ss, a.inv_cols, a.eps));
    if (lane == 0) a.rstd_pre[row] = rstd;
    const Row<T, ODD> y(a.y, row, a.cols);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int e = 0; e < 8; ++e) u[j][e] = u[j][e] * rstd * pre[j].at(e);
        y.store(j * NT + lane, u[j]);
    }
}

// Rows of no columns: the mean of no squares is NaN, and so are the roots.
__global__ __launch_bounds__(kBlk) void k_no_columns(float* rstd_post, float* rstd_pre, long long rows) {
    const long long row = (long long)blockIdx.x * kBlk + threadIdx.x;
    if (row >= rows) return;
    if (rstd_post) rstd_post[row] = NAN;
    if (rstd_pre) rstd_pre[row] = NAN;
}

struct BlockBwdArgs {
    BlockArgs b;
    const void *gy, *gout;
    void *gx, *gh, *ggate;
    // Runs of rows, one a workgroup: `run` rows of one gate's group (per_group runs a
    // group), whose teams take every kTeams-th row; or `groups` whole groups, of which
    // a team takes every kTeams-th and writes the gate's gradient itself.
    int run, per_group, groups;
    float* part;         // [2 or 3][runs][cols]: sums for pre, post, gate
    long long part_stride;
};

// A row's inputs stay as they lie in memory until they are used, and those of the
// team's next row are loaded as soon as their registers are free: gy, out and gout
// before the second sum, x after it; the weights and the gate before the sum that they
// wait for ([32768, 768] bfloat16 78 -> 74 us).  Above 8192 columns there are no registers for that
// (what is spilled is waited for with the loads: 785 us at [4096, 16384] bfloat16): a row
// is then loaded where it is used, and LDS holds two of the sums over rows (264 us).
// Loads at their uses and 256 threads of two vectors: 355 us at [16384, 4096], 244 so.
template <class T, class R, int NT, int NV, int ODD>
__global__ __launch_bounds__(Team<NT>::kThreads) void k_block_bwd(BlockBwdArgs q) {
    constexpr int kTeams = Team<NT>::kTeams, kCols = NT * NV * 8;
    constexpr bool kAhead = NT * NV <= 1024;
    __shared__ float sh1[2][NT / kWave], sh2[2][NT / kWave];
    __shared__ float join[kTeams > 1 ? kTeams - 1 : 1][kTeams > 1 ? kCols : 1];
    const BlockArgs& a = q.b;
    const int lane = Team<NT>::lane(), team = Team<NT>::index();
    const int run = blockIdx.x, group = a.group.d;
    int row, r1, gate, left = 0;   // left: rows of the present group after this one (whole groups)
    if (q.per_group) {
        gate = run / q.per_group;
        const int r0 = gate * group + (run - gate * q.per_group) * q.run;
        row = r0 + team;
        r1 = min(r0 + q.run, (gate + 1) * group);
    } else {
        const int r0 = run * q.groups * group;
        gate = run * q.groups + team;
        row = r0 + team * group;
        r1 = min(r0 + q.groups * group, a.rows);
        left = group - 1;
    }
    // sums over rows: in registers, or for two of the three in LDS, each thread its own
    constexpr int kHeld = kAhead ? NV : 1;
    __shared__ float held[2][kAhead ? 1 : NV * 8][kAhead ? 1 : NT];
    float dpre[kHeld][8] = {}, dpost[kHeld][8] = {}, dgate[NV][8] = {};
    if constexpr (!kAhead) {
#pragma unroll
        for (int i = 0; i < NV * 8; ++i) held[0][i][lane] = held[1][i][lane] = 0.0f;
    }
    auto add_pre = [&](int j, int e, float u, float v) {
        if constexpr (kAhead) dpre[j][e] = fmaf(u, v, dpre[j][e]);
        else held[0][j * 8 + e][lane] = fmaf(u, v, held[0][j * 8 + e][lane]);
    };
    auto add_post = [&](int j, int e, float u, float v) {
        if constexpr (kAhead) dpost[j][e] = fmaf(u, v, dpost[j][e]);
        else held[1][j * 8 + e][lane] = fmaf(u, v, held[1][j * 8 + e][lane]);
    };
    Raw8<T> gy[NV], x[NV];
    Raw8<R> h[NV], gout[NV];
    float rstd1 = 1.0f, rstd2 = 0.0f;
    auto load_first = [&](int i) {
        const bool on = i < r1;
        const int k = on ? i : 0;
        const Row<T, ODD> rgy(q.gy, k, a.cols, on);
        const Row<R, ODD> rh(a.h, k, a.cols, on), rgout(q.gout, k, a.cols, on && q.gout);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            gy[j] = rgy.load(j * NT + lane);
            h[j] = rh.load(j * NT + lane);
            if (kAhead) gout[j] = rgout.load(j * NT + lane);
        }
    };
    auto load_x = [&](int i) {
        const bool on = i < r1;
        const Row<T, ODD> rx(a.x, on ? i : 0, a.cols, on);
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (kAhead) x[j] = rx.load(j * NT + lane);
        rstd2 = on ? a.rstd_pre[i] : 0.0f;
        rstd1 = on && a.post ? a.rstd_post[i] : 1.0f;
    };
    load_first(row);
    load_x(row);
    const Row<T, ODD> rpre(a.pre, 0, a.cols), rpost(a.post, 0, a.cols, a.post);
    int flip = 0;               // the sums' LDS words alternate, so one barrier a sum is enough
    while (row < r1) {
        int next = row + kTeams;
        bool ends = false;      // the group does
        if (!q.per_group) {
            ends = left == 0;
            next = ends ? row + 1 + (kTeams - 1) * group : row + 1;
            left = ends ? group - 1 : left - 1;
        }
        float c = 0.0f;
        Raw8<T> pre[NV];
        if (kAhead) {
#pragma unroll
            for (int j = 0; j < NV; ++j) pre[j] = rpre.load(j * NT + lane);
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int vec = j * NT + lane;
            if (!kAhead) pre[j] = rpre.load(vec);
            rpre.fix(pre[j], vec);
            Row<T, ODD>(q.gy, row, a.cols).fix(gy[j], vec);
            Row<R, ODD>(a.h, row, a.cols).fix(h[j], vec);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float no = h[j].at(e) * rstd2, g = gy[j].at(e);
                add_pre(j, e, g, no);
                c = fmaf(g * pre[j].at(e), no, c);
            }
            gy[j].settle();
            h[j].settle();
            pre[j].settle();
            if (!kAhead) __builtin_amdgcn_sched_barrier(0);   // one vector at a time
        }
        const Row<T, ODD> rgate(a.gate, gate, a.cols, a.gate);
        Raw8<T> post[NV], gates[NV];
        if (kAhead) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                post[j] = rpost.load(j * NT + lane);
                gates[j] = rgate.load(j * NT + lane);
            }
        }
        c = team_sum_f<NT>(c, sh1[flip]) * a.inv_cols;
        float d[NV][8];
        float c1 = 0.0f;
        const Row<R, ODD> gh(q.gh, row, a.cols), rgout(q.gout, row, a.cols, q.gout);
        const Row<T, ODD> rx(a.x, row, a.cols);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int vec = j * NT + lane;
            if constexpr (!kAhead) {
                gout[j] = rgout.load(vec);
                x[j] = rx.load(vec);
            }
            if (!kAhead) {
                post[j] = rpost.load(vec);
                gates[j] = rgate.load(vec);
            }
            rpost.fix(post[j], vec);
            rgate.fix(gates[j], vec);
            if (q.gout) rgout.fix(gout[j], vec);
            rx.fix(x[j], vec);
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float no = h[j].at(e) * rstd2;
                const float g = rstd2 * fmaf(-no, c, gy[j].at(e) * pre[j].at(e));
                d[j][e] = q.gout ? gout[j].at(e) + g : g;
                o[e] = a.scale * d[j][e];
            }
            gh.store(vec, o);
            uint32_t keep = 0xFF;
            float up = 1.0f;
            if (a.d.below) {
                keep = drop_keep(a.d, vec, (uint32_t)row);
                up = a.d.up;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float nx = x[j].at(e) * rstd1, w = a.post ? post[j].at(e) : 1.0f;
                const bool kept = keep >> e & 1;
                if (a.gate) {
                    dgate[j][e] = fmaf(d[j][e], kept ? nx * w * up : 0.0f, dgate[j][e]);
                    d[j][e] *= gates[j].at(e);
                }
                d[j][e] = kept ? d[j][e] * up : 0.0f;
                add_post(j, e, d[j][e], nx);
                d[j][e] *= w;
                c1 = fmaf(d[j][e], nx, c1);
            }
            x[j].settle();
            if (!kAhead) __builtin_amdgcn_sched_barrier(0);
        }
        if (kAhead) load_first(next);
        if (a.post) c1 = team_sum_f<NT>(c1, sh2[flip]) * a.inv_cols;
        const Row<T, ODD> gx(q.gx, row, a.cols);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (a.post) {
#pragma unroll
                for (int e = 0; e < 8; ++e) d[j][e] = rstd1 * fmaf(-(x[j].at(e) * rstd1), c1, d[j][e]);
            }
            gx.store(j * NT + lane, d[j]);
        }
        if (!kAhead) load_first(next);
        load_x(next);
        if (a.gate && ends) {
            const Row<T, ODD> gg(q.ggate, gate, a.cols);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                gg.store(j * NT + lane, dgate[j]);
#pragma unroll
                for (int e = 0; e < 8; ++e) dgate[j][e] = 0.0f;
            }
        }
        if (ends) gate += kTeams;
        row = next;
        flip ^= 1;
    }
    if constexpr (!kAhead) {
        const Row<float, ODD> pre(q.part, run, a.cols), post(q.part + q.part_stride, run, a.cols);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float s[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = held[0][j * 8 + e][lane];
            pre.store(j * NT + lane, s);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = held[1][j * 8 + e][lane];
            if (a.post) post.store(j * NT + lane, s);
        }
    }
    // the teams' sums are added in order, by the first
    auto finish = [&](auto& s, int which) {
        if constexpr (kTeams > 1) {
            __syncthreads();
            if (team > 0) {
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e) join[team - 1][(j * 8 + e) * NT + lane] = s[j][e];
            }
            __syncthreads();
            if (team > 0) return;
#pragma unroll
            for (int k = 0; k < kTeams - 1; ++k)
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e) s[j][e] += join[k][(j * 8 + e) * NT + lane];
        }
        const Row<float, ODD> p(q.part + which * q.part_stride, run, a.cols);
#pragma unroll
        for (int j = 0; j < NV; ++j) p.store(j * NT + lane, s[j]);
    };
    if constexpr (kAhead) {
        finish(dpre, 0);
        if (a.post) finish(dpost, 1);
    }
    if (a.gate && q.per_group) finish(dgate, 2);
}

// Adds the runs' sums: blockIdx.y 0 the pre weight, 1 the post weight, 2 + g gate g.
// 64 columns a workgroup, 16 threads a column; the order is fixed.
struct RunSumArgs {
    const float* part;
    long long part_stride, runs, per_group;
    int cols;
    void *gpre, *gpost, *ggate;
};

template <class T>
__global__ __launch_bounds__(1024) void k_run_sum(RunSumArgs a) {
    constexpr int kCols = 64, kLanes = 1024 / kCols, kAhead = 4;
    __shared__ float sh[kLanes][kCols];
    const int what = (int)min(blockIdx.y, 2u);
    if (what == 1 && !a.gpost) return;
    const int col = blockIdx.x * kCols + threadIdx.x % kCols, lane = threadIdx.x / kCols;
    long long b = 0, e = a.runs;
    if (what == 2) {
        b = (long long)(blockIdx.y - 2) * a.per_group;
        e = min(b + a.per_group, a.runs);
    }
    const float* p = a.part + what * a.part_stride + col;
    float s[kAhead] = {};
    if (col < a.cols) {
        long long i = b + lane;
        for (; i + (kAhead - 1) * kLanes < e; i += kAhead * kLanes)
#pragma unroll
            for (int k = 0; k < kAhead; ++k) s[k] += p[(i + k * kLanes) * a.cols];
        for (; i < e; i += kLanes) s[0] += p[i * a.cols];
    }
    sh[lane][threadIdx.x % kCols] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (lane != 0 || col >= a.cols) return;
    float t = sh[0][threadIdx.x];
#pragma unroll
    for (int i = 1; i < kLanes; ++i) t += sh[i][threadIdx.x];
    T* out = static_cast<T*>(what == 0 ? a.gpre : what == 1 ? a.gpost : a.ggate);
    if (what == 2) out += (long long)(blockIdx.y - 2) * a.cols;
    out[col] = (T)t;
}

// ---- host ---------------------------------------------------------------------------
int check_block(const tpr_gated_norm_desc* d, const char* who, DropArgs& drop) {
    const std::string w = std::string(who) + ": ";
    if (!d) return fail(TPR_ERR_INVALID_ARG, w + "null descriptor");
    if (!is_elem(d->dtype)) return fail(TPR_ERR_UNSUPPORTED_DTYPE, w + "x must be float32, float16 or bfloat16");
    if (d->residual_dtype != d->dtype && d->residual_dtype != TPR_FLOAT32)
        return fail(TPR_ERR_UNSUPPORTED_DTYPE, w + "the residual must be of x's type or float32");
    if (d->rows < 0 || d->cols < 0 || d->gates < 0) return fail(TPR_ERR_INVALID_ARG, w + "negative extent");
    if (d->cols > TPR_GATED_NORM_MAX_COLS) return fail(TPR_ERR_NOT_IMPLEMENTED, w + "more than 16384 columns");
    if (d->rows >= (1LL << 30)) return fail(TPR_ERR_INVALID_ARG, w + "2^30 rows or more");
    if (d->gates > 0 && d->rows % d->gates != 0) return fail(TPR_ERR_INVALID_ARG, w + "gates must divide the rows");
    if (!(d->eps >= 0.0) || !std::isfinite(d->eps)) return fail(TPR_ERR_INVALID_ARG, w + "eps must not be negative");
    if (!std::isfinite(d->residual_scale)) return fail(TPR_ERR_INVALID_ARG, w + "residual_scale must be finite");
    if (!drop_args(d->p, d->seed, d->offset, drop))
        return fail(TPR_ERR_INVALID_ARG, w + "p must be in [0, 1) and leave something of each 2^16");
    return TPR_OK;
}

BlockArgs block_args(const tpr_gated_norm_desc* d, const DropArgs& drop) {
    BlockArgs a{};
    a.rows = (int)d->rows;
    a.group = FastDiv((uint32_t)(d->gates > 0 ? d->rows / d->gates : d->rows));
    a.cols = (int)d->cols;
    a.inv_cols = (float)(1.0 / (double)d->cols);
    a.eps = (float)d->eps;
    a.scale = (float)d->residual_scale;
    a.d = drop;
    return a;
}

template <int N>
using Int = std::integral_constant<int, N>;

// The threads a row takes, with one or two vectors of 8 columns each: a wave up to 1024
// columns, then a workgroup of 256 to 1024.  per_cu: workgroups of the backward kernel
// that a CU's registers hold.
struct Layout {
    int columns, threads, per_cu;
};
constexpr Layout kLayouts[] = {{512, 64, 4},  {1024, 64, 2},   {2048, 256, 4}, {4096, 512, 2},
                               {6144, 768, 1}, {8192, 1024, 1}, {12288, 512, 1}, {16384, 512, 1}};
int layout_of(int64_t cols) {
    int i = 0;
    while (kLayouts[i].columns < cols) ++i;
    return i;
}

// Calls fn(T, R, NT, NV, ODD) for a descriptor's types and layout.
template <class F>
int with_layout(const tpr_gated_norm_desc* d, F&& fn) {
    return with_elem(d->dtype, [&](auto t) -> int {
        auto with_res = [&](auto r) -> int {
            auto with_odd = [&](auto odd) -> int {
                auto go = [&](auto nt, auto nv) { return fn(t, r, nt, nv, odd); };
                switch (layout_of(d->cols)) {
                    case 0: return fn(t, r, Int<64>{}, Int<1>{}, Int<2 * decltype(odd)::value>{});
                    case 1: return go(Int<64>{}, Int<2>{});
                    case 2: return go(Int<256>{}, Int<1>{});
                    case 3: return go(Int<512>{}, Int<1>{});
                    case 4: return go(Int<768>{}, Int<1>{});
                    case 5: return go(Int<1024>{}, Int<1>{});
                    case 6: return go(Int<512>{}, Int<3>{});
                    default: return go(Int<512>{}, Int<4>{});
                }
            };
            return d->cols % 8 ? with_odd(Int<1>{}) : with_odd(Int<0>{});
        };
        if constexpr (std::is_same<decltype(t), float>::value) return with_res(t);
        else return d->residual_dtype == TPR_FLOAT32 ? with_res(float{}) : with_res(t);
    });
}

struct RunPlan {
    long long run, per_group, groups, runs;
};

// Runs of rows for the sums over rows: as many as there are workgroups on the card, of
// a row for each team at least.  A gate whose group is shorter than a run is summed
// within one run, and written by it.
RunPlan run_plan(const tpr_gated_norm_desc* d) {
    RunPlan p{};
    if (d->rows == 0) return p;
    const Layout& l = kLayouts[layout_of(d->cols)];
    const int teams = l.threads < kBlk ? kBlk / l.threads : 1;
    const long long most = (long long)device_info().cus * l.per_cu;
    p.run = std::max<long long>((d->rows + most - 1) / most, teams);
    const long long groups = d->gates > 0 ? d->gates : 1, group = d->rows / groups;
    if (group >= p.run) {
        p.per_group = (group + p.run - 1) / p.run;
        p.runs = p.per_group * groups;
    } else {
        p.groups = p.run / group;
        p.runs = (groups + p.groups - 1) / p.groups;
    }
    return p;
}

}  // namespace
}  // namespace tpr

using namespace tpr;

extern "C" int tpr_dropout(const void* in, int32_t dtype, int64_t rows, int64_t cols, double p, int64_t seed,
                           int64_t offset, void* out, void* stream) {
    const std::string who = "tpr_dropout: ";
    if (!is_elem(dtype)) return fail(TPR_ERR_UNSUPPORTED_DTYPE, who + "float32, float16 or bfloat16 only");
    if (rows < 0 || cols < 0) return fail(TPR_ERR_INVALID_ARG, who + "negative extent");
    DropArgs drop;
    if (!drop_args(p, seed, offset, drop))
        return fail(TPR_ERR_INVALID_ARG, who + "p must be in [0, 1) and leave something of each 2^16");
    if (rows == 0 || cols == 0) return TPR_OK;
    if (rows > (1LL << 32) || cols > (1LL << 34))
        return fail(TPR_ERR_INVALID_ARG, who + "more than 2^32 rows or 2^34 columns");
    if (!in || !out) return fail(TPR_ERR_INVALID_ARG, who + "null pointer");
    const long long vecs = (cols + 7) / 8, most = kMaxThreads / kBlk * kBlk;  // vecs < most
    return with_elem(dtype, [&](auto t) -> int {
        using T = decltype(t);
        for (long long r0 = 0; r0 < rows; r0 += most / vecs) {
            const long long n = std::min(most / vecs, (long long)rows - r0);
            DropoutArgs a{static_cast<const T*>(in) + r0 * cols, static_cast<T*>(out) + r0 * cols, drop,
                          FastDiv((uint32_t)vecs), (uint32_t)(n * vecs), (uint32_t)r0, cols};
            auto kernel = k_dropout<T, false>;
            if constexpr (sizeof(T) == 2)
                if (rows * cols * 2 >= kDropoutPass) kernel = k_dropout<T, true>;
            hipLaunchKernelGGL(kernel, dim3((unsigned)((n * vecs + kBlk - 1) / kBlk)), dim3(kBlk), 0,
                               static_cast<hipStream_t>(stream), a);
            const int rc = check_launch("tpr_dropout");
            if (rc != TPR_OK) return rc;
        }
        return TPR_OK;
    });
}

extern "C" int tpr_gated_norm(const tpr_gated_norm_desc* desc, const void* x, const void* h, const void* pre_weight,
                              const void* post_weight, const void* gate, void* out, void* y, float* rstd_post,
                              float* rstd_pre, void* stream) {
    const char* who = "tpr_gated_norm";
    DropArgs drop;
    const int rc = check_block(desc, who, drop);
    if (rc != TPR_OK) return rc;
    if (desc->rows == 0) return TPR_OK;
    if (desc->cols == 0) {
        if (!rstd_post && !rstd_pre) return TPR_OK;
        hipLaunchKernelGGL(k_no_columns, dim3((unsigned)((desc->rows + kBlk - 1) / kBlk)), dim3(kBlk), 0,
                           static_cast<hipStream_t>(stream), rstd_post, rstd_pre, desc->rows);
        return check_launch(who);
    }
    if (!x || !h || !pre_weight || !out || !y || !rstd_pre || (post_weight && !rstd_post) || (desc->gates > 0 && !gate))
        return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": null pointer");
    BlockArgs a = block_args(desc, drop);
    a.x = x;
    a.h = h;
    a.pre = pre_weight;
    a.post = post_weight;
    a.gate = desc->gates > 0 ? gate : nullptr;
    a.out = out;
    a.y = y;
    a.rstd_post = rstd_post;
    a.rstd_pre = rstd_pre;
    return with_layout(desc, [&](auto t, auto r, auto nt, auto nv, auto odd) -> int {
        constexpr int NT = decltype(nt)::value, kThreads = Team<NT>::kThreads, kTeams = Team<NT>::kTeams;
        const long long most = kMaxThreads / kThreads * kTeams;
        if (a.rows > most) return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": too many rows");
        hipLaunchKernelGGL((k_block_fwd<decltype(t), decltype(r), NT, decltype(nv)::value, decltype(odd)::value>),
                           dim3((unsigned)((a.rows + kTeams - 1) / kTeams)), dim3(kThreads), 0,
                           static_cast<hipStream_t>(stream), a);
        return check_launch(who);
    });
}

extern "C" size_t tpr_gated_norm_backward_workspace_bytes(const tpr_gated_norm_desc* desc) {
    DropArgs drop;
    if (check_block(desc, "tpr_gated_norm_backward", drop) != TPR_OK) return 0;
    const RunPlan p = run_plan(desc);
    return (size_t)p.runs * desc->cols * sizeof(float) * (desc->gates > 0 && p.per_group ? 3 : 2);
}

extern "C" int tpr_gated_norm_backward(const tpr_gated_norm_desc* desc, const void* grad_y, const void* grad_out,
                                       const void* x, const void* out, const float* rstd_post, const float* rstd_pre,
                                       const void* pre_weight, const void* post_weight, const void* gate, void* grad_x,
                                       void* grad_h, void* grad_pre, void* grad_post, void* grad_gate, void* workspace,
                                       size_t workspace_bytes, void* stream) {
    const char* who = "tpr_gated_norm_backward";
    DropArgs drop;
    int rc = check_block(desc, who, drop);
    if (rc != TPR_OK) return rc;
    if (desc->cols == 0) return TPR_OK;
    if (!grad_pre || (post_weight && !grad_post) || (desc->gates > 0 && !grad_gate))
        return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": null pointer");
    if (desc->rows > 0 && (!grad_y || !x || !out || !rstd_pre || !pre_weight || !grad_x || !grad_h ||
                           (post_weight && !rstd_post) || (desc->gates > 0 && !gate)))
        return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": null pointer");
    const size_t need = tpr_gated_norm_backward_workspace_bytes(desc);
    if (need && (!workspace || workspace_bytes < need))
        return fail(TPR_ERR_WORKSPACE,
                    std::string(who) + ": workspace smaller than tpr_gated_norm_backward_workspace_bytes");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const RunPlan p = run_plan(desc);
    BlockBwdArgs q{};
    q.part = static_cast<float*>(workspace);
    q.part_stride = p.runs * desc->cols;
    if (desc->rows > 0) {
        q.b = block_args(desc, drop);
        q.b.x = x;
        q.b.h = out;
        q.b.pre = pre_weight;
        q.b.post = post_weight;
        q.b.gate = desc->gates > 0 ? gate : nullptr;
        q.b.rstd_post = const_cast<float*>(rstd_post);
        q.b.rstd_pre = const_cast<float*>(rstd_pre);
        q.gy = grad_y;
        q.gout = grad_out;
        q.gx = grad_x;
        q.gh = grad_h;
        q.ggate = grad_gate;
        q.run = (int)p.run;
        q.per_group = (int)p.per_group;
        q.groups = (int)p.groups;
        rc = with_layout(desc, [&](auto t, auto r, auto nt, auto nv, auto odd) -> int {
            constexpr int NT = decltype(nt)::value;
            hipLaunchKernelGGL((k_block_bwd<decltype(t), decltype(r), NT, decltype(nv)::value, decltype(odd)::value>),
                               dim3((unsigned)p.runs), dim3(Team<NT>::kThreads), 0, st, q);
            return check_launch(who);
        });
        if (rc != TPR_OK) return rc;
    }
    RunSumArgs a{q.part, q.part_stride, p.runs, p.per_group, (int)desc->cols, grad_pre,
                 post_weight ? grad_post : nullptr, grad_gate};
    // gates that their runs have written need no sum; without rows theirs is 0
    const long long sums = 2 + (desc->gates > 0 && (p.per_group || desc->rows == 0) ? desc->gates : 0);
    if (sums > 65535) return fail(TPR_ERR_INVALID_ARG, std::string(who) + ": too many gates for no rows");
    return with_elem(desc->dtype, [&](auto t) -> int {
        hipLaunchKernelGGL(k_run_sum<decltype(t)>, dim3((unsigned)((desc->cols + 63) / 64), (unsigned)sums), dim3(1024), 0,
                           st, a);
        return check_launch(who);
    });
}
