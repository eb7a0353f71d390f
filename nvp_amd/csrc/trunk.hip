// The gated residual step of a conditioning stack with the norms on both sides of its block, forward and backward (rows of D values):
//     r1 = (mean h^2 + eps)^-1/2   n = h r1   y = x + s a(g) n p        (p: the norm behind the block, g: its gate, s: the residual scale)
//     r2 = (mean y^2 + eps)^-1/2   v = y r2   u = v w                   (w: the norm in front of the next block; from y before it is rounded)
// FORM both: y and u; last: y only; first: no h, u = norm(x) only.  a is the identity or the sigmoid; a gate row serves `share` rows of x.
// Backward, E = dL/dy in all:  dv = du w,  c2 = mean(dv v),  E = dy + r2 (dv - v c2),  dx = E,
//     dn = s a p E,  c1 = mean(dn n),  dh = r1 (dn - n c1),  dg = s E n p a'(g),  dp = sum s a E n,  dw = sum du v.
// c1 needs E and so c2; written out it is s [sum q (dy + r2 dv) - r2 c2 sum q v] / D with q = a p n: three sums that need neither, so both means come from
// ONE reduction per row instead of two in sequence.  r1, r2 are kept from forward (8 bytes per row); n, a, y, v are computed again from x, h, g.
// All arithmetic and every sum is fp32; each result is rounded once to its type.  Bound by memory: 4 - 5 streams forward, 6 (shared gate) to 8 backward, each touched once.
// One row is held in registers by a team of TEAM lanes, 8 values each (12 above 4096, 16 above 6144), in 16-byte accesses: V = 8 of 16 bits, 4 of 32.
// Measured: 16384 x 2048 bf16 with shared gates, forward 55 us (268 MB, 4.9 TB/s), backward 85 us (403 MB, 4.7 TB/s) and 4.5 us for the partial rows; 65536 x 4096
// forward 530 - 580 us (2.68 GB, 4.6 - 5.1 TB/s): the rate of a large copy.  Above 4096 columns the backward kernel runs
// short of registers: 16384 x 5000 at 4.6 - 4.7 TB/s, 8192 x 8192 at 4.3 - 4.6 (teams of 1024 lanes with 8 values each leave 128 registers per lane, spill, and
// reach 0.6 - 2.6).
#include "stream_types.h"

namespace {

enum { kBoth = 0, kFirst = 1, kLast = 2 };

// sum over a team of `TEAM` consecutive lanes; every lane gets the result, bit-identical in every lane (butterfly; across waves: same order everywhere)
template <int TEAM, int N> __device__ __forceinline__ void team_sum(float (&s)[N], float* red, int& flip) {
#pragma unroll
    for (int o = (TEAM < 64 ? TEAM : 64) / 2; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) s[k] += __shfl_xor(s[k], o);
    if (TEAM > 64) {
        constexpr int W = TEAM / 64;
        float* r = red + flip * (W * N);                       // two alternating buffers: one barrier per reduction
        flip ^= 1;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < N; ++k) r[(threadIdx.x >> 6) * N + k] = s[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) {
            float t = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) t += r[w * N + k];
            s[k] = t;
        }
    }
}

// number of this thread's team in its workgroup: a scalar wherever a wave belongs to one team, so that row addresses are scalars too
template <int TEAM, int TEAMS> __device__ __forceinline__ int team_index() {
    if (TEAMS == 1) return 0;
    const int t = threadIdx.x / TEAM;
    return TEAM >= 64 ? __builtin_amdgcn_readfirstlane(t) : t;
}

// A row as a team holds it: vectors of V, team-strided, so that a wave's access is contiguous.  Value j = k * V + e of a lane is column col(k) + e.
// Where V divides the width (ODD false) a lane behind the last column reads column 0 and holds zeros.  Where it does not (ODD), the vectors that reach behind the
// end are moved back to end there: some columns are then held twice, with the same values and so the same results (they are stored twice), and only sums
// across the row have to drop the second copy (keep()).  Loads are unconditional: no branch separates the loads of several rows, and nothing waits for them
// before they are converted.
template <typename T, int TEAM, int V, int VALS, bool ODD> struct row_of {
    nvp_vec<T, V> q[VALS / V];
    static __device__ __forceinline__ int col(int k, int lane, int dim) {
        const int c = (k * TEAM + lane) * V;
        return ODD ? min(c, dim - V) : c < dim ? c : 0;
    }
    static __device__ __forceinline__ bool inside(int k, int lane, int dim) { return (k * TEAM + lane) * V < dim; }
    static __device__ __forceinline__ bool keep(int j, int lane, int dim) { return !ODD || col(j / V, lane, dim) + j % V >= (j / V * TEAM + lane) * V; }
    __device__ __forceinline__ void load(const T* __restrict__ p, int lane, int dim) {
#pragma unroll
        for (int k = 0; k < VALS / V; ++k) q[k] = nvp_load_raw<T, V>(p + col(k, lane, dim));
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int k = 0; k < VALS / V; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) q[k].v[e] = (T)0.f;
    }
    __device__ __forceinline__ void get(float (&f)[VALS], int lane, int dim) const {
#pragma unroll
        for (int k = 0; k < VALS / V; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) f[k * V + e] = ODD || inside(k, lane, dim) ? (float)q[k].v[e] : 0.f;
    }
    static __device__ __forceinline__ void put(T* __restrict__ p, int lane, int dim, const float (&f)[VALS]) {
#pragma unroll
        for (int k = 0; k < VALS / V; ++k) {
            float t[V];
#pragma unroll
            for (int e = 0; e < V; ++e) t[e] = f[k * V + e];
            if (inside(k, lane, dim)) nvp_store<T, V>(p + col(k, lane, dim), t);
        }
    }
};
template <typename T, int TEAM, int V, int VALS, bool ODD> __device__ __forceinline__ void load_row(const T* __restrict__ p, int lane, int dim, float (&f)[VALS]) {
    row_of<T, TEAM, V, VALS, ODD> r;
    r.load(p, lane, dim);
    r.get(f, lane, dim);
}

// The sigmoid.  exp2(-g log2 e) is off by half an ulp of its argument, |g| / 2 * 2^-24 of the result on top of the rest (40 * 2^-24 at |g| = 80): nothing beside a 16-bit stream's
// rounding (2^-9, 2^-12 of it), so those stop there.  fp32 streams take exp(-|g|) = e + e (r ln 2 - |g| c'), e = exp2(x), x = -|g| fp32(log2 e) rounded, r what that rounding
// lost, c' = 1 - ln 2 * fp32(log2 e): two roundings, wherever g is.  Beyond 104 the result is 0; a NaN stays one.
__device__ __forceinline__ float exp_minus_abs(float g) {
    float m = fabsf(g);
    m = m > 104.f ? 104.f : m;
    const float x = -1.44269504f * m, e = __builtin_amdgcn_exp2f(x), r = __fmaf_rn(-1.44269504f, m, -x);
    return __fmaf_rn(e, __fmaf_rn(r, 0.693147182f, -1.33497582e-8f * m), e);
}
// Its derivative as t a^2, t = exp(-g), and not as a (1 - a), which cancels for open gates (1 - a from a rounded a is off by 2^-24 / (1 - a) of itself: 1 % at g = 12, all of it
// from 17 on).
template <typename T> __device__ __forceinline__ float sigmoid(float g, float& slope) {
    if constexpr (sizeof(T) < 4) {
        const float t = __builtin_amdgcn_exp2f(-1.44269504f * g), a = __builtin_amdgcn_rcpf(1.f + t);
        slope = fminf(t, 1e38f) * a * a;                        // (t infinite: a is 0; a NaN is in a)
        return a;
    } else {
        const float t = exp_minus_abs(g), r = __builtin_amdgcn_rcpf(1.f + t), m = t * r;
        slope = m * r;
        return g < 0.f ? m : r;
    }
}
// Both in one register, where registers are short: m = t / (1 + t), t = exp(-|g|), is the smaller of a and 1 - a; a closed gate (g < 0) is kept as a, an open one as -(1 - a).
template <typename T> __device__ __forceinline__ float gate_side(float g) {
    const float t = sizeof(T) < 4 ? __builtin_amdgcn_exp2f(-1.44269504f * fabsf(g)) : exp_minus_abs(g);
    return copysignf(t * __builtin_amdgcn_rcpf(1.f + t), -g);
}
__device__ __forceinline__ float open_of(float s, int act) { return act && __float_as_int(s) < 0 ? 1.f + s : s; }      // act 0: s is the gate itself
__device__ __forceinline__ float slope_of(float s, int act) { return act ? __fmaf_rn(-s, s, fabsf(s)) : 1.f; }
__device__ __forceinline__ float inv_rms(float sum, float inv_dim, float eps) { return 1.f / sqrtf(sum * inv_dim + eps); }

struct Rows {
    int64_t rows, share;
    int dim, act;
    float scale, eps, inv_dim;
};

constexpr int threads_of(int team) { return team > 64 ? team : 256; }      // a team that spans waves is a workgroup

template <typename T, typename W, int FORM, int TEAM, int V, int VALS, bool ODD>
__global__ __launch_bounds__(threads_of(TEAM)) void residual_fwd_kernel(const T* __restrict__ x, const T* __restrict__ h, const T* __restrict__ gate, const W* __restrict__ post,
                                                                        const W* __restrict__ next, T* __restrict__ y, T* __restrict__ u, float* __restrict__ stats, Rows R) {
    constexpr int kTeams = threads_of(TEAM) / TEAM;
    typedef row_of<T, TEAM, V, VALS, ODD> Row;
    constexpr bool kAhead = VALS <= 12;                         // registers for a second row?
    __shared__ float red[TEAM > 64 ? 2 * TEAM / 64 : 1];
    int flip = 0;
    const int lane = kTeams == 1 ? threadIdx.x : threadIdx.x % TEAM, team = team_index<TEAM, kTeams>();
    const int64_t step = (int64_t)gridDim.x * kTeams;
    int64_t row = (int64_t)blockIdx.x * kTeams + team;
    if (row >= R.rows) return;                                  // whole teams; a team that spans waves is a workgroup
    Row rx, rh, rg;                                             // the next row's, one row ahead
    if (FORM != kFirst) rg.zero();
    const auto fetch = [&](int64_t r) {
        rx.load(x + r * R.dim, lane, R.dim);
        if (FORM != kFirst) {
            rh.load(h + r * R.dim, lane, R.dim);
            if (gate) rg.load(gate + (R.share == 1 ? r : (int64_t)((uint32_t)r / (uint32_t)R.share)) * R.dim, lane, R.dim);
        }
    };
    if (kAhead) fetch(row);
    float p[VALS], w[VALS];
    if (FORM != kFirst) load_row<W, TEAM, V, VALS, ODD>(post, lane, R.dim, p);
    if (FORM != kLast) load_row<W, TEAM, V, VALS, ODD>(next, lane, R.dim, w);
#pragma unroll 1
    for (; row < R.rows; row += step) {
        float yv[VALS], hv[VALS], a[VALS], r1 = 0.f, r2 = 0.f;
        if (!kAhead) fetch(row);
        rx.get(yv, lane, R.dim);
        if (FORM != kFirst) {
            rh.get(hv, lane, R.dim);
            rg.get(a, lane, R.dim);
        }
        if (kAhead && row + step < R.rows) fetch(row + step);
        if (FORM != kFirst) {
            float s[1] = {0.f};
#pragma unroll
            for (int j = 0; j < VALS; ++j)
                if (Row::keep(j, lane, R.dim)) s[0] = __fmaf_rn(hv[j], hv[j], s[0]);
            team_sum<TEAM, 1>(s, red, flip);
            r1 = inv_rms(s[0], R.inv_dim, R.eps);
            if (!gate) {
#pragma unroll
                for (int j = 0; j < VALS; ++j) a[j] = 1.f;
            } else if (R.act) {
#pragma unroll
                for (int j = 0; j < VALS; ++j) {
                    float unused;
                    a[j] = sigmoid<T>(a[j], unused);
                }
            }
#pragma unroll
            for (int j = 0; j < VALS; ++j) yv[j] = __fmaf_rn(R.scale * a[j] * p[j], hv[j] * r1, yv[j]);
            Row::put(y + row * R.dim, lane, R.dim, yv);
        }
        if (FORM != kLast) {
            float s[1] = {0.f};
#pragma unroll
            for (int j = 0; j < VALS; ++j)
                if (Row::keep(j, lane, R.dim)) s[0] = __fmaf_rn(yv[j], yv[j], s[0]);      // columns behind the last one hold zeros
            team_sum<TEAM, 1>(s, red, flip);
            r2 = inv_rms(s[0], R.inv_dim, R.eps);
#pragma unroll
            for (int j = 0; j < VALS; ++j) yv[j] = yv[j] * r2 * w[j];
            Row::put(u + row * R.dim, lane, R.dim, yv);
        }
        if (stats && lane == 0) *reinterpret_cast<float2*>(stats + 2 * row) = make_float2(r1, r2);
    }
}

// Rows are cut into units of at most `unit` rows that lie within one gate row's share; a team walks whole units, so a shared gate's gradient (SUMMED) is added
// up in registers (a unit that is only a piece of the share leaves a partial sum).  dp and dw are summed over everything the workgroup has seen, the workgroup's
// teams are added through LDS, and one partial row per workgroup goes to the workspace.  residual_reduce_kernel adds partial rows in a fixed order: no atomics,
// results do not vary from run to run.
struct Units {
    int64_t units, per_share;      // units in all; units per group of rows that share a gate row (1 group of all rows where no gate row is shared)
    int64_t share, unit;           // rows per such group, rows per unit
};

template <typename T, typename W, int FORM, bool SUMMED, int TEAM, int V, int VALS, bool ODD>
__global__ __launch_bounds__(threads_of(TEAM)) void residual_bwd_kernel(const T* __restrict__ x, const T* __restrict__ h, const T* __restrict__ gate, const W* __restrict__ post,
                                                                        const W* __restrict__ next, const float* __restrict__ stats, const T* __restrict__ dy, const T* __restrict__ du,
                                                                        T* __restrict__ dx, T* __restrict__ dh, T* __restrict__ dgate, float* __restrict__ dgate_part,
                                                                        float* __restrict__ dpost_part, float* __restrict__ dnext_part, Rows R, Units U) {
    constexpr int kTeams = threads_of(TEAM) / TEAM, N = FORM == kBoth ? 3 : 1;
    typedef row_of<T, TEAM, V, VALS, ODD> Row;
    constexpr bool kAhead = VALS == 8 || (VALS == 12 && sizeof(T) == 2);      // registers for a second row? (12 values, fp32: 434 us without, 444 with, 16384 x 4104)
    constexpr bool kSide = !SUMMED && VALS > 8;                 // (8192 x 8192 fp32: 498 us with one register for gate and slope, 560 with two)
    __shared__ float red[TEAM > 64 ? 2 * N * TEAM / 64 : 1];
    __shared__ float comb[kTeams > 1 ? kTeams : 1][kTeams > 1 ? TEAM * VALS : 1];
    int flip = 0;
    const int lane = kTeams == 1 ? threadIdx.x : threadIdx.x % TEAM, team = team_index<TEAM, kTeams>();
    float p[VALS], w[VALS], sp[VALS], sw[VALS];
#pragma unroll
    for (int j = 0; j < VALS; ++j) sp[j] = sw[j] = 0.f;
    if (FORM != kFirst) load_row<W, TEAM, V, VALS, ODD>(post, lane, R.dim, p);
    if (FORM != kLast) load_row<W, TEAM, V, VALS, ODD>(next, lane, R.dim, w);
    Row rx, rh, rg, re, rd;                                     // the next row's, one row ahead
    float2 rst;
    rg.zero();
    re.zero();
    rd.zero();
    const auto fetch = [&](int64_t r) {
        rst = *reinterpret_cast<const float2*>(stats + 2 * r);
        if (FORM != kLast) rx.load(x + r * R.dim, lane, R.dim);
        if (FORM != kFirst) rh.load(h + r * R.dim, lane, R.dim);
        if (FORM != kFirst && !SUMMED && gate) rg.load(gate + r * R.dim, lane, R.dim);
        if (FORM != kFirst && dy) re.load(dy + r * R.dim, lane, R.dim);
        if (FORM != kLast && du) rd.load(du + r * R.dim, lane, R.dim);
    };
#pragma unroll 1
    for (int64_t un = (int64_t)blockIdx.x * kTeams + team; un < U.units; un += (int64_t)gridDim.x * kTeams) {
        const int64_t grp = un / U.per_share, piece = un - grp * U.per_share;
        const int64_t first = grp * U.share + piece * U.unit, last = min(first + U.unit, (grp + 1) * U.share);
        float a[VALS], da[VALS], sg[VALS];                      // act(g) (kSide: gate_side(g)), its derivative, the sum of the gate's gradient
        if (kAhead) fetch(first);
        if (SUMMED) {
            load_row<T, TEAM, V, VALS, ODD>(gate + grp * R.dim, lane, R.dim, a);
#pragma unroll
            for (int j = 0; j < VALS; ++j) {
                da[j] = 1.f;
                if (R.act) a[j] = sigmoid<T>(a[j], da[j]);
                sg[j] = 0.f;
            }
        }
#pragma unroll 1
        for (int64_t row = first; row < last; ++row) {
            float xv[VALS], n[VALS], e[VALS], dv[VALS];
            if (!kAhead) fetch(row);
            const float2 st = rst;
            if (FORM != kLast) rx.get(xv, lane, R.dim);
            if (FORM != kFirst) rh.get(n, lane, R.dim);
            if (FORM != kFirst && !SUMMED) rg.get(a, lane, R.dim);
            re.get(e, lane, R.dim);
            rd.get(dv, lane, R.dim);
            if (kAhead && row + 1 < last) fetch(row + 1);
            if (FORM != kFirst && !SUMMED) {
#pragma unroll
                for (int j = 0; j < VALS; ++j) da[j] = 1.f;
                if (!gate) {
#pragma unroll
                    for (int j = 0; j < VALS; ++j) a[j] = 1.f;
                } else if (R.act) {
#pragma unroll
                    for (int j = 0; j < VALS; ++j) a[j] = kSide ? gate_side<T>(a[j]) : sigmoid<T>(a[j], da[j]);
                }
            }
            const int act = kSide && gate ? R.act : 0;
            float s[N];
#pragma unroll
            for (int k = 0; k < N; ++k) s[k] = 0.f;
#pragma unroll
            for (int j = 0; j < VALS; ++j) {
                float q = 0.f;
                if (FORM != kFirst) {
                    n[j] *= st.x;
                    q = open_of(a[j], act) * p[j] * n[j];
                }
                const bool keep = Row::keep(j, lane, R.dim);
                if (FORM == kLast) {
                    if (keep) s[0] = __fmaf_rn(q, e[j], s[0]);
                } else {
                    const float v = (FORM == kBoth ? __fmaf_rn(R.scale, q, xv[j]) : xv[j]) * st.y;
                    xv[j] = v;
                    sw[j] = __fmaf_rn(dv[j], v, sw[j]);
                    dv[j] *= w[j];
                    if (keep) s[0] = __fmaf_rn(dv[j], v, s[0]);
                    e[j] = __fmaf_rn(st.y, dv[j], e[j]);
                    if constexpr (FORM == kBoth) {
                        if (keep) {
                            s[N - 2] = __fmaf_rn(q, e[j], s[N - 2]);
                            s[N - 1] = __fmaf_rn(q, v, s[N - 1]);
                        }
                    }
                }
            }
            team_sum<TEAM, N>(s, red, flip);
            float c1 = 0.f;                                     // mean(dn n)
            if (FORM != kLast) {
                const float c2 = st.y * s[0] * R.inv_dim;
#pragma unroll
                for (int j = 0; j < VALS; ++j) e[j] = __fmaf_rn(-c2, xv[j], e[j]);
                if constexpr (FORM == kBoth) c1 = R.scale * R.inv_dim * (s[N - 2] - c2 * s[N - 1]);
            } else {
                c1 = R.scale * R.inv_dim * s[0];
            }
            if (dx) Row::put(dx + row * R.dim, lane, R.dim, e);
            if (FORM != kFirst) {
                float t[VALS];
                if (kSide)                                      // act(g) is worked out again from gate_side(g): the compiler is not to keep it from above
#pragma unroll
                    for (int j = 0; j < VALS; ++j) asm("" : "+v"(a[j]));
#pragma unroll
                for (int j = 0; j < VALS; ++j) {
                    const float en = R.scale * e[j] * n[j], open = open_of(a[j], act);
                    sp[j] = __fmaf_rn(open, en, sp[j]);
                    t[j] = en * p[j] * (kSide ? slope_of(a[j], act) : da[j]);
                    n[j] = st.x * __fmaf_rn(-c1, n[j], R.scale * open * p[j] * e[j]);
                }
                if (dh) Row::put(dh + row * R.dim, lane, R.dim, n);
                if (SUMMED) {
#pragma unroll
                    for (int j = 0; j < VALS; ++j) sg[j] += t[j];
                } else if (dgate) {
                    Row::put(dgate + row * R.dim, lane, R.dim, t);
                }
            }
        }
        if (SUMMED && dgate) {
            if (U.per_share == 1) Row::put(dgate + grp * R.dim, lane, R.dim, sg);
            else row_of<float, TEAM, V, VALS, ODD>::put(dgate_part + un * R.dim, lane, R.dim, sg);
        }
    }
    // one partial row per workgroup for each weight
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float* out = which ? dnext_part : dpost_part;
        if ((which ? FORM == kLast : FORM == kFirst) || !out) continue;
        if (kTeams > 1) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < VALS; ++j)
                if (Row::inside(j / V, lane, R.dim)) comb[team][Row::col(j / V, lane, R.dim) + j % V] = which ? sw[j] : sp[j];
            __syncthreads();
            for (int c = threadIdx.x; c < R.dim; c += 256) {
                float t = 0.f;
#pragma unroll
                for (int k = 0; k < kTeams; ++k) t += comb[k][c];
                out[(int64_t)blockIdx.x * R.dim + c] = t;
            }
        } else {
            row_of<float, TEAM, V, VALS, ODD>::put(out + (int64_t)blockIdx.x * R.dim, lane, R.dim, which ? sw : sp);
        }
    }
}

// out[j][c] = sum over `rows_of(job)` partial rows.  Jobs: 0 dpost, 1 dnext (rows = workgroups of the kernel above), 2 + g gate row g (rows = pieces).
// 32 columns x 32 row lanes per workgroup: every lane adds its rows in order, the lanes are added in order.
template <typename T, typename W>
__global__ __launch_bounds__(1024) void residual_reduce_kernel(const float* __restrict__ dpost_part, const float* __restrict__ dnext_part, const float* __restrict__ dgate_part,
                                                               W* __restrict__ dpost, W* __restrict__ dnext, T* __restrict__ dgate, int dim, int64_t groups, int64_t pieces) {
    __shared__ float part[32][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), r0 = threadIdx.x >> 5;
    const int job = blockIdx.y;
    const float* src = job == 0 ? dpost_part : job == 1 ? dnext_part : dgate_part + (int64_t)(job - 2) * pieces * dim;
    if ((job == 0 && !dpost) || (job == 1 && !dnext)) return;                  // uniform over the workgroup
    const int64_t rows = job < 2 ? groups : pieces;
    float s = 0.f;
    if (c < dim) {
        int64_t r = r0;
        for (; r + 7 * 32 < rows; r += 8 * 32) {                               // eight loads in flight, added in order
            float t[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) t[k] = src[(r + k * 32) * dim + c];
#pragma unroll
            for (int k = 0; k < 8; ++k) s += t[k];
        }
        for (; r < rows; r += 32) s += src[r * dim + c];
    }
    part[r0][threadIdx.x & 31] = s;
    __syncthreads();
    if (r0 == 0 && c < dim) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) t += part[k][threadIdx.x & 31];
        if (job == 0) dpost[c] = (W)t;
        else if (job == 1) dnext[c] = (W)t;
        else dgate[(int64_t)(job - 2) * dim + c] = (T)t;
    }
}

constexpr int kMaxDim = 8192;
// 8 values per lane; 12 above 4096, 16 above 6144.  The smallest team that holds the row (bf16, us, so / with a team of four times
// the lanes below 512 columns, twice above: 1 245 184 x 32 forward 97 / 169; 262 144 x 228 backward 230 / 238; 131 072 x 640 backward 283 / 512)
int team_of(int dim) { return dim <= 64 ? 8 : dim <= 128 ? 16 : dim <= 256 ? 32 : dim <= 512 ? 64 : dim <= 1024 ? 128 : dim <= 2048 ? 256 : 512; }

struct Plan {
    Units U;
    int64_t groups;        // workgroups of the backward kernel
    bool parts;            // gate gradients leave partial rows
    int64_t gate_rows;
};
Plan plan_of(const nvp_residual* a) {
    Plan P;
    const int team = team_of(a->dim), teams = threads_of(team) / team;
    const bool shared = a->gate && a->gate_rows < a->rows;
    P.gate_rows = shared ? a->gate_rows : 0;
    P.U.share = shared ? a->rows / a->gate_rows : a->rows;
    // as many workgroups as the chip holds at once (8 waves per CU at the kernel's registers): more would leave a second, partly filled round and more partial
    // rows to add up
    const int64_t wgs = 256 * 512 / threads_of(team), want = wgs * teams;
    const int64_t rows_per = (a->rows + want - 1) / want;
    P.U.unit = rows_per < P.U.share ? rows_per : P.U.share;
    P.U.per_share = (P.U.share + P.U.unit - 1) / P.U.unit;
    P.U.units = (shared ? a->gate_rows : 1) * P.U.per_share;
    P.parts = shared && P.U.per_share > 1;
    const int64_t g = (P.U.units + teams - 1) / teams;
    const int64_t most = wgs > 512 ? wgs : 512;
    P.groups = g < most ? g : most;
    return P;
}

int check(const nvp_residual* a) {
    if (!a || a->rows < 0 || a->rows > (1ll << 31) - 1 || a->dim < 1 || !nvp_type_size(a->type) || !nvp_type_size(a->weight_type)) return NVP_ERR_BADARG;
    if (a->weight_type != NVP_F32 && a->weight_type != a->type) return NVP_ERR_BADARG;
    if (a->gate_act < 0 || a->gate_act > 1 || !(a->eps >= 0.f)) return NVP_ERR_BADARG;
    if (!a->h && !a->next) return NVP_ERR_BADARG;
    if ((a->h != nullptr) != (a->post != nullptr) || (a->gate && !a->h)) return NVP_ERR_BADARG;
    if (a->gate && (a->gate_rows < 1 || (a->rows && (a->gate_rows > a->rows || a->rows % a->gate_rows)))) return NVP_ERR_BADARG;
    return a->dim > kMaxDim ? NVP_ERR_UNSUPPORTED : 0;
}

struct Call {
    const nvp_residual* a;
    void *y, *u, *dx, *dh, *dgate, *dpost, *dnext;
    float* stats;
    const void *dy, *du;
    float *dgate_part, *dpost_part, *dnext_part;
    Plan P;
    bool backward;
    hipStream_t st;
};

template <typename T, typename W, int FORM, int TEAM, int V, int VALS, bool ODD> int launch(const Call& c) {
    const nvp_residual* a = c.a;
    constexpr int kThreads = threads_of(TEAM), kTeams = kThreads / TEAM;
    const Rows R{a->rows, a->gate ? a->rows / a->gate_rows : 1, a->dim, a->gate_act, a->scale, a->eps, 1.f / (float)a->dim};
    if (!c.backward) {
        const int64_t need = (a->rows + kTeams - 1) / kTeams, cap = 256 * (2048 / kThreads);
        hipLaunchKernelGGL((residual_fwd_kernel<T, W, FORM, TEAM, V, VALS, ODD>), dim3((unsigned)(need < cap ? need : cap)), dim3(kThreads), 0, c.st, (const T*)a->x, (const T*)a->h,
                           (const T*)a->gate, (const W*)a->post, (const W*)a->next, (T*)c.y, (T*)c.u, c.stats, R);
        NVP_LAUNCH_CHECK();
        return 0;
    }
    const auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)c.P.groups), dim3(kThreads), 0, c.st, (const T*)a->x, (const T*)a->h, (const T*)a->gate, (const W*)a->post, (const W*)a->next, c.stats,
                           (const T*)c.dy, (const T*)c.du, (T*)c.dx, (T*)c.dh, (T*)c.dgate, c.dgate_part, c.dpost ? c.dpost_part : nullptr, c.dnext ? c.dnext_part : nullptr, R, c.P.U);
    };
    if constexpr (FORM != kFirst) {
        if (R.share > 1) go(residual_bwd_kernel<T, W, FORM, true, TEAM, V, VALS, ODD>);
        else go(residual_bwd_kernel<T, W, FORM, false, TEAM, V, VALS, ODD>);
    } else {
        go(residual_bwd_kernel<T, W, FORM, false, TEAM, V, VALS, ODD>);
    }
    NVP_LAUNCH_CHECK();
    const bool gsum = c.P.parts && c.dgate;
    if (c.dpost || c.dnext || gsum) {
        hipLaunchKernelGGL((residual_reduce_kernel<T, W>), dim3((unsigned)((a->dim + 31) / 32), (unsigned)(2 + (gsum ? c.P.gate_rows : 0))), dim3(1024), 0, c.st, c.dpost_part, c.dnext_part,
                           c.dgate_part, (W*)c.dpost, (W*)c.dnext, (T*)c.dgate, a->dim, c.P.groups, c.P.U.per_share);
        NVP_LAUNCH_CHECK();
    }
    return 0;
}

template <typename T, typename W, int FORM, bool ODD> int by_team(const Call& c) {
    constexpr int V = 16 / sizeof(T);
    switch (team_of(c.a->dim)) {
        case 8: return launch<T, W, FORM, 8, V, 8, ODD>(c);
        case 16: return launch<T, W, FORM, 16, V, 8, ODD>(c);
        case 32: return launch<T, W, FORM, 32, V, 8, ODD>(c);
        case 64: return launch<T, W, FORM, 64, V, 8, ODD>(c);
        case 128: return launch<T, W, FORM, 128, V, 8, ODD>(c);
        case 256: return launch<T, W, FORM, 256, V, 8, ODD>(c);
        default:
            if (c.a->dim <= 4096) return launch<T, W, FORM, 512, V, 8, ODD>(c);
            // 12 values per lane up to 6144, in accesses of four (16384 x 5000, backward: 287 us bf16, 555 us fp32; 16 values: 329, 802), 16 above (fp32 always
            // as an odd width: 8192 x 8192 in 498 us; the even way took 530 where this one took 469)
            return c.a->dim <= 6144 ? launch<T, W, FORM, 512, 4, 12, ODD>(c) : launch<T, W, FORM, 512, V, 16, ODD || V == 4>(c);
    }
}
template <typename T, typename W, int FORM> int by_width(const Call& c) {
    constexpr int V = 16 / sizeof(T);
    if (c.a->dim < V) return launch<T, W, FORM, 8, 1, 8, false>(c);
    return c.a->dim % V ? by_team<T, W, FORM, true>(c) : by_team<T, W, FORM, false>(c);
}
template <typename T, typename W> int by_form(const Call& c) {
    if (!c.a->h) return by_width<T, W, kFirst>(c);
    return c.a->next ? by_width<T, W, kBoth>(c) : by_width<T, W, kLast>(c);
}
int by_type(const Call& c) {
    const bool wide = c.a->weight_type == NVP_F32;
    if (c.a->type == NVP_F32) return by_form<float, float>(c);
    if (c.a->type == NVP_BF16) return wide ? by_form<nvp_bf16, float>(c) : by_form<nvp_bf16, nvp_bf16>(c);
    return wide ? by_form<nvp_f16, float>(c) : by_form<nvp_f16, nvp_f16>(c);
}

int64_t gate_part_rows(const Plan& P) { return P.parts ? P.U.units : 0; }

}  // namespace

extern "C" int nvp_residual_fwd(const nvp_residual* a, void* y, void* u, float* stats, void* stream) {
    const int rc = check(a);
    if (rc) return rc;
    if (a->rows == 0) return 0;
    if (!a->x || (a->h && !y) || (a->next && !u)) return NVP_ERR_BADARG;
    Call c{};
    c.a = a;
    c.y = y;
    c.u = u;
    c.stats = stats;
    c.st = (hipStream_t)stream;
    return by_type(c);
}

extern "C" int64_t nvp_residual_bwd_workspace_bytes(const nvp_residual* a) {
    const int rc = check(a);
    if (rc) return rc;
    if (a->rows == 0) return 0;
    const Plan P = plan_of(a);
    return (gate_part_rows(P) + P.groups * ((a->h ? 1 : 0) + (a->next ? 1 : 0))) * a->dim * 4;
}

extern "C" int nvp_residual_bwd(const nvp_residual* a, const float* stats, const void* dy, const void* du, void* dx, void* dh, void* dgate, void* dpost, void* dnext, void* workspace,
                                int64_t workspace_bytes, void* stream) {
    const int rc = check(a);
    if (rc) return rc;
    if (a->rows == 0) return 0;
    if (!a->x || !stats || workspace_bytes < nvp_residual_bwd_workspace_bytes(a) || !workspace || ((uintptr_t)workspace & 15)) return NVP_ERR_BADARG;
    if ((!a->h && (dh || dpost || dy)) || (!a->next && (dnext || du)) || (!a->gate && dgate)) return NVP_ERR_BADARG;
    Call c{};
    c.a = a;
    c.backward = true;
    c.stats = const_cast<float*>(stats);
    c.dy = dy;
    c.du = du;
    c.dx = dx;
    c.dh = dh;
    c.dgate = dgate;
    c.dpost = dpost;
    c.dnext = dnext;
    c.P = plan_of(a);
    c.dgate_part = (float*)workspace;
    c.dpost_part = c.dgate_part + gate_part_rows(c.P) * a->dim;
    c.dnext_part = c.dpost_part + (a->h ? c.P.groups * a->dim : 0);
    c.st = (hipStream_t)stream;
    return by_type(c);
}
