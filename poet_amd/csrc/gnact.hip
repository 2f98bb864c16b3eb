// GroupNorm with an activation on channels-last rows for gfx950, forward and backward.
//
//   forward :  m, v over the HW x (C / G) values of (image n, group g);  h = (x - m) / sqrt(v + eps);  y = act(gamma h + beta)
//   backward:  z = gamma h + beta,  dz = dy act'(z);  dbeta = sum dz,  dgamma = sum dz h  (over n and the rows);
//              dx = rstd (gamma dz - mean_g(gamma dz) - h mean_g(gamma dz h))
//
// Both are bound by HBM: a forward pass moves x in and y out, a backward pass x and dy in and dx out, plus one re-read for the
// statistics.  Any C / G (a 16-byte vector of a row may span several groups: sums are kept per channel and folded into groups
// at the end), any image / row strides, fp32 / bf16 / fp16.
//
// Three launches per direction; the first and the last have one grid (a chunk of rows x a slab of channels per workgroup, so the last
// finds its chunk where the first left it: in the L2 of its XCD or in the memory-side cache):
//   1. partial sums of the chunk.  Forward: (mean, M2) per group -- a lane accumulates x - p and (x - p)^2 against its OWN first
//      sample p of the channel (with n <= 64 samples per lane sum (x-p)^2 <= (n + 1) M2, so a lane loses at most n ulp whatever the
//      mean / spread ratio or outliers are) and lanes / channels / chunks combine by the parallel-variance formula.  A sum at the magnitude of
//      n mean is rounded by ulps of the mean, which 1 / sqrt(eps) shows where a group is constant: the mean is that sum / n, and then the
//      mean of the deviations from it (a constant group comes out exactly beta).
//      Backward: sum dz and sum dz h per channel, and their gamma-weighted sums per group.
//   2. a wave per (image, group) folds the chunks' partials (4 .. 5 us; every workgroup of 3 folding for itself took longer: a few KB of
//      dependent loads at the head of each of ~1000 workgroups).
//   3. the chunk once more: y, or dx.  In backward its first workgroups reduce dgamma / dbeta over images and chunks.
// A few groups of an image whose rows fit a workgroup's registers need ONE launch and one read (gna_fit_kernel below).
// Nothing is accumulated with atomics: results do not depend on the order of workgroups.
//
// Measured: 8 x 19200 x 256 fp16 + GELU forward 63 us, 53 with x still in the cache (1 19.6, 2 4.6, 3 32.3: 4.9 TB/s in 3; the mean's correction costs
// 1.7 in 1); the same in fp32, forward and backward, 251 us (32.7 + 4.8 + 54.4, 70.0 + 4.9 + 78.7: 5.8 and 6.0 TB/s in 3, what the cache kept
// included); 16 x 4800 x 256 bf16 + SiLU 22 us forward in one launch (3.6 TB/s: one workgroup of 1024 a CU, the load, the sums and the store one
// after the other; 0.8 of it the correction).
#include "common.cuh"

#include <type_traits>

namespace poet {

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

constexpr int NT = 256;

struct GnaP {
    const void* x; int64_t xn, xr;          // image / row strides in elements; channels are contiguous
    const void* dy; int64_t dn, dr;
    void* y; int64_t yn, yr;                // forward: y; backward: dx
    const float* gamma;
    const float* beta;
    float* stats;                           // (N, G, 2) mean, rstd: written by forward, read by backward
    float2* part;                           // (N, G, T * P) partials of a group
    float2* folded;                         // (N, G): forward (mean, rstd) -- the stats when asked for --, backward the two means over the group
    float2* cpart;                          // (N, T, C) backward: (sum dz, sum dz h) per channel
    float* dgamma;
    float* dbeta;
    int N, HW, C, G, cpg;
    int T, R;                               // row chunks of R rows
    int nslab, gps, P, cpp;                 // slabs of gps whole groups (P == 1), or a group in P pieces of cpp channels
    int tail;                               // backward, second launch: leading workgroups that reduce dgamma / dbeta
    int accumulate, act;
    int reverse;                            // second pass: from the last row to the first
    float eps;
};

template <typename T, int V> __device__ __forceinline__ void ldv(const T* p, float* o) {
    if constexpr (V == 1) o[0] = io<T>::ld(p);
    else vec<T, V>::ld(p, o);
}
template <typename T, int V> __device__ __forceinline__ void stv(T* p, const float* o) {
    if constexpr (V == 1) io<T>::st(p, o[0]);
    else vec<T, V>::st(p, o);
}

// ---- activations (POET_ACT_*) -----------------------------------------------------------------------
enum { A_NONE = 0, A_RELU = 1, A_GELU = 2, A_SILU = 3 };

// Phi(-u) = e q(t), e = exp(-u^2 / 2), t = 1 / (1 + 0.3 u), u >= 0: a degree-8 relative minimax fit (1.5e-7) of
// exp(u^2 / 2) erfc(u / sqrt 2) / 2 -- one exp and one reciprocal serve Phi AND the density of the backward pass, where erff alone
// costs twice as many instructions and these kernels have ~30 per bf16 element before they stop being bound by HBM.
__device__ __forceinline__ float gauss_cdf(float z, float& e) {
    const float u = fabsf(z);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3f, u, 1.f));
    e = __builtin_amdgcn_exp2f(-0.72134752f * u * u);
    float q = 0.0356747722f;
    q = fmaf(q, t, -0.157203075f);
    q = fmaf(q, t, 0.206353494f);
    q = fmaf(q, t, -0.0536836334f);
    q = fmaf(q, t, 0.128561621f);
    q = fmaf(q, t, 0.0999134936f);
    q = fmaf(q, t, 0.120753956f);
    q = fmaf(q, t, 0.119629299f);
    q *= t * e;
    return z < 0.f ? q : 1.f - q;
}
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * z)); }

template <int ACT> __device__ __forceinline__ float act_f(float z) {
    if constexpr (ACT == A_RELU) return z < 0.f ? 0.f : z;               // (a NaN stays one)
    if constexpr (ACT == A_GELU) { float e; return z * gauss_cdf(z, e); }
    if constexpr (ACT == A_SILU) return z * sigmoid(z);
    return z;
}
template <int ACT> __device__ __forceinline__ float act_df(float z, float dy) {       // dy act'(z)
    if constexpr (ACT == A_RELU) return z > 0.f ? dy : 0.f;
    if constexpr (ACT == A_GELU) { float e; const float c = gauss_cdf(z, e); return dy * fmaf(z * 0.39894228f, e, c); }
    if constexpr (ACT == A_SILU) { const float s = sigmoid(z); return dy * (s * fmaf(z, 1.f - s, 1.f)); }
    return dy;
}

// ---- statistics -----------------------------------------------------------------------------------------
__device__ __forceinline__ float not_below_zero(float v) { return v < 0.f ? 0.f : v; }                 // (a NaN stays one)
// Sums of squares beyond fp32 (deviations from 1.8e19 / sqrt(n) on) are infinite, or infinity - infinity: such a group comes out NaN, like one that
// holds an infinity, not finite and wrong.
__device__ __forceinline__ float rstd_of(float var, float eps) { return var < INFINITY ? 1.f / sqrtf(var + eps) : NAN; }

// ---- this workgroup's chunk and slab ------------------------------------------------------------------
struct Blk {
    int n, t, s, row0, row1;          // image, chunk, slab; rows [row0, row1)
    int g0, ng, c0, Cs, cps, piece;   // first group, groups, first channel, channels, channels per group in this slab
    int LPR, RP, r, l;                // lanes per row, rows per pass, this thread's row / lane
    bool active;
};
// Where the first pass read more than the memory-side cache keeps, the second takes the chunks, and their rows, in the opposite order, each on
// the XCD (b % 8) of the first: what was read last is still there (backward, 8 x 19200 x 256 fp32, 315 MB: 171 -> 148 us; below the
// cache's size the way back is 5 % slower)
__device__ __forceinline__ int turned(const GnaP& p, int b, int total) {
    const int q = total >> 3;
    return p.reverse && b < q * 8 ? (q - 1 - (b >> 3)) * 8 + (b & 7) : b;
}
template <int V> __device__ __forceinline__ Blk decode(const GnaP& p, int b) {
    Blk k;
    k.t = b % p.T;
    const int q = b / p.T;
    k.s = q % p.nslab;
    k.n = q / p.nslab;
    k.row0 = k.t * p.R;
    k.row1 = min(p.HW, k.row0 + p.R);
    if (p.P == 1) {
        k.g0 = k.s * p.gps;
        k.ng = min(p.G - k.g0, p.gps);
        k.c0 = k.g0 * p.cpg;
        k.cps = p.cpg;
        k.Cs = k.ng * p.cpg;
        k.piece = 0;
    } else {
        k.g0 = k.s / p.P;
        k.piece = k.s - k.g0 * p.P;
        k.ng = 1;
        k.c0 = k.g0 * p.cpg + k.piece * p.cpp;
        k.cps = k.Cs = min(p.cpp, p.cpg - k.piece * p.cpp);
    }
    k.LPR = k.Cs / V;
    k.RP = NT / k.LPR;
    k.r = threadIdx.x / k.LPR;
    k.l = threadIdx.x - k.r * k.LPR;
    k.active = k.r < k.RP;
    return k;
}

constexpr int ROWS_AHEAD = 2;      // vectors of a thread in flight (4: 84 -> 94 us backward at 8 x 19200 x 256 fp16, GELU; 8: 104)
// this thread's first row in the chunk (the last one of its strides of ROWS_AHEAD RP when reversed), and the stride
__device__ __forceinline__ int first_row(const GnaP& p, const Blk& k, int& step) {
    step = ROWS_AHEAD * k.RP;
    const int n = k.row1 - k.row0 - k.r;
    if (!p.reverse || n <= 0) return k.row0 + k.r;
    const int last = k.row0 + k.r + (n - 1) / step * step;
    step = -step;
    return last;
}

// per-thread, per-channel values -> one sum per channel (chan) -> one per group of the slab (grp).  red: RP x Cs floats.
template <int V> __device__ __forceinline__ void to_channels(const Blk& k, const float* v, float* red, float* chan) {
    __syncthreads();
    if (k.active)
#pragma unroll
        for (int i = 0; i < V; ++i) red[k.r * k.Cs + k.l * V + i] = v[i];
    __syncthreads();
    for (int c = threadIdx.x; c < k.Cs; c += NT) {
        float s = 0.f;
        for (int r = 0; r < k.RP; ++r) s += red[r * k.Cs + c];
        chan[c] = s;
    }
    __syncthreads();
}
__device__ __forceinline__ float team_sum(float v, int team) {             // team: a power of two <= 64 of consecutive lanes
    for (int o = team >> 1; o; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ int team_of(int ng) { return ng <= 4 ? 64 : 8; }
__device__ __forceinline__ void to_groups(const Blk& k, const float* chan, float* grp) {
    const int team = team_of(k.ng), per = NT / team, m = threadIdx.x & (team - 1);
    for (int b = 0; b < k.ng; b += per) {
        const int g = b + threadIdx.x / team;
        float s = 0.f;
        if (g < k.ng)
            for (int c = m; c < k.cps; c += team) s += chan[g * k.cps + c];
        s = team_sum(s, team);
        if (g < k.ng && m == 0) grp[g] = s;
    }
    __syncthreads();
}


// ---- forward, 1: (mean, M2) per group of the chunk ------------------------------------------------------
template <typename TX, int V> __global__ __launch_bounds__(NT) void gna_stats_kernel(const GnaP p) {
    __shared__ float red[NT * V], chan[NT * V], grp[NT * V], grp2[NT * V];
    const Blk k = decode<V>(p, blockIdx.x);
    const TX* x = (const TX*)p.x + k.n * p.xn + k.c0 + k.l * V;
    float pv[V], S[V], Q[V];
#pragma unroll
    for (int i = 0; i < V; ++i) pv[i] = S[i] = Q[i] = 0.f;
    int cnt = 0;
    if (k.active) {
        int row = k.row0 + k.r;
        if (row < k.row1) ldv<TX, V>(x + (int64_t)row * p.xr, pv);
        for (; row < k.row1; row += ROWS_AHEAD * k.RP) {
            float v[ROWS_AHEAD][V];
#pragma unroll
            for (int u = 0; u < ROWS_AHEAD; ++u)
                if (row + u * k.RP < k.row1) ldv<TX, V>(x + (int64_t)(row + u * k.RP) * p.xr, v[u]);
#pragma unroll
            for (int u = 0; u < ROWS_AHEAD; ++u)
                if (row + u * k.RP < k.row1) {
                    ++cnt;
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float d = v[u][i] - pv[i];
                        S[i] += d;
                        Q[i] = fmaf(d, d, Q[i]);
                    }
                }
        }
    }
    const float fc = (float)cnt, rc = cnt ? 1.f / fc : 0.f;
    float w[V], d[V];
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = fmaf(fc, pv[i], S[i]);
    to_channels<V>(k, w, red, chan);
    to_groups(k, chan, grp);
    const float n = (float)(k.row1 - k.row0) * (float)k.cps, inv = 1.f / n;
#pragma unroll
    for (int i = 0; i < V; ++i) {                          // about grp inv, some ulps off the mean
        d[i] = k.active ? pv[i] - grp[(k.l * V + i) / k.cps] * inv : 0.f;
        w[i] = fmaf(fc, d[i], S[i]);
    }
    to_channels<V>(k, w, red, chan);
    to_groups(k, chan, grp2);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        d[i] = fmaf(S[i], rc, d[i]);
        w[i] = fmaf(-S[i] * rc, S[i], Q[i]) + fc * d[i] * d[i];
    }
    to_channels<V>(k, w, red, chan);
    to_groups(k, chan, red);
    for (int g = threadIdx.x; g < k.ng; g += NT) {
        const float c = grp2[g] / n;
        p.part[(((int64_t)k.n * p.G + k.g0 + g) * p.T + k.t) * p.P + k.piece] = make_float2(fmaf(grp[g], inv, c), not_below_zero(fmaf(-grp2[g], c, red[g])));
    }
}

// ---- forward, 2: fold the chunks, normalise, activate ----------------------------------------------------
template <typename TX, typename TY, int V, int ACT>
__device__ __forceinline__ void apply_rows(const GnaP& p, const Blk& k, const float* mean, const float* sc, const float* sh) {
    const TX* x = (const TX*)p.x + k.n * p.xn + k.c0 + k.l * V;
    TY* y = (TY*)p.y + k.n * p.yn + k.c0 + k.l * V;
    int step;
    for (int row = first_row(p, k, step); row < k.row1 && row >= k.row0; row += step) {
        float v[ROWS_AHEAD][V];
#pragma unroll
        for (int u = 0; u < ROWS_AHEAD; ++u)
            if (row + u * k.RP < k.row1) ldv<TX, V>(x + (int64_t)(row + u * k.RP) * p.xr, v[u]);
#pragma unroll
        for (int u = 0; u < ROWS_AHEAD; ++u)
            if (row + u * k.RP < k.row1) {
#pragma unroll
                for (int i = 0; i < V; ++i) v[u][i] = act_f<ACT>(fmaf(v[u][i] - mean[i], sc[i], sh[i]));
                stv<TY, V>(y + (int64_t)(row + u * k.RP) * p.yr, v[u]);
            }
    }
}

// a wave per (image, group): the partials of its chunks -> (mean, rstd), or backward (BWD) the two means of dx's formula
template <bool BWD> __global__ __launch_bounds__(NT) void gna_fold_kernel(const GnaP p) {
    const int64_t ng = (int64_t)blockIdx.x * (NT / 64) + (threadIdx.x >> 6);
    if (ng >= (int64_t)p.N * p.G) return;
    const int lane = threadIdx.x & 63, E = p.T * p.P;
    const float total = (float)p.HW * (float)p.cpg;
    const float2* e = p.part + ng * E;
    if constexpr (BWD) {
        float s1 = 0.f, s2 = 0.f;
#pragma unroll 4
        for (int i = lane; i < E; i += 64) s1 += e[i].x, s2 += e[i].y;
        s1 = team_sum(s1, 64);
        s2 = team_sum(s2, 64);
        if (lane == 0) p.folded[ng] = make_float2(s1 / total, s2 / total);
    } else {
        auto weight = [&](int i) {
            const int t = p.P == 1 ? i : i / p.P, q = i - t * p.P;
            return (float)(min(p.HW, (t + 1) * p.R) - t * p.R) * (float)(p.P == 1 ? p.cpg : min(p.cpp, p.cpg - q * p.cpp));
        };
        const float m0 = e[0].x;
        float s = 0.f;
#pragma unroll 4
        for (int i = lane; i < E; i += 64) s = fmaf(weight(i), e[i].x - m0, s);
        const float mean = m0 + team_sum(s, 64) / total;
        float q = 0.f;
#pragma unroll 4
        for (int i = lane; i < E; i += 64) {
            const float d = e[i].x - mean;
            q += fmaf(weight(i) * d, d, e[i].y);
        }
        q = team_sum(q, 64);
        if (lane == 0) p.folded[ng] = make_float2(mean, rstd_of(q / total, p.eps));
    }
}

template <typename TX, typename TY, int V, int ACT> __global__ __launch_bounds__(NT) void gna_apply_kernel(const GnaP p) {
    const Blk k = decode<V>(p, turned(p, blockIdx.x, gridDim.x));
    if (!k.active) return;
    float mean[V], sc[V], sh[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = k.l * V + i;
        const float2 st = p.folded[(int64_t)k.n * p.G + k.g0 + c / k.cps];
        mean[i] = st.x;
        sc[i] = p.gamma[k.c0 + c] * st.y;
        sh[i] = p.beta[k.c0 + c];
    }
    apply_rows<TX, TY, V, ACT>(p, k, mean, sc, sh);
}

// ---- backward, 1: sum dz and sum dz h per channel, gamma-weighted per group ---------------------------------
struct Chan { float mean, rstd, gamma, beta; };
template <int V> __device__ __forceinline__ void load_chan(const GnaP& p, const Blk& k, Chan* ch) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = k.l * V + i, g = k.g0 + c / k.cps;
        const float2 st = *reinterpret_cast<const float2*>(p.stats + 2 * ((int64_t)k.n * p.G + g));
        ch[i] = {st.x, st.y, p.gamma[k.c0 + c], p.beta[k.c0 + c]};
    }
}

template <typename TX, typename TY, int V, int ACT> __global__ __launch_bounds__(NT) void gna_bwd_stats_kernel(const GnaP p) {
    __shared__ float red[NT * V], chan[NT * V], chan2[NT * V], grp[NT * V], grp2[NT * V];
    const Blk k = decode<V>(p, blockIdx.x);
    float a[V], b[V];
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] = b[i] = 0.f;
    if (k.active) {
        Chan ch[V];
        load_chan<V>(p, k, ch);
        const TX* x = (const TX*)p.x + k.n * p.xn + k.c0 + k.l * V;
        const TY* dy = (const TY*)p.dy + k.n * p.dn + k.c0 + k.l * V;
        for (int row = k.row0 + k.r; row < k.row1; row += ROWS_AHEAD * k.RP) {
            float v[ROWS_AHEAD][V], w[ROWS_AHEAD][V];
#pragma unroll
            for (int u = 0; u < ROWS_AHEAD; ++u)
                if (row + u * k.RP < k.row1) {
                    ldv<TX, V>(x + (int64_t)(row + u * k.RP) * p.xr, v[u]);
                    ldv<TY, V>(dy + (int64_t)(row + u * k.RP) * p.dr, w[u]);
                }
#pragma unroll
            for (int u = 0; u < ROWS_AHEAD; ++u)
                if (row + u * k.RP < k.row1)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float h = (v[u][i] - ch[i].mean) * ch[i].rstd;
                        const float dz = act_df<ACT>(fmaf(h, ch[i].gamma, ch[i].beta), w[u][i]);
                        a[i] += dz;
                        b[i] = fmaf(dz, h, b[i]);
                    }
        }
    }
    to_channels<V>(k, a, red, chan);
    to_channels<V>(k, b, red, chan2);
    float2* cp = p.cpart + ((int64_t)k.n * p.T + k.t) * p.C + k.c0;
    for (int c = threadIdx.x; c < k.Cs; c += NT) {
        const float g = p.gamma[k.c0 + c];
        cp[c] = make_float2(chan[c], chan2[c]);
        chan[c] *= g;
        chan2[c] *= g;
    }
    __syncthreads();
    to_groups(k, chan, grp);
    to_groups(k, chan2, grp2);
    for (int g = threadIdx.x; g < k.ng; g += NT)
        p.part[(((int64_t)k.n * p.G + k.g0 + g) * p.T + k.t) * p.P + k.piece] = make_float2(grp[g], grp2[g]);
}

// ---- backward, 2: dx of the chunk; the first p.tail workgroups reduce dgamma / dbeta of 16 channels each -------
__device__ __forceinline__ void reduce_params(const GnaP& p, int b) {
    __shared__ double ra[16][17], rb[16][17];
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4, cc = b * 16 + c;
    double sa = 0.0, sb = 0.0;
    const int E = p.N * p.T;
    if (cc < p.C) {
#pragma unroll 8
        for (int e = r; e < E; e += 16) {
            const float2 v = p.cpart[(int64_t)e * p.C + cc];
            sa += v.x;
            sb += v.y;
        }
    }
    ra[r][c] = sa;
    rb[r][c] = sb;
    __syncthreads();
    if (r == 0 && cc < p.C) {
        for (int i = 1; i < 16; ++i) sa += ra[i][c], sb += rb[i][c];
        p.dbeta[cc] = (p.accumulate ? p.dbeta[cc] : 0.f) + (float)sa;
        p.dgamma[cc] = (p.accumulate ? p.dgamma[cc] : 0.f) + (float)sb;
    }
}

template <typename TX, typename TY, int V, int ACT> __global__ __launch_bounds__(NT) void gna_bwd_apply_kernel(const GnaP p) {
    if ((int)blockIdx.x < p.tail) return reduce_params(p, blockIdx.x);
    const Blk k = decode<V>(p, turned(p, blockIdx.x - p.tail, gridDim.x - p.tail));
    if (!k.active) return;
    Chan ch[V];
    load_chan<V>(p, k, ch);
    float k2[V], k3[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float2 m = p.folded[(int64_t)k.n * p.G + k.g0 + (k.l * V + i) / k.cps];
        k2[i] = -ch[i].rstd * m.x;
        k3[i] = -ch[i].rstd * m.y;
    }
    const TX* x = (const TX*)p.x + k.n * p.xn + k.c0 + k.l * V;
    const TY* dy = (const TY*)p.dy + k.n * p.dn + k.c0 + k.l * V;
    TX* dx = (TX*)p.y + k.n * p.yn + k.c0 + k.l * V;
    int step;
    for (int row = first_row(p, k, step); row < k.row1 && row >= k.row0; row += step) {
        float v[ROWS_AHEAD][V], w[ROWS_AHEAD][V];
#pragma unroll
        for (int u = 0; u < ROWS_AHEAD; ++u)
            if (row + u * k.RP < k.row1) {
                ldv<TX, V>(x + (int64_t)(row + u * k.RP) * p.xr, v[u]);
                ldv<TY, V>(dy + (int64_t)(row + u * k.RP) * p.dr, w[u]);
            }
#pragma unroll
        for (int u = 0; u < ROWS_AHEAD; ++u)
            if (row + u * k.RP < k.row1) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float h = (v[u][i] - ch[i].mean) * ch[i].rstd;
                    const float dz = act_df<ACT>(fmaf(h, ch[i].gamma, ch[i].beta), w[u][i]);
                    v[u][i] = fmaf(ch[i].gamma * ch[i].rstd, dz, fmaf(k3[i], h, k2[i]));
                }
                stv<TX, V>(dx + (int64_t)(row + u * k.RP) * p.yr, v[u]);
            }
    }
}

// ---- whole images in registers: one launch ------------------------------------------------------------------------------------
// Where the rows of a few groups of an image fit a workgroup's registers (up to 192 KB), x is read once, the statistics are plain two-pass
// sums over registers (the mean corrected by the deviations from it), and a forward pass is ONE launch: what small calls cost is launches, and a level of 4800 rows saves its re-read.  Needs
// whole vectors in a group.  A workgroup takes gpw neighbouring groups: lanes l of a row's LPR = gpw * cpg / V, rows threadIdx / LPR + u RP.
template <typename T, int V> struct Raw {
    u32x4_t w;
    __device__ __forceinline__ void ld(const T* p) { w = *reinterpret_cast<const u32x4_t*>(p); }
    __device__ __forceinline__ void get(float* o) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = __uint_as_float(w[i]);
        } else if constexpr (std::is_same<T, bf16_t>::value) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[2 * i] = __uint_as_float(w[i] << 16), o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[2 * i] = h_lo(w[i]), o[2 * i + 1] = h_hi(w[i]);
        }
    }
};
template <typename T> struct Raw<T, 1> {
    float w;
    __device__ __forceinline__ void ld(const T* p) { w = io<T>::ld(p); }
    __device__ __forceinline__ void get(float* o) const { o[0] = w; }
};
// sums of v over the workgroup's threads that share this thread's group (lanes lg * g .. of every LPR): lg and LPR powers of two up to 64, or
// one group for the whole workgroup.  sh: K BT floats.
template <int BT, int K> __device__ __forceinline__ void group_sums(float (&v)[K], float* sh, int lg, int LPR, bool one, int grp) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1)
        if (one || o < lg || o >= LPR)
#pragma unroll
            for (int q = 0; q < K; ++q) v[q] += __shfl_xor(v[q], o, 64);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    __syncthreads();
    if (one ? lane == 0 : lane < LPR && (lane & (lg - 1)) == 0)
#pragma unroll
        for (int q = 0; q < K; ++q) sh[q * BT + wave * 64 + (one ? 0 : lane / lg)] = v[q];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < K; ++q) {
        v[q] = 0.f;
#pragma unroll
        for (int w = 0; w < BT / 64; ++w) v[q] += sh[q * BT + w * 64 + grp];
    }
}
struct Fit {                            // where this thread works
    int n, g0, c, grp, l, r, LPR, RP, lg;
    bool one, active;
};
template <int BT, int V> __device__ __forceinline__ Fit fit_of(const GnaP& p) {
    Fit f;
    const int b = blockIdx.x, total = gridDim.x, q = total >> 3, rem = total & 7, x = b & 7;
    const int k = x * q + min(x, rem) + (b >> 3);          // neighbouring groups share 128-byte lines: the same XCD, at about the same time
    const int per = p.G / p.gps;
    f.n = k / per;
    f.g0 = (k - f.n * per) * p.gps;
    f.lg = p.cpg / V;
    f.LPR = f.lg * p.gps;
    f.RP = BT / f.LPR;
    f.r = threadIdx.x / f.LPR;
    f.l = threadIdx.x - f.r * f.LPR;
    f.one = p.gps == 1;
    f.grp = f.one ? 0 : f.l / f.lg;
    f.c = f.g0 * p.cpg + f.l * V;
    f.active = f.r < f.RP;
    return f;
}

template <typename TX, int V, int BT, int NR> __global__ __launch_bounds__(BT) void gna_fit_kernel(const GnaP p) {
    __shared__ float sh[2 * BT];
    const Fit f = fit_of<BT, V>(p);
    const TX* x = (const TX*)p.x + f.n * p.xn + f.c;
    Raw<TX, V> raw[NR];
    float s[2] = {0.f, 0.f}, first = 0.f;                  // (sums against the thread's first value)
    const int rows = f.active ? p.HW : 0;
#pragma unroll
    for (int u = 0; u < NR; ++u)
        if (f.r + u * f.RP < rows) raw[u].ld(x + (f.r + u * f.RP) * p.xr);
    int cnt = 0;
#pragma unroll
    for (int u = 0; u < NR; ++u)
        if (f.r + u * f.RP < rows) {
            float v[V];
            raw[u].get(v);
            if (u == 0) first = v[0];
            cnt += V;
#pragma unroll
            for (int i = 0; i < V; ++i) s[0] += v[i] - first;
        }
    const float n = (float)p.HW * (float)p.cpg;
    float about[1] = {fmaf((float)cnt, first, s[0])};
    group_sums<BT>(about, sh, f.lg, f.LPR, f.one, f.grp);
    about[0] /= n;                                         // some ulps off the mean: the deviations from it say how many
    s[0] = 0.f;
#pragma unroll
    for (int u = 0; u < NR; ++u)
        if (f.r + u * f.RP < rows) {
            float v[V];
            raw[u].get(v);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = v[i] - about[0];
                s[0] += d;
                s[1] = fmaf(d, d, s[1]);
            }
        }
    group_sums<BT>(s, sh, f.lg, f.LPR, f.one, f.grp);
    const float c = s[0] / n, mean = about[0] + c, rstd = rstd_of(not_below_zero(fmaf(-s[0], c, s[1])) / n, p.eps);
    if (p.stats && f.r == 0 && f.l % f.lg == 0) *reinterpret_cast<float2*>(p.stats + 2 * ((int64_t)f.n * p.G + f.g0 + f.grp)) = make_float2(mean, rstd);
    if (!f.active) return;
    float sc[V], b[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sc[i] = p.gamma[f.c + i] * rstd, b[i] = p.beta[f.c + i];
    TX* y = (TX*)p.y + f.n * p.yn + f.c;
    auto rest = [&](auto act) {
#pragma unroll
        for (int u = 0; u < NR; ++u)
            if (f.r + u * f.RP < rows) {
                float v[V];
                raw[u].get(v);
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] = act_f<decltype(act)::value>(fmaf(v[i] - mean, sc[i], b[i]));
                stv<TX, V>(y + (f.r + u * f.RP) * p.yr, v);
            }
    };
    if (p.act == A_NONE) rest(std::integral_constant<int, A_NONE>());
    else if (p.act == A_RELU) rest(std::integral_constant<int, A_RELU>());
    else if (p.act == A_GELU) rest(std::integral_constant<int, A_GELU>());
    else rest(std::integral_constant<int, A_SILU>());
}

// backward: x and dy stay in registers; leaves the channel sums of the image in cpart (N, C), or in dgamma / dbeta when N == 1
template <typename TX, int V, int BT, int NR> __global__ __launch_bounds__(BT) void gna_fit_bwd_kernel(const GnaP p) {
    constexpr int W = BT / 64;
    __shared__ float red[BT * V], tot[64 * V][2];
    const Fit f = fit_of<BT, V>(p);
    const TX* x = (const TX*)p.x + f.n * p.xn + f.c;
    const TX* dy = (const TX*)p.dy + f.n * p.dn + f.c;
    Raw<TX, V> raw[NR], rdy[NR];
    const int rows = f.active ? p.HW : 0;
#pragma unroll
    for (int u = 0; u < NR; ++u)
        if (f.r + u * f.RP < rows) {
            raw[u].ld(x + (f.r + u * f.RP) * p.xr);
            rdy[u].ld(dy + (f.r + u * f.RP) * p.dr);
        }
    const float2 st = *reinterpret_cast<const float2*>(p.stats + 2 * ((int64_t)f.n * p.G + f.g0 + f.grp));
    const float mean = st.x, rstd = st.y;
    float ga[V], be[V], a[V], b[V];
#pragma unroll
    for (int i = 0; i < V; ++i) ga[i] = p.gamma[f.c + i], be[i] = p.beta[f.c + i], a[i] = b[i] = 0.f;
    auto sums = [&](auto act) {
#pragma unroll
        for (int u = 0; u < NR; ++u)
            if (f.r + u * f.RP < rows) {
                float v[V], w[V];
                raw[u].get(v);
                rdy[u].get(w);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float h = (v[i] - mean) * rstd, dz = act_df<decltype(act)::value>(fmaf(h, ga[i], be[i]), w[i]);
                    a[i] += dz;
                    b[i] = fmaf(dz, h, b[i]);
                }
            }
    };
    if (p.act == A_NONE) sums(std::integral_constant<int, A_NONE>());
    else if (p.act == A_RELU) sums(std::integral_constant<int, A_RELU>());
    else if (p.act == A_GELU) sums(std::integral_constant<int, A_GELU>());
    else sums(std::integral_constant<int, A_SILU>());
    // rows -> one sum per channel.  LPR a power of two: lanes of one column meet by exchanges; else every thread's own go through LDS
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, Cs = f.LPR * V;
    const bool pow2 = (f.LPR & (f.LPR - 1)) == 0;          // (LPR <= 64)
    if (pow2) {
#pragma unroll
        for (int o = 1; o < 64; o <<= 1)
            if (o >= f.LPR) {
#pragma unroll
                for (int i = 0; i < V; ++i) a[i] += __shfl_xor(a[i], o, 64), b[i] += __shfl_xor(b[i], o, 64);
            }
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const float* v = q ? b : a;
        __syncthreads();
        if (pow2) {
            if (lane < f.LPR)
#pragma unroll
                for (int i = 0; i < V; ++i) red[wave * Cs + lane * V + i] = v[i];
        } else if (f.active) {
#pragma unroll
            for (int i = 0; i < V; ++i) red[threadIdx.x * V + i] = v[i];
        }
        __syncthreads();
        if (pow2) {
            for (int c = threadIdx.x; c < Cs; c += BT) {
                float s = 0.f;
#pragma unroll
                for (int w = 0; w < W; ++w) s += red[w * Cs + c];
                tot[c][q] = s;
            }
        } else {
            for (int c = wave; c < Cs; c += W) {           // a wave per channel
                float s = 0.f;
                for (int r = lane; r < f.RP; r += 64) s += red[r * Cs + c];
                s = team_sum(s, 64);
                if (lane == 0) tot[c][q] = s;
            }
        }
    }
    __syncthreads();
    if (p.dgamma)
        for (int c = threadIdx.x; c < Cs; c += BT) {
            const int cc = f.g0 * p.cpg + c;
            if (p.N == 1) {
                p.dbeta[cc] = (p.accumulate ? p.dbeta[cc] : 0.f) + tot[c][0];
                p.dgamma[cc] = (p.accumulate ? p.dgamma[cc] : 0.f) + tot[c][1];
            } else p.cpart[(int64_t)f.n * p.C + cc] = make_float2(tot[c][0], tot[c][1]);
        }
    if (!p.y || !f.active) return;
    float s1 = 0.f, s2 = 0.f;
    for (int c = f.grp * p.cpg; c < (f.grp + 1) * p.cpg; ++c) {
        const float g = p.gamma[f.g0 * p.cpg + c];
        s1 = fmaf(g, tot[c][0], s1);
        s2 = fmaf(g, tot[c][1], s2);
    }
    const float inv = rstd / ((float)p.HW * (float)p.cpg), k2 = -s1 * inv, k3 = -s2 * inv;
    TX* dx = (TX*)p.y + f.n * p.yn + f.c;
    auto rest = [&](auto act) {
#pragma unroll
        for (int u = 0; u < NR; ++u)
            if (f.r + u * f.RP < rows) {
                float v[V], w[V];
                raw[u].get(v);
                rdy[u].get(w);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float h = (v[i] - mean) * rstd, dz = act_df<decltype(act)::value>(fmaf(h, ga[i], be[i]), w[i]);
                    v[i] = fmaf(ga[i] * rstd, dz, fmaf(k3, h, k2));
                }
                stv<TX, V>(dx + (f.r + u * f.RP) * p.yr, v);
            }
    };
    if (p.act == A_NONE) rest(std::integral_constant<int, A_NONE>());
    else if (p.act == A_RELU) rest(std::integral_constant<int, A_RELU>());
    else if (p.act == A_GELU) rest(std::integral_constant<int, A_GELU>());
    else rest(std::integral_constant<int, A_SILU>());
}
__global__ __launch_bounds__(NT) void gna_params_kernel(const GnaP p) { reduce_params(p, blockIdx.x); }

// ---- host ----------------------------------------------------------------------------------------------
constexpr int FIT_BLOCKS = 256;
constexpr int64_t MAX_THREADS = 1ll << 32;                // of a launch
bool aligned16(const void* p, int64_t a, int64_t b, int esz) { return ((uintptr_t)p % 16) == 0 && (a * esz) % 16 == 0 && (b * esz) % 16 == 0; }
int esize(int dt) { return dt == POET_F32 ? 4 : 2; }

// slabs and chunks for vectors of V elements; false: the channel layout does not split into such vectors
bool plan(GnaP& p, int V) {
    const int maxc = NT * V;
    if (p.C % V) return false;
    int gv = V;                                             // groups per slab: a multiple of gv keeps slab starts on vectors
    while (gv > 1 && (gv / 2 * (int64_t)p.cpg) % V == 0) gv /= 2;
    if ((int64_t)gv * p.cpg <= maxc || p.C <= maxc) {
        p.P = 1;
        p.cpp = p.cpg;
        if (p.C <= maxc) p.gps = p.G;
        else {
            const int most = maxc / p.cpg / gv * gv, n = cdiv(p.G, most);
            p.gps = cdiv(cdiv(p.G, n), gv) * gv;
        }
        p.nslab = cdiv(p.G, p.gps);
    } else {
        if (p.cpg % V) return false;
        p.cpp = cdiv(cdiv(p.cpg, cdiv(p.cpg, maxc)), V) * V;
        p.P = cdiv(p.cpg, p.cpp);
        p.gps = 1;
        p.nslab = p.G * p.P;
    }
    // chunks: ~1024 workgroups (4 per CU), 8 .. 64 rows per lane
    const int cs = p.P == 1 ? p.gps * p.cpg : p.cpp, rp = NT / (cs / V);
    const int64_t want = 1024 / ((int64_t)p.N * p.nslab) + 1;
    int64_t rows = (p.HW + want - 1) / want;
    rows = (rows + rp - 1) / rp * rp;
    if (rows < 8 * rp) rows = 8 * rp;
    if (rows > 64 * rp) rows = 64 * rp;
    p.R = (int)rows;
    p.T = cdiv(p.HW, p.R);
    return true;
}

int64_t ws_need(const GnaP& p, bool bwd) { return 8 * ((int64_t)p.N * p.G * (p.T * p.P + 1) + (bwd ? (int64_t)p.N * p.T * p.C : 0)); }

template <template <typename, typename, int, int> class L, typename TX, typename TY, int V> void by_act(const GnaP& p, int act, hipStream_t s) {
    if (act == A_NONE) L<TX, TY, V, A_NONE>::go(p, s);
    else if (act == A_RELU) L<TX, TY, V, A_RELU>::go(p, s);
    else if (act == A_GELU) L<TX, TY, V, A_GELU>::go(p, s);
    else L<TX, TY, V, A_SILU>::go(p, s);
}
template <template <typename, typename, int, int> class L, typename TX, typename TY> void by_vec(const GnaP& p, int act, bool wide, hipStream_t s) {
    if (wide) by_act<L, TX, TY, 16 / (int)sizeof(TX)>(p, act, s);
    else by_act<L, TX, TY, 1>(p, act, s);
}
// x and y of one type, or one of them fp32
template <template <typename, typename, int, int> class L> bool by_type(const GnaP& p, int xt, int yt, int act, bool wide, hipStream_t s) {
    if (xt == POET_F32 && yt == POET_F32) by_vec<L, float, float>(p, act, wide, s);
    else if (xt == POET_BF16 && yt == POET_BF16) by_vec<L, bf16_t, bf16_t>(p, act, wide, s);
    else if (xt == POET_F16 && yt == POET_F16) by_vec<L, f16_t, f16_t>(p, act, wide, s);
    else if (xt == POET_BF16 && yt == POET_F32) by_vec<L, bf16_t, float>(p, act, wide, s);
    else if (xt == POET_F32 && yt == POET_BF16) by_vec<L, float, bf16_t>(p, act, wide, s);
    else return false;
    return true;
}
int blocks(const GnaP& p) { return p.N * p.nslab * p.T; }
int fold_blocks(const GnaP& p) { return cdiv((int64_t)p.N * p.G, NT / 64); }

template <typename TX, typename TY, int V, int ACT> struct Fwd {
    static void go(const GnaP& p, hipStream_t s) {
        hipLaunchKernelGGL((gna_stats_kernel<TX, V>), dim3(blocks(p)), dim3(NT), 0, s, p);
        hipLaunchKernelGGL((gna_fold_kernel<false>), dim3(fold_blocks(p)), dim3(NT), 0, s, p);
        hipLaunchKernelGGL((gna_apply_kernel<TX, TY, V, ACT>), dim3(blocks(p)), dim3(NT), 0, s, p);
    }
};
template <typename TX, typename TY, int V, int ACT> struct Bwd {
    static void go(const GnaP& p, hipStream_t s) {
        hipLaunchKernelGGL((gna_bwd_stats_kernel<TX, TY, V, ACT>), dim3(blocks(p)), dim3(NT), 0, s, p);
        const int main = p.y ? blocks(p) : 0;
        if (main) hipLaunchKernelGGL((gna_fold_kernel<true>), dim3(fold_blocks(p)), dim3(NT), 0, s, p);
        if (main + p.tail) hipLaunchKernelGGL((gna_bwd_apply_kernel<TX, TY, V, ACT>), dim3(main + p.tail), dim3(NT), 0, s, p);
    }
};

// Whether the rows of some groups of an image fit a workgroup (`most` vectors), and how many groups: enough neighbouring ones for 64-byte pieces
// of a row as long as that leaves two workgroups a CU.  Vectors of V, or single elements for a small image.
bool fit(GnaP& p, int& V, int esz, int most) {
    if (p.cpg % V) V = 1;
    const int lg = p.cpg / V;
    if ((int64_t)p.HW * lg > most || lg > 64) return false;
    if ((int64_t)p.N * p.G >= MAX_THREADS / 1024) return false;
    p.gps = 1;
    p.T = 1;
    if ((lg & (lg - 1)) == 0)
        while (p.G % (2 * p.gps) == 0 && p.gps * lg * V * esz < 64 && 2 * p.gps * lg <= 64 && (int64_t)p.HW * lg * p.gps * 2 <= most &&
               (int64_t)p.N * (p.G / (2 * p.gps)) >= FIT_BLOCKS)
            p.gps *= 2;
    return true;
}
template <typename T, int V, int BT, int NR> void go_fit(const GnaP& p, bool bwd, hipStream_t s) {
    const int blocks = p.N * (p.G / p.gps);
    if (bwd) {
        if constexpr (NR <= 6) hipLaunchKernelGGL((gna_fit_bwd_kernel<T, V, BT, NR>), dim3(blocks), dim3(BT), 0, s, p);
    } else hipLaunchKernelGGL((gna_fit_kernel<T, V, BT, NR>), dim3(blocks), dim3(BT), 0, s, p);
}
template <typename T, int V> void fit_size(const GnaP& p, bool bwd, hipStream_t s) {
    auto holds = [&](int bt, int nr) { return (int64_t)(bt / (p.cpg / V * p.gps)) * nr >= p.HW; };
    if (holds(256, 2)) go_fit<T, V, 256, 2>(p, bwd, s);
    else if (holds(256, 6)) go_fit<T, V, 256, 6>(p, bwd, s);
    else if (holds(1024, 3)) go_fit<T, V, 1024, 3>(p, bwd, s);
    else if (holds(1024, 6)) go_fit<T, V, 1024, 6>(p, bwd, s);
    else go_fit<T, V, 1024, 12>(p, bwd, s);
}
template <typename T> void fit_vec(const GnaP& p, int V, bool bwd, hipStream_t s) {
    if (V == 1) fit_size<T, 1>(p, bwd, s);
    else fit_size<T, 16 / (int)sizeof(T)>(p, bwd, s);
}
bool launch_fit(GnaP& p, int xt, int yt, bool wide_ok, bool bwd, hipStream_t s) {
    if (xt != yt || (xt != POET_F32 && xt != POET_BF16 && xt != POET_F16)) return false;
    GnaP f = p;
    int V = !wide_ok ? 1 : xt == POET_F32 ? 4 : 8;
    // (lanes of a row that do not divide the workgroup leave up to LPR - 1 threads idle: 60 of 64 rows of 3 lanes still hold)
    const int most = bwd ? 6 * 960 : 12 * 960;
    if (!fit(f, V, esize(xt), most)) return false;
    // (16-byte pieces of 128-byte lines, twice: 16 x 4800 x 256 bf16 takes 52 us this way, 45 in chunks)
    if (bwd && f.gps * (f.cpg / V) * V * esize(xt) < 32 && f.HW * (f.cpg / V) > 3 * 960) return false;
    if (xt == POET_F32) fit_vec<float>(f, V, bwd, s);
    else if (xt == POET_BF16) fit_vec<bf16_t>(f, V, bwd, s);
    else fit_vec<f16_t>(f, V, bwd, s);
    if (bwd && p.dgamma && p.N > 1) hipLaunchKernelGGL(gna_params_kernel, dim3(cdiv(p.C, 16)), dim3(NT), 0, s, f);
    return true;
}

// the part of the checks and of the plan that both directions share; returns POET_OK or an error
int setup(GnaP& p, const char* what, int N, int HW, int C, int G, int act, int x_dtype, int y_dtype, bool wide_ok, void* ws, int64_t ws_bytes, bool bwd, bool& wide) {
    POET_CHECK(N > 0 && HW > 0 && C > 0 && G > 0 && C % G == 0, POET_ERR_ARG, "%s: bad dims (N %d, HW %d, C %d, G %d)", what, N, HW, C, G);
    POET_CHECK(act >= A_NONE && act <= A_SILU, POET_ERR_ARG, "%s: unknown activation %d", what, act);
    POET_CHECK(C <= (1 << 20) && HW <= (1 << 30), POET_ERR_UNSUPPORTED, "%s: C > 2^20 or HW > 2^30", what);
    p.N = N; p.HW = HW; p.C = C; p.G = G; p.cpg = C / G;
    wide = wide_ok && plan(p, x_dtype == POET_F32 ? 4 : 8);
    if (!wide) plan(p, 1);
    POET_CHECK((int64_t)N * p.nslab * p.T + cdiv(C, 16) < MAX_THREADS / NT && (int64_t)N * G < MAX_THREADS / 64, POET_ERR_UNSUPPORTED,
               "%s: N %d, HW %d, C %d, G %d would need 2^32 threads", what, N, HW, C, G);
    const int64_t need = ws_need(p, bwd);
    POET_CHECK(ws && ((uintptr_t)ws % 8) == 0 && ws_bytes >= need, POET_ERR_ARG, "%s: workspace of %lld bytes needed (8-byte aligned), %lld given", what,
               (long long)need, (long long)ws_bytes);
    p.reverse = (int64_t)N * HW * C * (esize(x_dtype) + (bwd ? esize(y_dtype) : 0)) > (200ll << 20);
    p.part = (float2*)ws;
    p.folded = p.part + (int64_t)N * G * p.T * p.P;
    p.cpart = p.folded + (int64_t)N * G;
    return POET_OK;
}

}  // namespace

}  // namespace poet

using namespace poet;

extern "C" int64_t poet_groupnorm_act_workspace(int N, int HW, int C, int G) {
    POET_CHECK(N > 0 && HW > 0 && C > 0 && G > 0 && C % G == 0 && C <= (1 << 20) && HW <= (1 << 30), POET_ERR_ARG, "groupnorm_act: bad dims (N %d, HW %d, C %d, G %d)", N, HW, C, G);
    int64_t need = 0;
    for (int V : {1, 4, 8}) {                                // the largest of the layouts the launch may choose
        GnaP p = {};
        p.N = N; p.HW = HW; p.C = C; p.G = G; p.cpg = C / G;
        if (plan(p, V)) need = ws_need(p, true) > need ? ws_need(p, true) : need;
    }
    return need;
}

extern "C" int poet_groupnorm_act_fwd(const void* x, int64_t x_n, int64_t x_r, const float* gamma, const float* beta, void* y, int64_t y_n, int64_t y_r,
                                      float* stats, int N, int HW, int C, int G, float eps, int act, int x_dtype, int y_dtype, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
    POET_CHECK(x && gamma && beta && y, POET_ERR_ARG, "groupnorm_act_fwd: null pointer");
    GnaP p = {};
    bool wide = false;
    const bool wide_ok = aligned16(x, x_n, x_r, esize(x_dtype)) && aligned16(y, y_n, y_r, esize(y_dtype));
    const int rc = setup(p, "groupnorm_act_fwd", N, HW, C, G, act, x_dtype, y_dtype, wide_ok, workspace, workspace_bytes, false, wide);
    if (rc != POET_OK) return rc;
    POET_CHECK(!stats || ((uintptr_t)stats % 8) == 0, POET_ERR_ARG, "groupnorm_act_fwd: stats must be 8-byte aligned");
    p.x = x; p.xn = x_n; p.xr = x_r;
    p.y = y; p.yn = y_n; p.yr = y_r;
    p.gamma = gamma; p.beta = beta; p.stats = stats; p.eps = eps; p.act = act;
    if (launch_fit(p, x_dtype, y_dtype, wide_ok, false, (hipStream_t)stream)) {
        POET_LAUNCH_CHECK();
        return POET_OK;
    }
    if (stats) p.folded = (float2*)stats;
    POET_CHECK(by_type<Fwd>(p, x_dtype, y_dtype, act, wide, (hipStream_t)stream), POET_ERR_UNSUPPORTED, "groupnorm_act_fwd: dtypes %d -> %d", x_dtype, y_dtype);
    POET_LAUNCH_CHECK();
    return POET_OK;
}

extern "C" int poet_groupnorm_act_bwd(const void* dy, int64_t dy_n, int64_t dy_r, const void* x, int64_t x_n, int64_t x_r, const float* stats,
                                      const float* gamma, const float* beta, void* dx, int64_t dx_n, int64_t dx_r, float* dgamma, float* dbeta,
                                      int accumulate, int N, int HW, int C, int G, int act, int x_dtype, int y_dtype, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
    POET_CHECK(dy && x && stats && gamma && beta, POET_ERR_ARG, "groupnorm_act_bwd: null pointer");
    POET_CHECK((dgamma == nullptr) == (dbeta == nullptr) && (dx || dgamma), POET_ERR_ARG, "groupnorm_act_bwd: dgamma and dbeta go together, and something must be asked for");
    POET_CHECK(((uintptr_t)stats % 8) == 0, POET_ERR_ARG, "groupnorm_act_bwd: stats must be 8-byte aligned");
    GnaP p = {};
    bool wide = false;
    const bool wide_ok = aligned16(x, x_n, x_r, esize(x_dtype)) && aligned16(dy, dy_n, dy_r, esize(y_dtype)) && (!dx || aligned16(dx, dx_n, dx_r, esize(x_dtype)));
    const int rc = setup(p, "groupnorm_act_bwd", N, HW, C, G, act, x_dtype, y_dtype, wide_ok, workspace, workspace_bytes, true, wide);
    if (rc != POET_OK) return rc;
    p.x = x; p.xn = x_n; p.xr = x_r;
    p.dy = dy; p.dn = dy_n; p.dr = dy_r;
    p.y = dx; p.yn = dx_n; p.yr = dx_r;
    p.gamma = gamma; p.beta = beta; p.stats = const_cast<float*>(stats);
    p.dgamma = dgamma; p.dbeta = dbeta; p.accumulate = accumulate;
    p.tail = dgamma ? cdiv(C, 16) : 0;
    p.act = act;
    if (launch_fit(p, x_dtype, y_dtype, wide_ok, true, (hipStream_t)stream)) {
        POET_LAUNCH_CHECK();
        return POET_OK;
    }
    POET_CHECK(by_type<Bwd>(p, x_dtype, y_dtype, act, wide, (hipStream_t)stream), POET_ERR_UNSUPPORTED, "groupnorm_act_bwd: dtypes %d, %d", x_dtype, y_dtype);
    POET_LAUNCH_CHECK();
    return POET_OK;
}
