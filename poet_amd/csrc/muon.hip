// Orthogonalised (Muon) updates of weight matrices for gfx950: momentum, Newton-Schulz iteration, weight update.
//
//   u = the update direction (the gradient itself, or Nesterov momentum);  X_0 = u / (|u|_F + eps), turned so that it has d <= n rows;
//   X_{k+1} = q_k X_k,   q_k = a I + b A + c A^2,   A = X_k X_k^T   (steps times; a, b, c may differ from step to step).
//
// Bound: the products.  With A and A^2 symmetric (only tiles on and below the diagonal are computed, then mirrored) a step is
// d^2 n + d^3 + 2 d^2 n multiply-adds x 2 / 2.  What shaped the kernels:
//
//  * PRECISION.  The iteration amplifies small singular values up to 3.4^steps times, roundings with them: one fp16 / bf16 product per
//    step is off by 1e-3 .. 4e-3 of the result's norm (simulated over Gaussian, power-law and rank-deficient spectra), fp32 by 2e-6.
//    So every operand is TWO fp16 numbers, hi = fp16(x 2^s) and lo = fp16(x 2^s - hi), 22 bits together, and a product is three matrix
//    instructions, hi hi + hi lo + lo hi, summed in fp32 (the missing lo lo is 2^-22): the error of an fp32 product (1.8e-6 .. 9e-5 in
//    the same simulation, to within 10 %) at a third of the fp16 rate, five times the rate of the fp32 matrix instructions.  The exponents s
//    come from bounds of the scalar iteration on [0, 1] (host), so that nothing overflows and lo parts stay normal numbers.
//  * Iterating on A alone (d x d, cheaper for n >> d) was rejected: it squares the condition number, 2e-4 off at fp32.
//  * A LIST of matrices of any shapes runs in ONE chain of launches (2 + 3 steps): a device table of records, each workgroup finds
//    its (matrix, tile) by binary search.  A stage's tiles of all matrices overlap; PoET's encoder alone has 30 matrices of which none
//    fills the chip.
//  * No atomics anywhere: results do not depend on workgroup order, nor on the other matrices of the list.
#include "common.cuh"

#include <math.h>

namespace poet {

namespace {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef short v4s_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s_t lds_v4s_t;

constexpr int NT = 256;
constexpr int MAX_STEPS = 16;
constexpr int CHUNK = 24;                  // matrices per launch of the first kernel (records by value)
constexpr int NORM_ELEMS = 4096;           // elements per workgroup of the norm pass (and at most 256 workgroups per matrix)

// One matrix.  Offsets in 16-bit elements from the start of the workspace's plane area; a plane pair is hi followed by lo.
struct Rec {
    const void* g;                         // gradient / input, rows x cols, row stride ldg
    void* o;                               // output (orthogonalize) or parameter (muon)
    float* mom;                            // momentum (muon)
    uint16_t* p16;                         // optional bf16 images of the parameter: hi, and the residual lo
    uint16_t* p16lo;
    const float* lr_scale;                 // optional device word
    int64_t ldg, ldo;
    int64_t x0, x1, am, bm;                // planes: X (two buffers, dp x np), A and q (dp x dp)
    int rows, cols, d, n, dp, np, turned;  // X = u^T when turned (rows > cols)
    int nb, part0;                         // workgroups of the norm pass, first partial sum
    int sym0, upd0, pack0;                 // first tile of the matrix in the symmetric / update / pack grids
    float out_scale;                       // muon: the shape's learning-rate factor
};
struct Recs { Rec r[CHUNK]; };

struct NormP {
    Rec* table;
    double* part;
    int first, count;                      // records of this launch
    int g_dtype, muon, nesterov;
    float mu, omu, gscale, max_norm;       // momentum, 1 - momentum (each rounded once)
    const float* sqnorm;
};
struct StageP {
    const Rec* table;
    const double* part;
    _Float16* planes;
    int count, total;                      // matrices, workgroups
    int g_dtype, o_dtype, muon, nesterov;
    float mu, omu, eps;
    float gscale, max_norm;
    const float* sqnorm;
    float in_scale;                        // 2^-(exponents of the two operands)
    float out_exp;                         // 2^(exponent of the result)
    float a, b, c;                         // q stage; b carries A's exponent
    int flip;                              // which X buffer holds the input
    float lr, wd;
};

template <typename T> __device__ __forceinline__ float ld1(const void* p, int64_t i) { return io<T>::ld((const T*)p + i); }
__device__ __forceinline__ float ld_any(const void* p, int64_t i, int dt) {
    return dt == POET_F32 ? ld1<float>(p, i) : dt == POET_BF16 ? ld1<bf16_t>(p, i) : ld1<f16_t>(p, i);
}
__device__ __forceinline__ void st_any(void* p, int64_t i, float v, int dt) {
    if (dt == POET_F32) io<float>::st((float*)p + i, v);
    else if (dt == POET_BF16) io<bf16_t>::st((bf16_t*)p + i, v);
    else io<f16_t>::st((f16_t*)p + i, v);
}
__device__ __forceinline__ float grad_scale_of(float gscale, const float* sqnorm, float max_norm) {
    if (!sqnorm) return gscale;
    return gscale * fminf(max_norm / (sqrtf(*sqnorm) * gscale + 1e-6f), 1.f);
}

// ---- 1: momentum, partial sums of squares (in 64 bits: neither tiny nor huge gradients lose the norm), the table --------------
__global__ __launch_bounds__(NT) void muon_norm_kernel(const NormP p, const Recs recs) {
    int k = 0, b = blockIdx.x;
    while (b >= recs.r[k].nb) b -= recs.r[k].nb, ++k;
    const Rec& r = recs.r[k];
    if (b == 0) {
        const uint32_t* src = (const uint32_t*)&r;
        uint32_t* dst = (uint32_t*)(p.table + p.first + k);
        for (int i = threadIdx.x; i < (int)(sizeof(Rec) / 4); i += NT) dst[i] = src[i];
    }
    const float gs = grad_scale_of(p.gscale, p.sqnorm, p.max_norm);
    const int64_t E = (int64_t)r.rows * r.cols;
    double s = 0.0;
    for (int64_t i = (int64_t)b * NT + threadIdx.x; i < E; i += (int64_t)r.nb * NT) {
        float v;
        if (p.muon) {
            const float g = ((const float*)r.g)[i] * gs;
            const float m = fmaf(p.mu, r.mom[i], p.omu * g);
            r.mom[i] = m;
            v = p.nesterov ? fmaf(p.mu, m, p.omu * g) : m;
        } else {
            const int64_t row = i / r.cols;
            v = ld_any(r.g, row * r.ldg + (i - row * r.cols), p.g_dtype);
        }
        s += (double)v * (double)v;
    }
    __shared__ double red[NT / 64];
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) p.part[r.part0 + b] = (red[0] + red[1]) + (red[2] + red[3]);
}

// workgroup -> record whose [first tile, next first tile) holds b (FIRST: member of Rec); tiles of one matrix go to one XCD range
template <int Rec::*FIRST> __device__ __forceinline__ int find(const Rec* table, int count, int b) {
    int lo = 0, hi = count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (table[mid].*FIRST <= b) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
__device__ __forceinline__ int xcd_order(int b, int total) {          // workgroup b runs on XCD b % 8: give each a contiguous range of tiles
    const int q = total >> 3, rem = total & 7, x = b & 7;
    return x * q + min(x, rem) + (b >> 3);
}

__device__ __forceinline__ void split16(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

// ---- 2: X_0 as scaled hi / lo planes, zero-padded to whole tiles ------------------------------------------------------------
__global__ __launch_bounds__(NT) void muon_pack_kernel(const StageP p) {
    const int b = blockIdx.x, k = find<&Rec::pack0>(p.table, p.count, b);
    const Rec r = p.table[k];
    __shared__ float tile[64][65];
    __shared__ double s_inv;
    if (threadIdx.x < 64) {
        double s = 0.0;
        for (int i = threadIdx.x; i < r.nb; i += 64) s += p.part[r.part0 + i];
        for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, 64);
        if (threadIdx.x == 0) {
            s_inv = s < INFINITY ? (double)p.out_exp / (sqrt(s) + (double)p.eps) : (double)NAN;      // a NaN or an infinity anywhere: the whole update is NaN
        }
    }
    const float gs = grad_scale_of(p.gscale, p.sqnorm, p.max_norm);
    const int t = b - r.pack0, tn = r.np >> 6, i0 = (t / tn) << 6, j0 = (t % tn) << 6;
    const int sr = r.turned ? j0 : i0, sc = r.turned ? i0 : j0;       // the tile's place in u
    const int c = threadIdx.x & 63;
    for (int q = threadIdx.x >> 6; q < 64; q += 4) {
        const int row = sr + q, col = sc + c;
        float v = 0.f;
        if (row < r.rows && col < r.cols) {
            if (p.muon) {
                const int64_t i = (int64_t)row * r.cols + col;
                const float m = r.mom[i];
                v = p.nesterov ? fmaf(p.mu, m, p.omu * (((const float*)r.g)[i] * gs)) : m;
            } else v = ld_any(r.g, row * r.ldg + col, p.g_dtype);
        }
        tile[q][c] = v;
    }
    __syncthreads();
    const double inv = s_inv;
    _Float16* hi = p.planes + r.x0 + (int64_t)i0 * r.np + j0;
    _Float16* lo = hi + (int64_t)r.dp * r.np;
    for (int q = threadIdx.x >> 6; q < 64; q += 4) {
        const float v = (float)((double)(r.turned ? tile[c][q] : tile[q][c]) * inv);
        const bool in = i0 + q < r.d && j0 + c < r.n;
        _Float16 h, l;
        split16(in ? v : 0.f, h, l);
        hi[(int64_t)q * r.np + c] = h;
        lo[(int64_t)q * r.np + c] = l;
    }
}

// ---- 3: split-operand products ----------------------------------------------------------------------------------------------
// 16-byte chunk swizzles of row-major LDS images (rows of 128 / 64 bytes: the 16 lanes of a ds_read_b128 phase meet all banks once)
template <int ROWB> __device__ __forceinline__ int swz_row(int row) {
    if constexpr (ROWB == 128) {
        const int j = (row >> 1) & 7;
        return j ^ (((j + 2) >> 2) & 1);
    } else {
        const int x = (row >> 2) & 3;
        return x ^ ((x & 1) << 1);
    }
}
// 32-byte pieces of a [k][column] image, for the transposing read (rows of 256 / 128 bytes)
template <int ROWB> __device__ __forceinline__ int swz_col(int krow) {
    if constexpr (ROWB == 256) return (krow & 3) | (((krow >> 3) & 1) << 2);
    else return ((krow >> 1) & 1) | (((krow >> 3) & 1) << 1);
}

// acc[f][s][r] += sum_k first[f 16 + 4 (lane / 16) + r][k] second[s 16 + lane % 16][k] over a T x T tile, 4 waves of T/2 x T/2.
// second: rows of K contiguous elements.  first: the same, or (KM) stored [k][column].  K % BK == 0; every row / column read exists
// (planes are padded to whole tiles).
template <int T, int BK, bool KM> struct Core {
    static constexpr int ROWB = BK * 2, CPR = BK / 8, F = T / 32, PLANE = T * BK * 2, STAGE = 4 * PLANE;
    static constexpr int NL = PLANE / 16 / NT;                                            // 16-byte loads per thread and plane
    static constexpr int COLB = T * 2, CPC = T / 8;
    static __device__ __forceinline__ void run(const _Float16* fh, const _Float16* fl, int64_t ldf, const _Float16* sh, const _Float16* sl, int64_t lds_,
                                               int K, char* smem, f32x4_t (&acc)[F][F]) {
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wf = (wave >> 1) * (T / 2), ws = (wave & 1) * (T / 2);
        const int m16 = lane & 15, kc = lane >> 4;
        int64_t go[NL], so[NL];
        int lo_f[NL], lo_s[NL];
#pragma unroll
        for (int q = 0; q < NL; ++q) {
            const int idx = q * NT + tid, row = idx / CPR, c = idx % CPR;
            so[q] = row * lds_ + c * 8;
            lo_s[q] = row * ROWB + ((c ^ swz_row<ROWB>(row)) & (CPR - 1)) * 16;
            if constexpr (KM) {
                const int kr = idx / CPC, cc = idx % CPC;
                go[q] = kr * ldf + cc * 8;
                lo_f[q] = kr * COLB + (((cc >> 1) ^ swz_col<COLB>(kr)) * 32) + (cc & 1) * 16;
            } else {
                go[q] = row * ldf + c * 8;
                lo_f[q] = lo_s[q];
            }
        }
        u32x4_t rf[2][NL], rs[2][NL];
        auto fetch = [&](int k) {
            const int64_t kf = KM ? (int64_t)k * ldf : k;
#pragma unroll
            for (int q = 0; q < NL; ++q) {
                rf[0][q] = *reinterpret_cast<const u32x4_t*>(fh + go[q] + kf);
                rf[1][q] = *reinterpret_cast<const u32x4_t*>(fl + go[q] + kf);
                rs[0][q] = *reinterpret_cast<const u32x4_t*>(sh + so[q] + k);
                rs[1][q] = *reinterpret_cast<const u32x4_t*>(sl + so[q] + k);
            }
        };
        auto store = [&](char* st) {
#pragma unroll
            for (int q = 0; q < NL; ++q) {
                *reinterpret_cast<u32x4_t*>(st + lo_f[q]) = rf[0][q];
                *reinterpret_cast<u32x4_t*>(st + PLANE + lo_f[q]) = rf[1][q];
                *reinterpret_cast<u32x4_t*>(st + 2 * PLANE + lo_s[q]) = rs[0][q];
                *reinterpret_cast<u32x4_t*>(st + 3 * PLANE + lo_s[q]) = rs[1][q];
            }
        };
        fetch(0);
        store(smem);
        __syncthreads();
        int cur = 0;
        for (int k = 0; k < K; k += BK) {
            const bool more = k + BK < K;
            if (more) fetch(k + BK);
            const char* st = smem + cur * STAGE;
#pragma unroll
            for (int h = 0; h < BK / 32; ++h) {
                f16x8_t fhv[F], flv[F];
#pragma unroll
                for (int f = 0; f < F; ++f) {
                    if constexpr (KM) {
                        const int kr = h * 32 + 8 * kc + (m16 >> 2), piece = (wf >> 4) + f;
                        const int a0 = kr * COLB + ((piece ^ swz_col<COLB>(kr)) * 32) + (m16 & 3) * 8;
                        const int a1 = (kr + 4) * COLB + ((piece ^ swz_col<COLB>(kr + 4)) * 32) + (m16 & 3) * 8;
                        struct { v4s_t lo, hi; } u;
                        u.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t*)(st + a0));
                        u.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t*)(st + a1));
                        fhv[f] = __builtin_bit_cast(f16x8_t, u);
                        u.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t*)(st + PLANE + a0));
                        u.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t*)(st + PLANE + a1));
                        flv[f] = __builtin_bit_cast(f16x8_t, u);
                    } else {
                        const int row = wf + f * 16 + m16, a = row * ROWB + (((h * 4 + kc) ^ swz_row<ROWB>(row)) & (CPR - 1)) * 16;
                        fhv[f] = *reinterpret_cast<const f16x8_t*>(st + a);
                        flv[f] = *reinterpret_cast<const f16x8_t*>(st + PLANE + a);
                    }
                }
#pragma unroll
                for (int s = 0; s < F; ++s) {
                    const int row = ws + s * 16 + m16, a = row * ROWB + (((h * 4 + kc) ^ swz_row<ROWB>(row)) & (CPR - 1)) * 16;
                    const f16x8_t shv = *reinterpret_cast<const f16x8_t*>(st + 2 * PLANE + a), slv = *reinterpret_cast<const f16x8_t*>(st + 3 * PLANE + a);
#pragma unroll
                    for (int f = 0; f < F; ++f) acc[f][s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(flv[f], shv, acc[f][s], 0, 0, 0);
#pragma unroll
                    for (int f = 0; f < F; ++f) acc[f][s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fhv[f], slv, acc[f][s], 0, 0, 0);
#pragma unroll
                    for (int f = 0; f < F; ++f) acc[f][s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fhv[f], shv, acc[f][s], 0, 0, 0);
                }
            }
            if (more) {
                store(smem + (cur ^ 1) * STAGE);       // (the slot's readers passed the barrier that ended the last step)
                __syncthreads();
                cur ^= 1;
            }
        }
    }
};

union H4 { _Float16 h[4]; uint2 u; };

// A = X X^T (Q = 0), or q = a I + b A + c A A (Q = 1): tiles on and below the diagonal, written twice
template <int T, int BK, int Q> __global__ __launch_bounds__(NT, 2) void muon_sym_kernel(const StageP p) {
    __shared__ __attribute__((aligned(16))) char smem[2 * Core<T, BK, false>::STAGE];
    constexpr int F = T / 32;
    const int b = xcd_order(blockIdx.x, p.total), kk = find<&Rec::sym0>(p.table, p.count, b);
    const Rec& r = p.table[kk];
    const int t = b - r.sym0, dp = r.dp;
    int bi = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while ((bi + 1) * (bi + 2) / 2 <= t) ++bi;
    while (bi * (bi + 1) / 2 > t) --bi;
    const int i0 = bi * T, j0 = (t - bi * (bi + 1) / 2) * T;
    const int64_t ld = Q ? dp : r.np, plane = (int64_t)dp * ld;
    const _Float16* in = p.planes + (Q ? r.am : p.flip ? r.x1 : r.x0);
    const int K = Q ? (r.d + BK - 1) / BK * BK : (r.n + BK - 1) / BK * BK;
    f32x4_t acc[F][F];
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
        for (int s = 0; s < F; ++s) acc[f][s] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    Core<T, BK, false>::run(in + j0 * ld, in + plane + j0 * ld, ld, in + i0 * ld, in + plane + i0 * ld, ld, K, smem, acc);

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wf = (wave >> 1) * (T / 2), ws = (wave & 1) * (T / 2), m16 = lane & 15, kc = lane >> 4;
    const int64_t sq = (int64_t)dp * dp;
    const _Float16* am = p.planes + r.am;
    _Float16* out = p.planes + (Q ? r.bm : r.am);
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
        for (int s = 0; s < F; ++s) {
            const int i = i0 + ws + s * 16 + m16, j = j0 + wf + f * 16 + 4 * kc;          // row i, columns j .. j + 3
            H4 h, l;
            if constexpr (Q) {
                H4 ah, al;
                ah.u = *reinterpret_cast<const uint2*>(am + (int64_t)i * dp + j);
                al.u = *reinterpret_cast<const uint2*>(am + sq + (int64_t)i * dp + j);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v = fmaf(p.c * p.in_scale, acc[f][s][e], p.b * ((float)ah.h[e] + (float)al.h[e]));
                    if (i == j + e && i < r.d) v += p.a;
                    split16(v * p.out_exp, h.h[e], l.h[e]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) split16(acc[f][s][e] * (p.in_scale * p.out_exp), h.h[e], l.h[e]);
            }
            if (i >= j + 3) {
                *reinterpret_cast<uint2*>(out + (int64_t)i * dp + j) = h.u;
                *reinterpret_cast<uint2*>(out + sq + (int64_t)i * dp + j) = l.u;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (i < j + 3 && i >= j + e) {
                    out[(int64_t)i * dp + j + e] = h.h[e];
                    out[sq + (int64_t)i * dp + j + e] = l.h[e];
                }
                if (i > j + e) {
                    out[(int64_t)(j + e) * dp + i] = h.h[e];
                    out[sq + (int64_t)(j + e) * dp + i] = l.h[e];
                }
            }
        }
}

// X' = q X; the last step leaves the planes: the output matrix, or the weight update
template <int T, int BK, bool LAST> __global__ __launch_bounds__(NT, 2) void muon_update_kernel(const StageP p) {
    __shared__ __attribute__((aligned(16))) char smem[2 * Core<T, BK, true>::STAGE];
    constexpr int F = T / 32;
    const int b = xcd_order(blockIdx.x, p.total), kk = find<&Rec::upd0>(p.table, p.count, b);
    const Rec& r = p.table[kk];
    const int t = b - r.upd0, tn = r.np / T, i0 = (t / tn) * T, j0 = (t % tn) * T, dp = r.dp;
    const int64_t np = r.np, plane = (int64_t)dp * np, sq = (int64_t)dp * dp;
    const _Float16* x = p.planes + (p.flip ? r.x1 : r.x0);
    const _Float16* qm = p.planes + r.bm;
    f32x4_t acc[F][F];
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
        for (int s = 0; s < F; ++s) acc[f][s] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    Core<T, BK, true>::run(x + j0, x + plane + j0, np, qm + (int64_t)i0 * dp, qm + sq + (int64_t)i0 * dp, dp, (r.d + BK - 1) / BK * BK, smem, acc);

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wf = (wave >> 1) * (T / 2), ws = (wave & 1) * (T / 2), m16 = lane & 15, kc = lane >> 4;
    const float lr = p.lr * (r.lr_scale ? fabsf(*r.lr_scale) : 1.f);
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
        for (int s = 0; s < F; ++s) {
            const int i = i0 + ws + s * 16 + m16, j = j0 + wf + f * 16 + 4 * kc;
            if constexpr (!LAST) {
                _Float16* out = p.planes + (p.flip ? r.x0 : r.x1) + (int64_t)i * np + j;
                H4 h, l;
#pragma unroll
                for (int e = 0; e < 4; ++e) split16(acc[f][s][e] * (p.in_scale * p.out_exp), h.h[e], l.h[e]);
                *reinterpret_cast<uint2*>(out) = h.u;
                *reinterpret_cast<uint2*>(out + plane) = l.u;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (i >= r.d || j + e >= r.n) continue;
                    const float v = acc[f][s][e] * p.in_scale;
                    const int64_t row = r.turned ? j + e : i, col = r.turned ? i : j + e, at = row * r.ldo + col;
                    if (p.muon) {
                        float* w = (float*)r.o;
                        const float nw = fmaf(-lr * r.out_scale, v, w[at] - lr * p.wd * w[at]);
                        w[at] = nw;
                        if (r.p16) {
                            const bf16_t hi = f2bf(nw);
                            r.p16[at] = hi;
                            if (r.p16lo) r.p16lo[at] = f2bf(nw - bf2f(hi));
                        }
                    } else st_any(r.o, at, v, p.o_dtype);
                }
            }
        }
}

// ---- host -----------------------------------------------------------------------------------------------------------------
struct Layout {
    int64_t table, part, planes, total;      // byte offsets
    int parts, sym, upd, pack;
};
int up(int v, int m) { return (v + m - 1) / m * m; }

int tile_of(const int* rows, const int* cols, int n) {
    // 128 x 128 tiles halve the operand traffic per product, 64 x 64 tiles make four times as many workgroups: the large tiles once they
    // fill half the chip in the update products
    int64_t tiles = 0;
    for (int i = 0; i < n; ++i) tiles += (int64_t)cdiv(rows[i], 128) * cdiv(cols[i], 128);
    return tiles >= 128 ? 128 : 64;
}

// fills the shape-dependent members of rec (when given) and the layout; false: too large
bool layout(const int* rows, const int* cols, int n, int T, Layout& L, Rec* rec) {
    int64_t planes = 0, sym = 0, upd = 0, pack = 0, parts = 0;
    for (int i = 0; i < n; ++i) {
        Rec r = {};
        r.rows = rows[i];
        r.cols = cols[i];
        r.turned = rows[i] > cols[i];
        r.d = r.turned ? cols[i] : rows[i];
        r.n = r.turned ? rows[i] : cols[i];
        r.dp = up(r.d, T);
        r.np = up(r.n, T);
        r.x0 = planes;
        r.x1 = r.x0 + 2 * (int64_t)r.dp * r.np;
        r.am = r.x1 + 2 * (int64_t)r.dp * r.np;
        r.bm = r.am + 2 * (int64_t)r.dp * r.dp;
        planes = r.bm + 2 * (int64_t)r.dp * r.dp;
        const int64_t e = (int64_t)r.rows * r.cols;
        r.nb = (int)(e > 256ll * NORM_ELEMS ? 256 : cdiv(e, NORM_ELEMS));
        const int64_t td = r.dp / T, tn = r.np / T;
        if (sym + td * (td + 1) / 2 > (1 << 29) || upd + td * tn > (1 << 29) || pack + (int64_t)(r.dp / 64) * (r.np / 64) > (1 << 29)) return false;
        r.part0 = (int)parts;
        r.sym0 = (int)sym;
        r.upd0 = (int)upd;
        r.pack0 = (int)pack;
        parts += r.nb;
        sym += td * (td + 1) / 2;
        upd += td * tn;
        pack += (int64_t)(r.dp / 64) * (r.np / 64);
        if (rec) rec[i] = r;
    }
    L.parts = (int)parts;
    L.sym = (int)sym;
    L.upd = (int)upd;
    L.pack = (int)pack;
    L.table = 0;
    L.part = ((int64_t)n * sizeof(Rec) + 15) / 16 * 16;
    L.planes = (L.part + parts * 8 + 255) / 256 * 256;
    L.total = L.planes + planes * 2;
    return true;
}

// exponents that keep X_k, A and q of every step within a quarter of fp16's range; false: the iteration leaves any useful range
struct Steps { int ex[MAX_STEPS + 1], ea[MAX_STEPS], eq[MAX_STEPS]; };
bool ranges(const double* coeffs, int steps, Steps& S) {
    auto exponent = [](double bound) { return 13 - (int)ceil(log2(bound > 1e-6 ? bound : 1e-6)); };
    double xb = 1.0001;
    for (int k = 0; k < steps; ++k) {
        const double a = coeffs[3 * k], b = coeffs[3 * k + 1], c = coeffs[3 * k + 2];
        double qb = fabs(a), nx = 0.0;                       // (the padding and A = 0 count: q(0) = a)
        for (int i = 0; i <= 2000; ++i) {
            const double x = xb * i / 2000.0, q = a + b * x * x + c * x * x * x * x;
            if (fabs(q) > qb) qb = fabs(q);
            if (fabs(x * q) > nx) nx = fabs(x * q);
        }
        if (!(qb < 1e4) || !(nx * 1.01 < 1e3)) return false;
        S.ex[k] = exponent(xb);
        S.ea[k] = exponent(xb * xb);
        S.eq[k] = exponent(qb);
        xb = nx * 1.01 + 1e-4;
    }
    S.ex[steps] = 0;
    return true;
}
float pow2(int e) { return ldexpf(1.f, e); }

struct Job {
    const void* const* g;
    const int64_t* ldg;
    void* const* o;
    const int64_t* ldo;
    float* const* mom;
    uint16_t* const* p16;
    uint16_t* const* p16lo;
    const float* const* lr_scale;
    const float* out_scale;
    const int* rows;
    const int* cols;
    int n, g_dtype, o_dtype, muon, nesterov, steps;
    const double* coeffs;
    double mu;
    float eps, lr, wd, gscale, max_norm;
    const float* sqnorm;
};

template <int T, int BK> void chain(const Layout& L, const Job& j, const Steps& S, char* ws, hipStream_t st) {
    StageP p = {};
    p.table = (const Rec*)(ws + L.table);
    p.part = (const double*)(ws + L.part);
    p.planes = (_Float16*)(ws + L.planes);
    p.count = j.n;
    p.g_dtype = j.g_dtype; p.o_dtype = j.o_dtype; p.muon = j.muon; p.nesterov = j.nesterov;
    p.mu = (float)j.mu; p.omu = (float)(1.0 - j.mu); p.eps = j.eps; p.gscale = j.gscale; p.max_norm = j.max_norm; p.sqnorm = j.sqnorm;
    p.lr = j.lr; p.wd = j.wd;
    p.out_exp = pow2(S.ex[0]);
    hipLaunchKernelGGL(muon_pack_kernel, dim3(L.pack), dim3(NT), 0, st, p);
    for (int k = 0; k < j.steps; ++k) {
        p.flip = k & 1;
        p.total = L.sym;
        p.in_scale = pow2(-2 * S.ex[k]);
        p.out_exp = pow2(S.ea[k]);
        hipLaunchKernelGGL((muon_sym_kernel<T, BK, 0>), dim3(L.sym), dim3(NT), 0, st, p);
        p.a = (float)j.coeffs[3 * k];
        p.b = (float)(j.coeffs[3 * k + 1] * pow2(-S.ea[k]));
        p.c = (float)j.coeffs[3 * k + 2];
        p.in_scale = pow2(-2 * S.ea[k]);
        p.out_exp = pow2(S.eq[k]);
        hipLaunchKernelGGL((muon_sym_kernel<T, BK, 1>), dim3(L.sym), dim3(NT), 0, st, p);
        p.total = L.upd;
        p.in_scale = pow2(-S.eq[k] - S.ex[k]);
        p.out_exp = pow2(S.ex[k + 1]);
        if (k + 1 < j.steps) hipLaunchKernelGGL((muon_update_kernel<T, BK, false>), dim3(L.upd), dim3(NT), 0, st, p);
        else hipLaunchKernelGGL((muon_update_kernel<T, BK, true>), dim3(L.upd), dim3(NT), 0, st, p);
    }
}

int run_job(const char* what, const Job& j, void* ws, int64_t ws_bytes, void* stream) {
    POET_CHECK(j.n > 0 && j.g && j.o && j.rows && j.cols && j.coeffs, POET_ERR_ARG, "%s: null list or no matrices", what);
    POET_CHECK(j.steps >= 1 && j.steps <= MAX_STEPS, POET_ERR_ARG, "%s: 1 .. %d steps, got %d", what, MAX_STEPS, j.steps);
    POET_CHECK(j.eps >= 0.f, POET_ERR_ARG, "%s: eps must not be negative", what);
    for (int i = 0; i < j.n; ++i) {
        POET_CHECK(j.g[i] && j.o[i] && (!j.muon || j.mom[i]), POET_ERR_ARG, "%s: null matrix %d", what, i);
        POET_CHECK(j.rows[i] > 0 && j.cols[i] > 0 && j.rows[i] <= (1 << 20) && j.cols[i] <= (1 << 20), POET_ERR_ARG, "%s: matrix %d is %d x %d", what, i, j.rows[i], j.cols[i]);
        POET_CHECK((!j.ldg || j.ldg[i] >= j.cols[i]) && (!j.ldo || j.ldo[i] >= j.cols[i]), POET_ERR_ARG, "%s: rows of matrix %d overlap", what, i);
    }
    Steps S;
    POET_CHECK(ranges(j.coeffs, j.steps, S), POET_ERR_ARG, "%s: these coefficients leave the range the iteration can hold", what);
    const int T = tile_of(j.rows, j.cols, j.n);
    Layout L;
    POET_CHECK(layout(j.rows, j.cols, j.n, T, L, nullptr), POET_ERR_UNSUPPORTED, "%s: too many tiles", what);
    POET_CHECK(ws && ((uintptr_t)ws % 256) == 0 && ws_bytes >= L.total, POET_ERR_ARG, "%s: workspace of %lld bytes needed (256-byte aligned), %lld given", what,
               (long long)L.total, (long long)ws_bytes);
    hipStream_t st = (hipStream_t)stream;
    NormP np = {};
    np.table = (Rec*)((char*)ws + L.table);
    np.part = (double*)((char*)ws + L.part);
    np.g_dtype = j.g_dtype; np.muon = j.muon; np.nesterov = j.nesterov;
    np.mu = (float)j.mu; np.omu = (float)(1.0 - j.mu); np.gscale = j.gscale; np.max_norm = j.max_norm; np.sqnorm = j.sqnorm;
    int64_t base[4] = {0, 0, 0, 0};                       // planes, partials | tiles before this chunk
    int sym = 0, upd = 0, pack = 0;
    for (int f = 0; f < j.n; f += CHUNK) {
        Recs recs = {};
        const int c = j.n - f < CHUNK ? j.n - f : CHUNK;
        Layout C;
        layout(j.rows + f, j.cols + f, c, T, C, recs.r);
        int blocks = 0;
        for (int i = 0; i < c; ++i) {
            Rec& r = recs.r[i];
            r.x0 += base[0]; r.x1 += base[0]; r.am += base[0]; r.bm += base[0];
            r.part0 += (int)base[1];
            r.sym0 += sym; r.upd0 += upd; r.pack0 += pack;
            r.g = j.g[f + i];
            r.o = j.o[f + i];
            r.mom = j.muon ? j.mom[f + i] : nullptr;
            r.p16 = j.p16 ? j.p16[f + i] : nullptr;
            r.p16lo = j.p16lo ? j.p16lo[f + i] : nullptr;
            r.lr_scale = j.lr_scale ? j.lr_scale[f + i] : nullptr;
            r.ldg = j.ldg ? j.ldg[f + i] : r.cols;
            r.ldo = j.ldo ? j.ldo[f + i] : r.cols;
            r.out_scale = j.out_scale ? j.out_scale[f + i] : 1.f;
            blocks += r.nb;
        }
        np.first = f;
        np.count = c;
        hipLaunchKernelGGL(muon_norm_kernel, dim3(blocks), dim3(NT), 0, st, np, recs);
        base[0] += (C.total - C.planes) / 2;
        base[1] += C.parts;
        sym += C.sym; upd += C.upd; pack += C.pack;
    }
    if (T == 128) chain<128, 32>(L, j, S, (char*)ws, st);
    else chain<64, 64>(L, j, S, (char*)ws, st);
    POET_LAUNCH_CHECK();
    return POET_OK;
}

}  // namespace

}  // namespace poet

using namespace poet;

extern "C" int64_t poet_muon_workspace(const int* rows_host, const int* cols_host, int n) {
    POET_CHECK(rows_host && cols_host && n > 0, POET_ERR_ARG, "muon_workspace: null list or no matrices");
    for (int i = 0; i < n; ++i)
        POET_CHECK(rows_host[i] > 0 && cols_host[i] > 0 && rows_host[i] <= (1 << 20) && cols_host[i] <= (1 << 20), POET_ERR_ARG, "muon_workspace: matrix %d is %d x %d", i, rows_host[i], cols_host[i]);
    Layout L;
    POET_CHECK(layout(rows_host, cols_host, n, tile_of(rows_host, cols_host, n), L, nullptr), POET_ERR_UNSUPPORTED, "muon_workspace: too many tiles");
    return L.total;
}

extern "C" int poet_orthogonalize(const void* const* g_host, const int64_t* ldg_host, void* const* o_host, const int64_t* ldo_host, const int* rows_host,
                                  const int* cols_host, int n, int g_dtype, int o_dtype, int steps, const double* coeffs_host, float eps, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
    POET_CHECK(g_dtype >= POET_F32 && g_dtype <= POET_F16 && o_dtype >= POET_F32 && o_dtype <= POET_F16, POET_ERR_UNSUPPORTED, "orthogonalize: dtypes %d -> %d", g_dtype, o_dtype);
    POET_CHECK(ldg_host && ldo_host, POET_ERR_ARG, "orthogonalize: null strides");
    Job j = {};
    j.g = g_host; j.ldg = ldg_host; j.o = o_host; j.ldo = ldo_host;
    j.rows = rows_host; j.cols = cols_host; j.n = n;
    j.g_dtype = g_dtype; j.o_dtype = o_dtype; j.steps = steps; j.coeffs = coeffs_host; j.eps = eps; j.gscale = 1.f;
    return run_job("orthogonalize", j, workspace, workspace_bytes, stream);
}

extern "C" int poet_muon_step(float* const* p_host, const float* const* g_host, float* const* m_host, uint16_t* const* p_bf16_host,
                              uint16_t* const* p_bf16_lo_host, const float* const* lr_scale_host, const float* shape_scale_host, const int* rows_host,
                              const int* cols_host, int n, float lr, double momentum, int nesterov, float weight_decay, int steps,
                              const double* coeffs_host, float eps, const float* sqnorm, float max_norm, float grad_scale, void* workspace,
                              int64_t workspace_bytes, void* stream) {
    POET_CHECK(m_host, POET_ERR_ARG, "muon_step: null list of momenta");
    POET_CHECK(!p_bf16_lo_host || p_bf16_host, POET_ERR_ARG, "muon_step: the lo image needs the hi image");
    POET_CHECK(momentum >= 0.0 && momentum < 1.0, POET_ERR_ARG, "muon_step: momentum must be in [0, 1)");
    Job j = {};
    j.g = (const void* const*)g_host; j.o = (void* const*)p_host; j.mom = m_host;
    j.p16 = p_bf16_host; j.p16lo = p_bf16_lo_host; j.lr_scale = lr_scale_host; j.out_scale = shape_scale_host;
    j.rows = rows_host; j.cols = cols_host; j.n = n;
    j.g_dtype = POET_F32; j.o_dtype = POET_F32; j.muon = 1; j.nesterov = nesterov; j.steps = steps; j.coeffs = coeffs_host; j.eps = eps;
    j.mu = momentum; j.lr = lr; j.wd = weight_decay; j.gscale = grad_scale; j.max_norm = max_norm; j.sqnorm = sqnorm;
    return run_job("muon_step", j, workspace, workspace_bytes, stream);
}
