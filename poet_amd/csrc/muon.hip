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
//  * A LIST of matrices of any shapes is worked on together: its matrices fall into groups by their own shape (group_of below), and the matrices
//    of a group share launches -- one for the narrowest, 2 + steps for narrow ones in slabs, a chain of 2 + 3 steps for the rest: a device table
//    of records, each workgroup finds its (matrix, tile) from the first tiles.  PoET's encoder alone has 30 matrices of which none fills the chip.
//  * No atomics anywhere: results do not depend on workgroup order, nor on the other matrices of the list.
#include "common.cuh"

#include <math.h>

#include <algorithm>
#include <new>

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
enum { SYM = 0, UPD = 1, PACK = 2, GRIDS = 3 };      // (narrow matrices: SYM = slabs)

// One matrix.  Offsets in 16-bit elements from the start of the workspace's plane area; a plane pair is hi followed by lo.
struct Rec {
    const void* g;                         // gradient / input, rows x cols, row stride ldg
    void* o;                               // output (orthogonalize) or parameter (muon)
    float* mom;                            // momentum (muon)
    uint16_t* p16;                         // optional bf16 images of the parameter: hi, and the residual lo
    uint16_t* p16lo;
    const float* lr_scale;                 // optional device word
    int64_t ldg, ldo;
    int64_t x0, x1, am, bm;                // planes: X (two buffers, dp x np), A and q (dp x dp).  Narrow matrices in slabs: X, and two buffers
                                           // of fp32 partial Gram matrices in am, bm
    int rows, cols, d, n, dp, np, turned;  // X = u^T when turned (rows > cols)
    int nb, part0;                         // workgroups of the norm pass, first partial sum
    int first[GRIDS];                      // first tile of the matrix in each grid
    int W;                                 // narrow matrices: columns of a slab
    int gvec, rows_vec, ovec;              // vectors of g and the moment as one flat range / of 4 columns of their rows / of the output rows
    float out_scale;                       // muon: the shape's learning-rate factor
};
struct Recs { Rec r[CHUNK]; };

struct NormP {
    Rec* table;
    int* firsts;                           // [GRIDS][n]: the records' first tiles
    double* part;
    int first, count, n;                   // records of this launch, of the list
    int g_dtype, muon, nesterov;
    float mu, omu, gscale, max_norm;       // momentum, 1 - momentum (each rounded once)
    const float* sqnorm;
};
// what a product needs of a record
struct Shape {
    int64_t x0, x1, am, bm;
    int d, n, dp, np;
};
struct StageP {                            // (what every launch of a chain reads first lies in its first 128 bytes: two lines of the scalar cache)
    _Float16* planes;
    int64_t stride;                        // > 0: all matrices are of the shape `uniform` (the first one's), matrix k's planes lie k * stride further
    Shape uniform;
    int per[2];                            // ... and has this many tiles (SYM, UPD)
    int total;                             // workgroups
    int flip;                              // which X buffer holds the input
    float in_scale;                        // 2^-(exponents of the two operands)
    float out_exp;                         // 2^(exponent of the result)
    float a, b, c;                         // q stage; b carries A's exponent
    int count;                             // matrices
    const Rec* table;
    const int* firsts;
    const double* part;
    const float* sqnorm;
    int g_dtype, o_dtype, muon, nesterov;
    float mu, omu, eps, gscale, max_norm, lr, wd;
};

// a / b for 0 <= a < 2^30, 0 < b, and the remainder (the compiler's exact division costs a launch of these sizes several hundred cycles)
__device__ __forceinline__ int divide(int a, int b, int& rem) {
    int q = (int)((float)a * __builtin_amdgcn_rcpf((float)b));
    rem = a - q * b;
    while (rem < 0) --q, rem += b;
    while (rem >= b) ++q, rem -= b;
    return q;
}

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
__device__ __forceinline__ float direction(float g, float& m, float mu, float omu, int nesterov) {
    m = fmaf(mu, m, omu * g);
    return nesterov ? fmaf(mu, m, omu * g) : m;
}
__global__ __launch_bounds__(NT) void muon_norm_kernel(const NormP p, const Recs recs) {
    int k = 0, b = blockIdx.x;
    while (b >= recs.r[k].nb) b -= recs.r[k].nb, ++k;
    const Rec& r = recs.r[k];
    if (b == 0) {
        const uint32_t* src = (const uint32_t*)&r;
        uint32_t* dst = (uint32_t*)(p.table + p.first + k);
        for (int i = threadIdx.x; i < (int)(sizeof(Rec) / 4); i += NT) dst[i] = src[i];
        if (threadIdx.x < GRIDS) p.firsts[threadIdx.x * p.n + p.first + k] = r.first[threadIdx.x];
    }
    const float gs = grad_scale_of(p.gscale, p.sqnorm, p.max_norm);
    const int64_t E = (int64_t)r.rows * r.cols, step = (int64_t)r.nb * NT;
    double s = 0.0;
    if (p.muon && r.gvec) {
        for (int64_t i = (int64_t)b * NT + threadIdx.x; i < E / 4; i += step) {
            const f32x4_t g = ((const f32x4_t*)r.g)[i];
            f32x4_t m = ((f32x4_t*)r.mom)[i];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float me = m[e];
                const double v = (double)direction(g[e] * gs, me, p.mu, p.omu, p.nesterov);
                m[e] = me;
                s = fma(v, v, s);
            }
            ((f32x4_t*)r.mom)[i] = m;
        }
    } else if (p.muon) {
        for (int64_t i = (int64_t)b * NT + threadIdx.x; i < E; i += step) {
            float m = r.mom[i];
            const double v = (double)direction(((const float*)r.g)[i] * gs, m, p.mu, p.omu, p.nesterov);
            r.mom[i] = m;
            s = fma(v, v, s);
        }
    } else if (r.gvec && p.g_dtype == POET_F32) {
        for (int64_t i = (int64_t)b * NT + threadIdx.x; i < E / 4; i += step) {
            const f32x4_t g = ((const f32x4_t*)r.g)[i];
#pragma unroll
            for (int e = 0; e < 4; ++e) s = fma((double)g[e], (double)g[e], s);
        }
    } else if (r.gvec) {
        for (int64_t i = (int64_t)b * NT + threadIdx.x; i < E / 8; i += step) {
            float g[8];
            if (p.g_dtype == POET_BF16) vec<bf16_t, 8>::ld((const bf16_t*)r.g + i * 8, g);
            else vec<f16_t, 8>::ld((const f16_t*)r.g + i * 8, g);
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fma((double)g[e], (double)g[e], s);
        }
    } else {
        int row = (b * NT + (int)threadIdx.x) / r.cols, col = (b * NT + (int)threadIdx.x) % r.cols;
        const int drow = (int)(step / r.cols), dcol = (int)(step % r.cols);
        while (row < r.rows) {
            const double v = (double)ld_any(r.g, row * r.ldg + col, p.g_dtype);
            s = fma(v, v, s);
            row += drow;
            col += dcol;
            if (col >= r.cols) col -= r.cols, ++row;
        }
    }
    __shared__ double red[NT / 64];
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) p.part[r.part0 + b] = (red[0] + red[1]) + (red[2] + red[3]);
}

// workgroup -> the record whose [first tile, next first tile) holds b: the wave compares 64 first tiles at once (one load's latency, where
// a binary search pays one per halving)
__device__ __forceinline__ const Rec& find(const Rec* table, const int* firsts, int count, int b) {
    int k = -1;
    for (int c = 0; c < count; c += 64) {
        const int i = c + (threadIdx.x & 63);
        k += __popcll(__ballot(i < count && firsts[min(i, count - 1)] <= b));
    }
    return table[__builtin_amdgcn_readfirstlane(k)];
}
// the shape behind workgroup b of grid G, and its tile; with one shape for all, two dependent loads less at the head of every launch
template <int G> __device__ __forceinline__ Shape locate(const StageP& p, int b, int& tile) {
    if (p.stride) {
        const int k = __builtin_amdgcn_readfirstlane(divide(b, p.per[G], tile));
        tile = __builtin_amdgcn_readfirstlane(tile);
        Shape s = p.uniform;
        const int64_t o = k * p.stride;
        s.x0 += o; s.x1 += o; s.am += o; s.bm += o;
        return s;
    }
    const Rec& r = find(p.table, p.firsts + G * p.count, p.count, b);
    tile = b - r.first[G];
    return {r.x0, r.x1, r.am, r.bm, r.d, r.n, r.dp, r.np};
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
    const int b = blockIdx.x;
    const Rec r = find(p.table, p.firsts + PACK * p.count, p.count, b);
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
    const int t = b - r.first[PACK], tn = r.np >> 6, i0 = (t / tn) << 6, j0 = (t % tn) << 6;
    const int sr = r.turned ? j0 : i0, sc = r.turned ? i0 : j0;       // the tile's place in u
    const int c4 = (threadIdx.x & 15) * 4, q0 = threadIdx.x >> 4;     // 4 columns of rows q0 + 16 k
    float v[4][4];
    if (r.rows_vec && sr + 64 <= r.rows && sc + 64 <= r.cols) {       // a whole tile of aligned rows: 16-byte (8-byte) loads, all in flight
        if (p.muon) {
            f32x4_t g[4], m[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int64_t i = (int64_t)(sr + q0 + 16 * k) * r.cols + sc + c4;
                g[k] = *reinterpret_cast<const f32x4_t*>((const float*)r.g + i);
                m[k] = *reinterpret_cast<const f32x4_t*>(r.mom + i);                     // (already this step's)
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[k][e] = p.nesterov ? fmaf(p.mu, m[k][e], p.omu * (g[k][e] * gs)) : m[k][e];
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int64_t i = (sr + q0 + 16 * k) * r.ldg + sc + c4;
                if (p.g_dtype == POET_F32) vec<float, 4>::ld((const float*)r.g + i, v[k]);
                else if (p.g_dtype == POET_BF16) vec<bf16_t, 4>::ld((const bf16_t*)r.g + i, v[k]);
                else vec<f16_t, 4>::ld((const f16_t*)r.g + i, v[k]);
            }
        }
    } else {                                                          // (behind an edge: the last element again, so that all loads are in flight)
        auto at = [&](int k, int e) { return min(sr + q0 + 16 * k, r.rows - 1) * r.ldg + min(sc + c4 + e, r.cols - 1); };
        auto all = [&](auto&& fetch) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[k][e] = fetch(at(k, e));
        };
        if (p.muon) {
            float m[4][4];
            all([&](int64_t i) { return ((const float*)r.g)[i]; });
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) m[k][e] = r.mom[at(k, e)];
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[k][e] = p.nesterov ? fmaf(p.mu, m[k][e], p.omu * (v[k][e] * gs)) : m[k][e];
        } else if (p.g_dtype == POET_F32) all([&](int64_t i) { return ld1<float>(r.g, i); });
        else if (p.g_dtype == POET_BF16) all([&](int64_t i) { return ld1<bf16_t>(r.g, i); });
        else all([&](int64_t i) { return ld1<f16_t>(r.g, i); });
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) tile[q0 + 16 * k][c4 + e] = v[k][e];
    __syncthreads();
    int ex = 0;
    const float inv = (float)frexp(s_inv, &ex);                       // (a mantissa and an exponent: the factor alone may leave fp32's range)
    _Float16* hi = p.planes + r.x0 + (int64_t)i0 * r.np + j0;
    _Float16* lo = hi + (int64_t)r.dp * r.np;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int q = q0 + 16 * k;
        _Float16 h[4], l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool in = i0 + q < r.d && j0 + c4 + e < r.n;        // (zeros behind the matrix, also when the factor is not a number)
            split16(in ? ldexpf((r.turned ? tile[c4 + e][q] : tile[q][c4 + e]) * inv, ex) : 0.f, h[e], l[e]);
        }
        *reinterpret_cast<uint2*>(hi + (int64_t)q * r.np + c4) = *reinterpret_cast<const uint2*>(h);
        *reinterpret_cast<uint2*>(lo + (int64_t)q * r.np + c4) = *reinterpret_cast<const uint2*>(l);
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

// Threads of a workgroup with a T x T tile, and its waves' shares of it: 64: 4 waves of 32 x 32; 128: 8 waves of 32 x 64 (first x second), so that
// two waves of a SIMD alternate between LDS reads and matrix instructions (4 waves of 64 x 64 that read their fragments a stage ahead: 858 us at
// 2048 x 2048 where these took 816).  A 2048^3 update takes 56 us (0.92 PFLOP/s of fp16 products, a large library product reaches 1.03); 44 are
// left without its loads, 39 without everything else.  A symmetric 2048 x 2048 x 2048 product, 528 tiles of
// 64 x 64 on 256 CUs, takes 50 us: three tiles after one another on some CUs, and 1 MB of operands through a CU's port per tile.
constexpr int threads_of(int T) { return T == 128 ? 512 : 256; }
// SETS > 1: stage k of BK goes to accumulator set k % SETS, so that the sum has the order of the split kernels below.
// acc[set][f][s][r] += sum_k first[f 16 + 4 (lane / 16) + r][k] second[s 16 + lane % 16][k] over a T x T tile.
// second: rows of K contiguous elements.  first: the same, or (KM) stored [k][column].  K % BK == 0; every row / column read exists
// (planes are padded to whole tiles).
template <int T, int BK, bool KM, int SETS, int SLOTS> struct Core {
    static constexpr int N = threads_of(T), F = 2, S = T / 32, WF = T / 32;                // a wave's 16 x 16 tiles; waves along the first operand
    static constexpr int ROWB = BK * 2, CPR = BK / 8, PLANE = T * BK * 2, STAGE = 4 * PLANE;
    static constexpr int NL = PLANE / 16 / N;                                            // 16-byte loads per thread and plane
    static constexpr int COLB = T * 2, CPC = T / 8;
    static constexpr int LDS = SLOTS * STAGE;
    // Stages reach LDS by DMA, a ring of SLOTS of them: a wave moves NL KB of each of the four planes.  Counted waits and a raw barrier, one a stage:
    // every wave's pieces of stage k have arrived and every wave has read stage k - 1, into whose slot stage k + SLOTS - 1 goes.  Two slots, and two
    // workgroups on a CU; four where no CU gets a second workgroup (1024 x 1024: 234 -> 210 us, ten 1024 x 256: 175 -> 169, 2048 x 2048: 816 -> 780;
    // 4 x 4096 x 1024 with four throughout: 1347 against 1246).  (Inline assembly because the compiler would drain the queue in front of every LDS
    // read.  M0 is written behind its back -- it takes no such clobber -- and nothing else in this file uses it.)
    static __device__ __forceinline__ void dma(uint32_t voff, const void* base, uint32_t lds) {
        asm volatile("s_nop 4\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(base), "s"(lds) : "memory");
    }
    static __device__ __forceinline__ void run(const _Float16* fh, const _Float16* fl, int64_t ldf, const _Float16* sh, const _Float16* sl, int64_t lds_,
                                                int K, char* smem, f32x4_t (&acc)[SETS][F][S]) {
        static_assert(LDS >= T * T * 4, "the tile fits the stages' LDS");
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wf = wave % WF * 32, ws = wave / WF * (T / 2);
        const int m16 = lane & 15, kc = lane >> 4;
        // which pieces of a stage belong at this thread's places of a plane
        uint32_t go[NL], so[NL];
#pragma unroll
        for (int q = 0; q < NL; ++q) {
            const int idx = q * N + tid, row = idx / CPR, c = ((idx % CPR) ^ swz_row<ROWB>(row)) & (CPR - 1);
            so[q] = (uint32_t)(row * lds_ + c * 8) * 2u;
            if constexpr (KM) {
                const int kr = idx / CPC, pc = idx % CPC;
                go[q] = (uint32_t)(kr * ldf + (((((pc >> 1) ^ swz_col<COLB>(kr)) << 1) | (pc & 1)) * 8)) * 2u;
            } else go[q] = (uint32_t)(row * ldf + c * 8) * 2u;
        }
        const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem + wave * 1024;
        auto issue = [&](int k, int slot) {
            const int64_t kf = (KM ? k * ldf : k) * BK, ks = (int64_t)k * BK;
#pragma unroll
            for (int q = 0; q < NL; ++q) {
                const uint32_t to = base + slot * STAGE + q * N * 16;
                dma(go[q], fh + kf, to);
                dma(go[q], fl + kf, to + PLANE);
                dma(so[q], sh + ks, to + 2 * PLANE);
                dma(so[q], sl + ks, to + 3 * PLANE);
            }
        };
        constexpr int UNROLL = SETS > SLOTS ? SETS : SLOTS;
        const int nk = K / BK;
#pragma unroll
        for (int a = 0; a < SLOTS - 1; ++a)
            if (a < nk) issue(a, a);
        for (int k0 = 0; k0 < nk; k0 += UNROLL) {
#pragma unroll
            for (int a = 0; a < UNROLL; ++a) {
                const int k = k0 + a;
                if (k >= nk) break;
                if (nk - 1 - k >= SLOTS - 2) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(4 * NL * (SLOTS - 2)) : "memory");
                else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                if (k + SLOTS - 1 < nk) issue(k + SLOTS - 1, (a + SLOTS - 1) % SLOTS);
                stage(smem + a % SLOTS * STAGE, acc[a % SETS], wf, ws, m16, kc);
            }
        }
    }
    static __device__ __forceinline__ void stage(const char* st, f32x4_t (&acc)[F][S], int wf, int ws, int m16, int kc) {
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
            for (int s = 0; s < S; ++s) {
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
    }
};

union H4 { _Float16 h[4]; uint2 u; };

__device__ __forceinline__ uint2 pack4(const f32x4_t& v, uint2& lo) {          // hi parts; lo: what they leave
    const uint2 hi = make_uint2(pack_h2(v[0], v[1]), pack_h2(v[2], v[3]));
    lo = make_uint2(pack_h2(v[0] - h_lo(hi.x), v[1] - h_hi(hi.x)), pack_h2(v[2] - h_lo(hi.y), v[3] - h_hi(hi.y)));
    return hi;
}
__device__ __forceinline__ void store_some(_Float16* o, _Float16* ol, const uint2& hi, const uint2& lo, int first, int last) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e >= first && e <= last) {
            reinterpret_cast<uint16_t*>(o)[e] = (uint16_t)((e & 2 ? hi.y : hi.x) >> (e & 1) * 16);
            reinterpret_cast<uint16_t*>(ol)[e] = (uint16_t)((e & 2 ? lo.y : lo.x) >> (e & 1) * 16);
        }
}
// A T x T fp32 tile in LDS, 16-byte pieces XORed so that rows and columns of 4 read without conflicts.  A workgroup's N threads hold it as
// pieces: piece u of a thread is row u (N / P) + threadIdx / P, columns 4 (threadIdx % P) .. + 3, P = T / 4.
template <int T> struct Meet {
    static constexpr int N = threads_of(T), P = T / 4, U = T * P / N, F = T / 16;
    static __device__ __forceinline__ int at(int i, int piece) { return i * T + ((piece ^ (i >> 2)) & (P - 1)) * 4; }
    static __device__ __forceinline__ int row(int u) { return u * (N / P) + threadIdx.x / P; }
    static __device__ __forceinline__ int col() { return (threadIdx.x % P) * 4; }
    // the tile in the accumulators of the waves (Core's shares) -> this thread's pieces
    static __device__ __forceinline__ void share(float* part, const f32x4_t (&acc)[2][T / 32], f32x4_t (&v)[U]) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m16 = lane & 15, kc = lane >> 4, wf = wave % (T / 32) * 32, ws = wave / (T / 32) * (T / 2);
        __syncthreads();                                                      // (the last stage's operands have been read)
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int s = 0; s < T / 32; ++s) *reinterpret_cast<f32x4_t*>(part + at(ws + s * 16 + m16, ((wf + f * 16) >> 2) + kc)) = acc[f][s];
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = *reinterpret_cast<const f32x4_t*>(part + at(row(u), col() >> 2));
    }
    // the partial tiles of the four waves -> this thread's pieces of their sum
    static __device__ __forceinline__ void sum(float* part, const f32x4_t (&acc)[F][F], int wave, int m16, int kc, f32x4_t (&v)[U]) {
        float* mine = part + wave * T * T;
#pragma unroll
        for (int q = 0; q < F * F; ++q) *reinterpret_cast<f32x4_t*>(mine + at((q % F) * 16 + m16, (q / F) * 4 + kc)) = acc[q / F][q % F];
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float* t = part + at(row(u), col() >> 2);
            v[u] = (*reinterpret_cast<const f32x4_t*>(t) + *reinterpret_cast<const f32x4_t*>(t + T * T)) +
                   (*reinterpret_cast<const f32x4_t*>(t + 2 * T * T) + *reinterpret_cast<const f32x4_t*>(t + 3 * T * T));
        }
    }
    // ... and turned: afterwards v[u][e] is element (col() + e, row(u)).  (Each thread rewrites the pieces that it alone read there.)
    static __device__ __forceinline__ void turn(float* part, f32x4_t (&v)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) *reinterpret_cast<f32x4_t*>(part + at(row(u), col() >> 2)) = v[u];
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[u][e] = part[at(col() + e, row(u) >> 2) + (row(u) & 3)];
    }
};
// four neighbouring elements of the output matrix, or of the weight update from the old weights o, where these are aligned (ovec)
__device__ __forceinline__ void put4(const Rec& m, const StageP& p, float lr, int64_t at, const f32x4_t& v, f32x4_t o) {
    if (p.muon) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(-lr * m.out_scale, v[e], o[e] - lr * p.wd * o[e]);
        *reinterpret_cast<f32x4_t*>((float*)m.o + at) = o;
        if (m.p16) {
            const uint2 hi = make_uint2(pack_bf2(o[0], o[1]), pack_bf2(o[2], o[3]));
            *reinterpret_cast<uint2*>(m.p16 + at) = hi;
            if (m.p16lo)
                *reinterpret_cast<uint2*>(m.p16lo + at) = make_uint2(pack_bf2(o[0] - __uint_as_float(hi.x << 16), o[1] - __uint_as_float(hi.x & 0xffff0000u)),
                                                                     pack_bf2(o[2] - __uint_as_float(hi.y << 16), o[3] - __uint_as_float(hi.y & 0xffff0000u)));
        }
    } else if (p.o_dtype == POET_F32) *reinterpret_cast<f32x4_t*>((float*)m.o + at) = v;
    else {
        const float w[4] = {v[0], v[1], v[2], v[3]};
        if (p.o_dtype == POET_BF16) vec<bf16_t, 4>::st((bf16_t*)m.o + at, w);
        else vec<f16_t, 4>::st((f16_t*)m.o + at, w);
    }
}
// columns col .. col + 3 of a row of the output matrix, or of the weight update
__device__ __forceinline__ void write4(const Rec& m, const StageP& p, float lr, int row, int col, const f32x4_t& v) {
    if (row >= m.rows || col >= m.cols) return;
    const int64_t at = row * m.ldo + col;
    if (m.ovec) put4(m, p, lr, at, v, p.muon ? *reinterpret_cast<const f32x4_t*>((const float*)m.o + at) : v);       // (cols % 4 == 0)
    else if (p.muon) {
        float* w = (float*)m.o + at;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (col + e >= m.cols) break;
            const float nw = fmaf(-lr * m.out_scale, v[e], w[e] - lr * p.wd * w[e]);
            w[e] = nw;
            if (m.p16) {
                const bf16_t hi = f2bf(nw);
                m.p16[at + e] = hi;
                if (m.p16lo) m.p16lo[at + e] = f2bf(nw - bf2f(hi));
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < m.cols) st_any(m.o, at + e, v[e], p.o_dtype);
    }
}

// A tile of A or of q (from A's pieces ah, al), written twice: as it is, and its mirror image
template <int T, int Q> __device__ __forceinline__ void leave_sym(const StageP& p, const Shape& r, int i0, int j0, float* part, f32x4_t (&v)[Meet<T>::U],
                                                                  const uint2 (&ah)[Meet<T>::U], const uint2 (&al)[Meet<T>::U]) {
    typedef Meet<T> M;
    const int dp = r.dp;
    const int64_t sq = (int64_t)dp * dp;
    const float cs = (Q ? p.c : 1.f) * p.in_scale * p.out_exp, bs = p.b * p.out_exp, as = p.a * p.out_exp;
    const bool diagonal = i0 == j0;
    _Float16* out = p.planes + (Q ? r.bm : r.am) + (int64_t)i0 * dp + j0;
#pragma unroll
    for (int u = 0; u < M::U; ++u) {
        v[u] *= cs;
        if constexpr (Q) {
            const float aa[4] = {h_lo(ah[u].x) + h_lo(al[u].x), h_hi(ah[u].x) + h_hi(al[u].x), h_lo(ah[u].y) + h_lo(al[u].y), h_hi(ah[u].y) + h_hi(al[u].y)};
#pragma unroll
            for (int e = 0; e < 4; ++e) v[u][e] = fmaf(bs, aa[e], v[u][e]);
            if (diagonal) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (M::row(u) == M::col() + e && i0 + M::row(u) < r.d) v[u][e] += as;
            }
        }
        uint2 lo;
        const uint2 hi = pack4(v[u], lo);
        _Float16* o = out + (M::row(u) * dp + M::col());
        if (!diagonal) {
            *reinterpret_cast<uint2*>(o) = hi;
            *reinterpret_cast<uint2*>(o + sq) = lo;
        } else store_some(o, o + sq, hi, lo, 0, M::row(u) - M::col());
    }
    M::turn(part, v);
    out = p.planes + (Q ? r.bm : r.am) + (int64_t)j0 * dp + i0;
#pragma unroll
    for (int u = 0; u < M::U; ++u) {
        uint2 lo;
        const uint2 hi = pack4(v[u], lo);
        _Float16* o = out + (M::row(u) * dp + M::col());
        if (!diagonal) {
            *reinterpret_cast<uint2*>(o) = hi;
            *reinterpret_cast<uint2*>(o + sq) = lo;
        } else store_some(o, o + sq, hi, lo, M::row(u) - M::col() + 1, 3);
    }
}
template <int T> __device__ __forceinline__ void a_pieces(const StageP& p, const Shape& r, int i0, int j0, uint2 (&ah)[Meet<T>::U], uint2 (&al)[Meet<T>::U]) {
    const _Float16* a = p.planes + r.am + (int64_t)i0 * r.dp + j0;
    const int64_t sq = (int64_t)r.dp * r.dp;
#pragma unroll
    for (int u = 0; u < Meet<T>::U; ++u) {
        const _Float16* at = a + (Meet<T>::row(u) * r.dp + Meet<T>::col());
        ah[u] = *reinterpret_cast<const uint2*>(at);
        al[u] = *reinterpret_cast<const uint2*>(at + sq);
    }
}
// A tile of X' into its planes, or of the result (LAST)
template <int T, bool LAST> __device__ __forceinline__ void leave_update(const StageP& p, const Shape& r, int b, int i0, int j0, float* part, f32x4_t (&v)[Meet<T>::U]) {
    typedef Meet<T> M;
    if constexpr (!LAST) {
        const int np = r.np;
        const int64_t plane = (int64_t)r.dp * np;
        _Float16* out = p.planes + (p.flip ? r.x0 : r.x1) + (int64_t)i0 * np + j0;
#pragma unroll
        for (int u = 0; u < M::U; ++u) {
            uint2 lo;
            const uint2 hi = pack4(v[u] * (p.in_scale * p.out_exp), lo);
            _Float16* o = out + (M::row(u) * np + M::col());
            *reinterpret_cast<uint2*>(o) = hi;
            *reinterpret_cast<uint2*>(o + plane) = lo;
        }
    } else {
        const Rec m = find(p.table, p.firsts + UPD * p.count, p.count, b);
        const float lr = p.lr * (m.lr_scale ? fabsf(*m.lr_scale) : 1.f);
        if (m.turned) M::turn(part, v);                                       // output rows are X's columns
#pragma unroll
        for (int u = 0; u < M::U; ++u) write4(m, p, lr, (m.turned ? j0 : i0) + M::row(u), (m.turned ? i0 : j0) + M::col(), v[u] * p.in_scale);
    }
}
__device__ __forceinline__ void triangle(int t, int& bi, int& bj) {           // tile t < 2^29 of the lower triangle
    int i = (int)((__builtin_amdgcn_sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while ((i + 1) * (i + 2) / 2 <= t) ++i;
    while (i * (i + 1) / 2 > t) --i;
    bi = __builtin_amdgcn_readfirstlane(i);
    bj = __builtin_amdgcn_readfirstlane(t - i * (i + 1) / 2);
}
__device__ __forceinline__ void rectangle(int t, int tn, int& bi, int& bj) {  // tile t of rows of tn tiles
    int j;
    bi = __builtin_amdgcn_readfirstlane(divide(t, tn, j));
    bj = __builtin_amdgcn_readfirstlane(j);
}
template <int SETS, int S> __device__ __forceinline__ void zero(f32x4_t (&acc)[SETS][2][S]) {
#pragma unroll
    for (int q = 0; q < SETS * 2 * S; ++q) acc[q / (2 * S)][q / S % 2][q % S] = f32x4_t{0.f, 0.f, 0.f, 0.f};
}
template <int SETS, int S> __device__ __forceinline__ void fold_sets(f32x4_t (&acc)[SETS][2][S]) {
    if constexpr (SETS == 4) {
#pragma unroll
        for (int q = 0; q < 2 * S; ++q) acc[0][q / S][q % S] = (acc[0][q / S][q % S] + acc[1][q / S][q % S]) + (acc[2][q / S][q % S] + acc[3][q / S][q % S]);
    }
}

// A = X X^T (Q = 0), or q = a I + b A + c A A (Q = 1): tiles on and below the diagonal
template <int T, int BK, int SETS, int SLOTS, int Q> __global__ __launch_bounds__(threads_of(T), T == 128 && SLOTS == 2 ? 4 : 2) void muon_sym_kernel(const StageP p) {
    typedef Core<T, BK, false, SETS, SLOTS> C;
    typedef Meet<T> M;
    static_assert(C::LDS >= T * T * 4, "the tile fits the stages' LDS");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    int t, bi, bj;
    const Shape r = locate<SYM>(p, xcd_order(blockIdx.x, p.total), t);
    triangle(t, bi, bj);
    const int i0 = bi * T, j0 = bj * T, dp = r.dp;
    const int64_t ld = Q ? dp : r.np, plane = (int64_t)dp * ld;
    const _Float16* in = p.planes + (Q ? r.am : p.flip ? r.x1 : r.x0);
    const int K = Q ? (r.d + BK - 1) / BK * BK : (r.n + BK - 1) / BK * BK;
    f32x4_t acc[SETS][C::F][C::S];
    zero(acc);
    uint2 ah[M::U], al[M::U];
    if constexpr (Q && T == 64) a_pieces<T>(p, r, i0, j0, ah, al);            // (ahead of the product: 16 registers)
    C::run(in + j0 * ld, in + plane + j0 * ld, ld, in + i0 * ld, in + plane + i0 * ld, ld, K, smem, acc);
    if constexpr (Q && T != 64) a_pieces<T>(p, r, i0, j0, ah, al);
    fold_sets(acc);
    f32x4_t v[M::U];
    M::share(reinterpret_cast<float*>(smem), acc[0], v);
    leave_sym<T, Q>(p, r, i0, j0, reinterpret_cast<float*>(smem), v, ah, al);
}

// X' = q X; the last step leaves the planes: the output matrix, or the weight update
template <int T, int BK, int SETS, int SLOTS, bool LAST> __global__ __launch_bounds__(threads_of(T), T == 128 && SLOTS == 2 ? 4 : 2) void muon_update_kernel(const StageP p) {
    typedef Core<T, BK, true, SETS, SLOTS> C;
    typedef Meet<T> M;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    int t;
    const int b = xcd_order(blockIdx.x, p.total);
    const Shape r = locate<UPD>(p, b, t);
    int bi, bj;
    rectangle(t, r.np / T, bi, bj);
    const int i0 = bi * T, j0 = bj * T, dp = r.dp;
    const int64_t np = r.np, plane = (int64_t)dp * np, sq = (int64_t)dp * dp;
    const _Float16* x = p.planes + (p.flip ? r.x1 : r.x0);
    const _Float16* qm = p.planes + r.bm;
    f32x4_t acc[SETS][C::F][C::S];
    zero(acc);
    const int K = (r.d + BK - 1) / BK * BK;
    C::run(x + j0, x + plane + j0, np, qm + (int64_t)i0 * dp, qm + sq + (int64_t)i0 * dp, dp, K, smem, acc);
    fold_sets(acc);
    f32x4_t v[M::U];
    M::share(reinterpret_cast<float*>(smem), acc[0], v);
    leave_update<T, LAST>(p, r, b, i0, j0, reinterpret_cast<float*>(smem), v);
}

// ---- 3b: the same products for short lists of matrices with d <= 256: 32 x 32 tiles, K split over the waves -------------------------
// With K = d <= 256 a launch is a few microseconds of latency: of the 64 x 64 tiles above, staged through LDS, a K = 256 product is
// four stages in turn with one wave per SIMD, and 128 KB of operands pass one CU's port.  Here the tile is a quarter, so that
// four times as many CUs pull operands, and every wave multiplies the whole tile over its own steps of 32 k, its fragments loaded straight
// into registers (a lane's 16 bytes of a row are the fragment), all in flight at once, no barrier; the partial tiles meet once in LDS.  Four
// 256 x 256 matrices: 110 -> 83 us.  Half as much reuse of every operand byte, and 64-byte pieces of rows instead of 128: ten 1024 x 256
// take 231 us this way against 169 with the staged tiles (and as much as 231 with 64 x 64 tiles that load like these).
struct Frags { f16x8_t h[2], l[2]; };
__device__ __forceinline__ void mfma_tile(f32x4_t (&acc)[2][2], const Frags& f, const Frags& s) {
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[q >> 1][q & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.l[q >> 1], s.h[q & 1], acc[q >> 1][q & 1], 0, 0, 0);
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[q >> 1][q & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.h[q >> 1], s.l[q & 1], acc[q >> 1][q & 1], 0, 0, 0);
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[q >> 1][q & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.h[q >> 1], s.h[q & 1], acc[q >> 1][q & 1], 0, 0, 0);
}
// 32 rows of a plane pair, k .. k + 31 (base: this lane's row and 16-byte piece)
__device__ __forceinline__ void rows_of(Frags& f, const _Float16* base, int ld16, int64_t plane, int k) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        f.h[q] = *reinterpret_cast<const f16x8_t*>(base + (q * ld16 + k));
        f.l[q] = *reinterpret_cast<const f16x8_t*>(base + plane + (q * ld16 + k));
    }
}
// wave w's steps of 32 k: 2 w, 2 w + 1, 2 w + 8, ... (pairs share the 128-byte lines of a row)
__device__ __forceinline__ int step_k(int wave, int u) { return ((u >> 1) * 8 + wave * 2 + (u & 1)) * 32; }

template <int Q> __global__ __launch_bounds__(NT, 2) void muon_sym_split_kernel(const StageP p) {
    constexpr int T = 32;
    typedef Meet<T> M;
    __shared__ __attribute__((aligned(16))) float part[NT / 64 * T * T];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m16 = lane & 15, kc = lane >> 4;
    int t, bi, bj;
    const Shape r = locate<SYM>(p, xcd_order(blockIdx.x, p.total), t);
    triangle(t, bi, bj);
    const int i0 = bi * T, j0 = bj * T, dp = r.dp;
    const int64_t ld = Q ? dp : r.np, plane = (int64_t)dp * ld;
    const _Float16* in = p.planes + (Q ? r.am : p.flip ? r.x1 : r.x0);
    const int K = ((Q ? r.d : r.n) + 31) / 32 * 32, ld16 = (int)ld * 16;
    const _Float16* fb = in + (j0 + m16) * ld + kc * 8;
    const _Float16* sb = in + (i0 + m16) * ld + kc * 8;
    constexpr int AHEAD = Q ? 2 : 4;                                          // (K <= 256: two steps a wave)
    Frags f[AHEAD], s[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
        if (const int k = step_k(wave, u); k < K) rows_of(f[u], fb, ld16, plane, k), rows_of(s[u], sb, ld16, plane, k);
    uint2 ah[M::U], al[M::U];
    if constexpr (Q) a_pieces<T>(p, r, i0, j0, ah, al);
    f32x4_t acc[1][2][2];
    zero(acc);
    for (int u0 = 0; step_k(wave, u0) < K; u0 += AHEAD) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (step_k(wave, u0 + u) >= K) break;
            mfma_tile(acc[0], f[u], s[u]);
            if (const int k = step_k(wave, u0 + u + AHEAD); k < K) rows_of(f[u], fb, ld16, plane, k), rows_of(s[u], sb, ld16, plane, k);
        }
    }
    f32x4_t v[M::U];
    M::sum(part, acc[0], wave, m16, kc, v);
    leave_sym<T, Q>(p, r, i0, j0, part, v, ah, al);
}

// between a wave's LDS stores and its loads of what other lanes stored: these complete in order, so only the compiler has to keep it
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
// X' = q X.  X is stored [k][column]: a wave's steps of 32 rows x 32 columns pass through its quarter of the LDS for the transposing read
// (32-byte pieces of the 64-byte rows XORed with bit 3 of the row: the 8 rows of a read meet all banks once)
template <bool LAST> __global__ __launch_bounds__(NT, 2) void muon_update_split_kernel(const StageP p) {
    constexpr int T = 32, ROWB = T * 2;
    typedef Meet<T> M;
    __shared__ __attribute__((aligned(16))) float part[NT / 64 * T * T];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m16 = lane & 15, kc = lane >> 4;
    const int b = xcd_order(blockIdx.x, p.total);
    int t;
    const Shape r = locate<UPD>(p, b, t);
    int bi, bj;
    rectangle(t, r.np / T, bi, bj);
    const int i0 = bi * T, j0 = bj * T, dp = r.dp, K = (r.d + 31) / 32 * 32;
    const int64_t np = r.np, plane = (int64_t)dp * np;
    const int xrow = lane >> 2, xc = lane & 3;
    const _Float16* x = p.planes + (p.flip ? r.x1 : r.x0) + xrow * np + j0 + xc * 8;
    const _Float16* sb = p.planes + r.bm + (i0 + m16) * dp + kc * 8;
    Frags s[2];
    u32x4_t xr[2][2][2];                                                      // step, plane, rows k + 16 h + lane / 4
#pragma unroll
    for (int u = 0; u < 2; ++u)
        if (const int k = step_k(wave, u); k < K) {                           // (K <= 256: two steps a wave)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                xr[u][0][h] = *reinterpret_cast<const u32x4_t*>(x + (k + h * 16) * np);
                xr[u][1][h] = *reinterpret_cast<const u32x4_t*>(x + plane + (k + h * 16) * np);
            }
            rows_of(s[u], sb, dp * 16, dp * dp, k);
        }
    f32x4_t acc[1][2][2];
    zero(acc);
    static_assert(2 * 32 * ROWB <= T * T * 4, "a step's two planes fit the wave's partial tile");
    char* mine = reinterpret_cast<char*>(part + wave * T * T);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        if (step_k(wave, u) >= K) break;
        wave_sync();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = h * 16 + xrow, at = row * ROWB + ((xc >> 1) ^ ((row >> 3) & 1)) * 32 + (xc & 1) * 16;
            *reinterpret_cast<u32x4_t*>(mine + at) = xr[u][0][h];
            *reinterpret_cast<u32x4_t*>(mine + 32 * ROWB + at) = xr[u][1][h];
        }
        wave_sync();
        Frags f;
#pragma unroll
        for (int q = 0; q < 2; ++q) {                                         // (bit 3 of rows 8 kc .. 8 kc + 7: kc & 1)
            const char* a = mine + (8 * kc + (m16 >> 2)) * ROWB + ((q ^ (kc & 1)) * 32) + (m16 & 3) * 8;
            struct { v4s_t lo, hi; } w;
            w.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t*)(a));
            w.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t*)(a + 4 * ROWB));
            f.h[q] = __builtin_bit_cast(f16x8_t, w);
            w.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t*)(a + 32 * ROWB));
            w.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t*)(a + 36 * ROWB));
            f.l[q] = __builtin_bit_cast(f16x8_t, w);
        }
        mfma_tile(acc[0], f, s[u]);
    }
    wave_sync();
    f32x4_t v[M::U];
    M::sum(part, acc[0], wave, m16, kc, v);
    leave_update<T, LAST>(p, r, b, i0, j0, part, v);
}

// ---- narrow matrices: d <= 96 ------------------------------------------------------------------------------------------------
// The chain above costs 3 dependent launches a step whatever the size, ~6 us each with next to no work in them.  With few rows a
// workgroup can hold everything that the step needs in LDS: q (dp x dp planes) and a SLAB of X's columns.  X' = q X stays inside a slab; only
// A = X X^T couples the slabs, through dp x dp partial sums.
//   * one slab (n <= W_max): ONE launch does momentum, norm, all steps and the update of a matrix per workgroup;
//   * up to 8 slabs: the norm pass, a launch for X_0 and its partial A, then one launch a step, in which every workgroup folds the partial
//     A's of its matrix, forms q for itself (redundant, but dp^3 is small), updates its slab and leaves the partial A of the next step.
// 8 waves.  All of it is bound by LDS bandwidth and latency (one workgroup a CU), so: A and A^2 in 32 x 32 macro tiles on and below the
// diagonal (each fragment read serves two tiles; a diagonal one reads its fragments once), the update in PAIRS of 16-column strips (each
// fragment of q serves both), rewritten in place by the wave that owns them.  Rows of the LDS images are padded by 16 bytes: an odd number
// of 16-byte pieces, so that the 16 rows of a fragment read start in different banks.
constexpr int NW_T = 512, NWAVES = NW_T / 64, MAX_SLABS = 8, MAX_D = 3, MAX_SLAB_D = 2;
template <int D> struct Narrow {
    static constexpr int DP = 32 * D, NM = D * (D + 1) / 2;
    static constexpr int PARTS = D == 1 ? 8 : D == 2 ? 2 : 1;             // few macro tiles: the columns in PARTS ranges, so that all waves have some
    static constexpr int ITEMS = NM * PARTS, ROUNDS = (ITEMS + NWAVES - 1) / NWAVES;
    static constexpr int AROW = DP * 2 + 16, APLANE = DP * AROW;
    static constexpr int SCRATCH = PARTS > 1 ? ITEMS * 4096 : 0;
    static constexpr int REGION = 2 * APLANE > SCRATCH ? 2 * APLANE : SCRATCH;      // A / q planes, or partial tiles
};
constexpr int W_MAX[MAX_D + 1] = {0, 896, 512, 288};       // columns that leave room for REGION in 160 KB
struct NarrowP {
    StageP s;
    int mode, k, steps;                              // N_*; this launch's step
    float a[MAX_STEPS], b[MAX_STEPS], c[MAX_STEPS];  // b carries A's exponent, c the square of it
    float ascale[MAX_STEPS], qscale[MAX_STEPS], xscale[MAX_STEPS];
};
enum { N_INIT, N_STEP, N_LAST };

template <int D> struct Slab {
    typedef Narrow<D> N;
    char* reg;                             // REGION bytes
    char* x;                               // hi plane, then lo plane: DP rows of W columns
    int W, xs, xplane;
    int lane, wave, m16, kc;

    __device__ __forceinline__ Slab(char* smem, int W_) : reg(smem), x(smem + N::REGION), W(W_), xs(W_ * 2 + 16), xplane(N::DP * (W_ * 2 + 16)) {
        lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        m16 = lane & 15;
        kc = lane >> 4;
    }
    static __device__ __forceinline__ void macro(int t, int& bi, int& bj) {
        bi = 0;
        while ((bi + 1) * (bi + 2) / 2 <= t) ++bi;
        bj = t - bi * (bi + 1) / 2;
    }
    // u's columns [j0, j0 + W) of X into the planes as the two halves of their fp32 bits, zero outside the matrix; `at(row, col)` order
    // follows the matrix's rows.  FIRST: the momentum is this step's only afterwards.  Returns this thread's sum of squares.
    template <bool FIRST> __device__ __forceinline__ double load(const Rec& r, const StageP& p, float gs, int j0) const {
        for (int o = threadIdx.x * 16; o < 2 * xplane; o += NW_T * 16) *reinterpret_cast<u32x4_t*>(x + o) = u32x4_t{0, 0, 0, 0};
        __syncthreads();
        const int jn = min(W, r.n - j0), cols = r.turned ? r.d : jn, total = r.d * jn;
        const int row0 = r.turned ? j0 : 0, col0 = r.turned ? 0 : j0;
        int a = threadIdx.x / cols, c = threadIdx.x % cols;
        const int da = NW_T / cols, dc = NW_T % cols;
        double sum = 0.0;
        constexpr int U = 8;                                                  // loads in flight
        if (r.rows_vec) {                                                     // (cols, j0 and the strides are multiples of 4; 32 x 896: 52 -> 40 us with finish())
            const int cols4 = cols / 4, total4 = total / 4, da4 = NW_T / cols4, dc4 = NW_T % cols4;
            int a4 = threadIdx.x / cols4, c4 = threadIdx.x % cols4;
            auto vectors = [&](auto&& fetch, auto&& value) {                  // fetch(u, offset), then value(u, offset) -> four values
                for (int e = threadIdx.x; e < total4; e += U * NW_T) {
                    int64_t at[U];
                    int ra[U], rc[U];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const bool in = e + u * NW_T < total4;                // (behind the end: the first vector again)
                        ra[u] = in ? a4 : 0;
                        rc[u] = in ? c4 * 4 : 0;
                        at[u] = (row0 + ra[u]) * r.ldg + col0 + rc[u];
                        fetch(u, at[u]);
                        a4 += da4;
                        c4 += dc4;
                        if (c4 >= cols4) c4 -= cols4, ++a4;
                    }
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        if (e + u * NW_T >= total4) break;
                        const f32x4_t v = value(u, at[u]);
                        uint32_t b[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            sum = fma((double)v[q], (double)v[q], sum);
                            b[q] = __float_as_uint(v[q]);
                        }
                        if (!r.turned) {
                            char* o = x + ra[u] * xs + rc[u] * 2;
                            *reinterpret_cast<uint2*>(o) = make_uint2((b[0] >> 16) | (b[1] & 0xffff0000u), (b[2] >> 16) | (b[3] & 0xffff0000u));
                            *reinterpret_cast<uint2*>(o + xplane) = make_uint2((b[0] & 0xffffu) | (b[1] << 16), (b[2] & 0xffffu) | (b[3] << 16));
                        } else {
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                char* o = x + (rc[u] + q) * xs + ra[u] * 2;
                                *reinterpret_cast<uint16_t*>(o) = (uint16_t)(b[q] >> 16);
                                *reinterpret_cast<uint16_t*>(o + xplane) = (uint16_t)b[q];
                            }
                        }
                    }
                }
            };
            f32x4_t g4[U], m4[U];
            if (p.muon)
                vectors([&](int u, int64_t at) { g4[u] = *reinterpret_cast<const f32x4_t*>((const float*)r.g + at), m4[u] = *reinterpret_cast<const f32x4_t*>(r.mom + at); },
                        [&](int u, int64_t at) {
                            f32x4_t v;
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                if constexpr (FIRST) {
                                    float m = m4[u][q];
                                    v[q] = direction(g4[u][q] * gs, m, p.mu, p.omu, p.nesterov);
                                    m4[u][q] = m;
                                } else v[q] = p.nesterov ? fmaf(p.mu, m4[u][q], p.omu * (g4[u][q] * gs)) : m4[u][q];
                            }
                            if constexpr (FIRST) *reinterpret_cast<f32x4_t*>(r.mom + at) = m4[u];
                            return v;
                        });
            else if (p.g_dtype == POET_F32)
                vectors([&](int u, int64_t at) { g4[u] = *reinterpret_cast<const f32x4_t*>((const float*)r.g + at); }, [&](int u, int64_t) { return g4[u]; });
            else {
                const bool bf = p.g_dtype == POET_BF16;
                uint2 h4[U];
                vectors([&](int u, int64_t at) { h4[u] = *reinterpret_cast<const uint2*>((const uint16_t*)r.g + at); },
                        [&](int u, int64_t) {
                            const uint2 w = h4[u];
                            return bf ? f32x4_t{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u)}
                                      : f32x4_t{h_lo(w.x), h_hi(w.x), h_lo(w.y), h_hi(w.y)};
                        });
            }
            return sum;
        }
        auto batches = [&](auto&& fetch, auto&& value) {                      // fetch(u, offset of the element), then value(u, offset)
            for (int e = threadIdx.x; e < total; e += U * NW_T) {
                int64_t at[U];
                int o[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const bool in = e + u * NW_T < total;                     // (behind the end: the first element again)
                    const int ra = in ? a : 0, rc = in ? c : 0;
                    at[u] = (row0 + ra) * r.ldg + col0 + rc;
                    o[u] = (r.turned ? rc : ra) * xs + (r.turned ? ra : rc) * 2;
                    fetch(u, at[u]);
                    a += da;
                    c += dc;
                    if (c >= cols) c -= cols, ++a;
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (e + u * NW_T >= total) break;
                    const float v = value(u, at[u]);
                    sum = fma((double)v, (double)v, sum);
                    *reinterpret_cast<uint16_t*>(x + o[u]) = (uint16_t)(__float_as_uint(v) >> 16);
                    *reinterpret_cast<uint16_t*>(x + xplane + o[u]) = (uint16_t)__float_as_uint(v);
                }
            }
        };
        float g[U], m[U];
        uint16_t h[U];
        if (p.muon) {
            batches([&](int u, int64_t at) { g[u] = ((const float*)r.g)[at], m[u] = r.mom[at]; },
                    [&](int u, int64_t at) {
                        if constexpr (!FIRST) return p.nesterov ? fmaf(p.mu, m[u], p.omu * (g[u] * gs)) : m[u];
                        const float v = direction(g[u] * gs, m[u], p.mu, p.omu, p.nesterov);
                        r.mom[at] = m[u];
                        return v;
                    });
        } else if (p.g_dtype == POET_F32)
            batches([&](int u, int64_t at) { g[u] = ((const float*)r.g)[at]; }, [&](int u, int64_t) { return g[u]; });
        else {
            const bool bf = p.g_dtype == POET_BF16;
            batches([&](int u, int64_t at) { h[u] = ((const uint16_t*)r.g)[at]; },
                    [&](int u, int64_t) { return bf ? bf2f(h[u]) : h_lo(h[u]); });
        }
        return sum;
    }
    // the fp32 halves -> normalised, scaled hi / lo planes: times `by` (a mantissa and an exponent: 64-bit arithmetic per element costs
    // several times the pass, and the factor alone may leave fp32's range)
    __device__ __forceinline__ void normalise(double by) const {
        int ex = 0;
        const float inv = (float)frexp(by, &ex);
        __syncthreads();
#pragma unroll 2
        for (int o = threadIdx.x * 16; o < xplane; o += NW_T * 16) {          // (rows are whole 16-byte pieces)
            const u32x4_t h = *reinterpret_cast<const u32x4_t*>(x + o), l = *reinterpret_cast<const u32x4_t*>(x + xplane + o);
            u32x4_t nh, nl;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float v0 = ldexpf(__uint_as_float((h[q] << 16) | (l[q] & 0xffffu)) * inv, ex), v1 = ldexpf(__uint_as_float((h[q] & 0xffff0000u) | (l[q] >> 16)) * inv, ex);
                nh[q] = pack_h2(v0, v1);
                nl[q] = pack_h2(v0 - h_lo(nh[q]), v1 - h_hi(nh[q]));
            }
            *reinterpret_cast<u32x4_t*>(x + o) = nh;
            *reinterpret_cast<u32x4_t*>(x + xplane + o) = nl;
        }
        __syncthreads();
    }
    static __device__ __forceinline__ void product(f32x4_t (&acc)[2][2], const char* fb, const char* sb, int row, int plane, bool diagonal) {
        f16x8_t fh[2], fl[2], sh[2], sl[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            fh[q] = *reinterpret_cast<const f16x8_t*>(fb + q * 16 * row);
            fl[q] = *reinterpret_cast<const f16x8_t*>(fb + q * 16 * row + plane);
        }
        if (diagonal) {
#pragma unroll
            for (int q = 0; q < 2; ++q) sh[q] = fh[q], sl[q] = fl[q];
        } else {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                sh[q] = *reinterpret_cast<const f16x8_t*>(sb + q * 16 * row);
                sl[q] = *reinterpret_cast<const f16x8_t*>(sb + q * 16 * row + plane);
            }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[q >> 1][q & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fl[q >> 1], sh[q & 1], acc[q >> 1][q & 1], 0, 0, 0);
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[q >> 1][q & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh[q >> 1], sl[q & 1], acc[q >> 1][q & 1], 0, 0, 0);
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[q >> 1][q & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh[q >> 1], sh[q & 1], acc[q >> 1][q & 1], 0, 0, 0);
    }
    // tiles of X X^T: acc[round] of item wave + 8 round = part * NM + macro tile
    typedef f32x4_t Tile[2][2];
    __device__ __forceinline__ void gram(Tile (&acc)[N::ROUNDS]) const {
        const int KS = W / 32;
#pragma unroll
        for (int u = 0; u < N::ROUNDS; ++u) {
            const int item = wave + u * NWAVES;
            if (item >= N::ITEMS) break;
            const int mt = item % N::NM, part = item / N::NM;
            int bi, bj;
            macro(mt, bi, bj);
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[u][q >> 1][q & 1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            const char* fb = x + (bj * 32 + m16) * xs + kc * 16;
            const char* sb = x + (bi * 32 + m16) * xs + kc * 16;
            for (int ks = part * KS / N::PARTS; ks < (part + 1) * KS / N::PARTS; ++ks) product(acc[u], fb + ks * 64, sb + ks * 64, xs, xplane, bi == bj);
        }
    }
    // a tile in memory: 32 rows of 8 pieces of 4 columns, XORed with the row (the 16 rows of a store in different banks)
    static __device__ __forceinline__ int tile_at(int i, int piece) { return i * 32 + ((piece ^ (i & 7)) * 4); }
    __device__ __forceinline__ void put_tile(float* out, const Tile& acc) const {
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int q = 0; q < 2; ++q) *reinterpret_cast<f32x4_t*>(out + tile_at(q * 16 + m16, f * 4 + kc)) = acc[f][q];
    }
    __device__ __forceinline__ void put_a(int i, int j, float v) const {
        _Float16 h, l;
        split16(v, h, l);
        *reinterpret_cast<_Float16*>(reg + i * N::AROW + j * 2) = h;
        *reinterpret_cast<_Float16*>(reg + N::APLANE + i * N::AROW + j * 2) = l;
        *reinterpret_cast<_Float16*>(reg + j * N::AROW + i * 2) = h;
        *reinterpret_cast<_Float16*>(reg + N::APLANE + j * N::AROW + i * 2) = l;
    }
    // this thread's 2 NM elements of the macro tiles, summed over the partial tiles at t[(q NM + m) 1024 ...], q < count
    __device__ __forceinline__ void sum_tiles(const float* t, int count, float* v) const {
#pragma unroll
        for (int m = 0; m < 2 * N::NM; ++m) v[m] = 0.f;
#pragma unroll D == 1 ? 4 : 1
        for (int q = 0; q < count; ++q) {                                     // (2 NM loads and more in flight)
            float w[2 * N::NM];
#pragma unroll
            for (int m = 0; m < 2 * N::NM; ++m) w[m] = t[(int64_t)q * N::NM * 1024 + m * 512 + threadIdx.x];
#pragma unroll
            for (int m = 0; m < 2 * N::NM; ++m) v[m] += w[m];
        }
    }
    // A's planes from partial tiles; in_region: these lie where the planes go
    __device__ __forceinline__ void fold(const float* t, int count, float scale, bool in_region) const {
        float v[2 * N::NM];
        sum_tiles(t, count, v);
        if (in_region) __syncthreads();
#pragma unroll
        for (int m = 0; m < 2 * N::NM; ++m) {
            int bi, bj;
            macro(m >> 1, bi, bj);
            const int li = (m & 1) * 16 + (threadIdx.x >> 5), lp = ((threadIdx.x >> 2) & 7) ^ (li & 7);
            const int i = bi * 32 + li, j = bj * 32 + lp * 4 + (threadIdx.x & 3);
            if (i >= j) put_a(i, j, v[m] * scale);
        }
        __syncthreads();
    }
    __device__ __forceinline__ void planes(const Tile& acc, int mt, float scale) const {
        int bi, bj;
        macro(mt, bi, bj);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int i = bi * 32 + (q & 1) * 16 + m16, j = bj * 32 + (q >> 1) * 16 + 4 * kc;
            if (bi == bj && (q & 1) < (q >> 1)) continue;                     // (above the diagonal)
            if (bi == bj && (q & 1) == (q >> 1)) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i >= j + e) put_a(i, j + e, acc[q >> 1][q & 1][e] * scale);
                continue;
            }
            H4 h, l;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                split16(acc[q >> 1][q & 1][e] * scale, h.h[e], l.h[e]);
                *reinterpret_cast<_Float16*>(reg + (j + e) * N::AROW + i * 2) = h.h[e];
                *reinterpret_cast<_Float16*>(reg + N::APLANE + (j + e) * N::AROW + i * 2) = l.h[e];
            }
            *reinterpret_cast<uint2*>(reg + i * N::AROW + j * 2) = h.u;
            *reinterpret_cast<uint2*>(reg + N::APLANE + i * N::AROW + j * 2) = l.u;
        }
    }
    // A of the whole slab, for a matrix of one slab
    __device__ __forceinline__ void gram_planes(float scale) const {
        Tile acc[N::ROUNDS];
        gram(acc);
        if constexpr (N::PARTS > 1) {
#pragma unroll
            for (int u = 0; u < N::ROUNDS; ++u)
                if (wave + u * NWAVES < N::ITEMS) put_tile(reinterpret_cast<float*>(reg) + (wave + u * NWAVES) * 1024, acc[u]);
            __syncthreads();
            fold(reinterpret_cast<const float*>(reg), N::PARTS, scale, true);
        } else {
#pragma unroll
            for (int u = 0; u < N::ROUNDS; ++u)
                if (wave + u * NWAVES < N::ITEMS) planes(acc[u], wave + u * NWAVES, scale);
            __syncthreads();
        }
    }
    // q = a I + b A + c A A in A's place
    __device__ __forceinline__ void square(float a, float b, float c, float scale, int d) const {
        constexpr int R = (N::NM + NWAVES - 1) / NWAVES;
        Tile acc[R];
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const int mt = wave + u * NWAVES;
            if (mt >= N::NM) break;
            int bi, bj;
            macro(mt, bi, bj);
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[u][q >> 1][q & 1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < D; ++ks)
                product(acc[u], reg + (bj * 32 + m16) * N::AROW + ks * 64 + kc * 16, reg + (bi * 32 + m16) * N::AROW + ks * 64 + kc * 16, N::AROW, N::APLANE, bi == bj);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int i = bi * 32 + (q & 1) * 16 + m16, j = bj * 32 + (q >> 1) * 16 + 4 * kc;
                H4 ah, al;
                ah.u = *reinterpret_cast<const uint2*>(reg + i * N::AROW + j * 2);
                al.u = *reinterpret_cast<const uint2*>(reg + N::APLANE + i * N::AROW + j * 2);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v = fmaf(c, acc[u][q >> 1][q & 1][e], b * ((float)ah.h[e] + (float)al.h[e]));
                    if (i == j + e && i < d) v += a;
                    acc[u][q >> 1][q & 1][e] = v;
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < R; ++u)
            if (wave + u * NWAVES < N::NM) planes(acc[u], wave + u * NWAVES, scale);
        __syncthreads();
    }
    // q X of S neighbouring strips from ct on: out(i, j, four columns of row i)
    template <int S, typename F> __device__ __forceinline__ void strip(int ct, F&& out) const {
        f32x4_t acc[S][2 * D];
#pragma unroll
        for (int q = 0; q < S; ++q)
#pragma unroll
            for (int t = 0; t < 2 * D; ++t) acc[q][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < D; ++ks) {
            f16x8_t fh[S], fl[S];
#pragma unroll
            for (int q = 0; q < S; ++q) {
                const char* xa = x + (ks * 32 + 8 * kc + (m16 >> 2)) * xs + (ct + q) * 32 + (m16 & 3) * 8;
                struct { v4s_t lo, hi; } u;
                u.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t*)(xa));
                u.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t*)(xa + 4 * xs));
                fh[q] = __builtin_bit_cast(f16x8_t, u);
                u.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t*)(xa + xplane));
                u.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t*)(xa + xplane + 4 * xs));
                fl[q] = __builtin_bit_cast(f16x8_t, u);
            }
#pragma unroll
            for (int t = 0; t < 2 * D; ++t) {
                const char* qa = reg + (t * 16 + m16) * N::AROW + ks * 64 + kc * 16;
                const f16x8_t sh = *reinterpret_cast<const f16x8_t*>(qa), sl = *reinterpret_cast<const f16x8_t*>(qa + N::APLANE);
#pragma unroll
                for (int q = 0; q < S; ++q) acc[q][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fl[q], sh, acc[q][t], 0, 0, 0);
#pragma unroll
                for (int q = 0; q < S; ++q) acc[q][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh[q], sl, acc[q][t], 0, 0, 0);
#pragma unroll
                for (int q = 0; q < S; ++q) acc[q][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh[q], sh, acc[q][t], 0, 0, 0);
            }
        }
#pragma unroll
        for (int q = 0; q < S; ++q)
#pragma unroll
            for (int t = 0; t < 2 * D; ++t) out(t * 16 + m16, (ct + q) * 16 + 4 * kc, acc[q][t]);
    }
    template <typename F> __device__ __forceinline__ void strips(F&& out) const {
        const int n = W / 16;                                                 // (even)
        if constexpr (W_MAX[D] / 16 >= 2 * NWAVES) {
            if (n >= 2 * NWAVES) {
                for (int ct = 2 * wave; ct < n; ct += 2 * NWAVES) strip<2>(ct, out);
                return;
            }
        }
        for (int ct = wave; ct < n; ct += NWAVES) strip<1>(ct, out);
    }
    __device__ __forceinline__ void update(float scale) const {
        strips([&](int i, int j, const f32x4_t& v) {
            H4 h, l;
#pragma unroll
            for (int e = 0; e < 4; ++e) split16(v[e] * scale, h.h[e], l.h[e]);
            *reinterpret_cast<uint2*>(x + i * xs + j * 2) = h.u;
            *reinterpret_cast<uint2*>(x + xplane + i * xs + j * 2) = l.u;
        });
        __syncthreads();
    }
    // the last step: results go back in place as the two halves of their fp32 bits, then out in whole rows of the matrix
    __device__ __forceinline__ void finish(const Rec& r, const StageP& p, float scale, int j0) const {
        strips([&](int i, int j, const f32x4_t& v) {
            uint32_t u[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) u[e] = __float_as_uint(v[e] * scale);
            *reinterpret_cast<uint2*>(x + i * xs + j * 2) = make_uint2((u[0] >> 16) | (u[1] & 0xffff0000u), (u[2] >> 16) | (u[3] & 0xffff0000u));
            *reinterpret_cast<uint2*>(x + xplane + i * xs + j * 2) = make_uint2((u[0] & 0xffffu) | (u[1] << 16), (u[2] & 0xffffu) | (u[3] << 16));
        });
        __syncthreads();
        const float lr = p.lr * (r.lr_scale ? fabsf(*r.lr_scale) : 1.f);
        const int jn = min(W, r.n - j0), cols = r.turned ? r.d : jn, total = r.d * jn;
        int a = threadIdx.x / cols, c = threadIdx.x % cols;                    // output row (of this slab) and column
        const int da = NW_T / cols, dc = NW_T % cols, row0 = r.turned ? j0 : 0, col0 = r.turned ? 0 : j0;
        if (r.ovec) {
            constexpr int U = 4;
            const int cols4 = cols / 4, total4 = total / 4, da4 = NW_T / cols4, dc4 = NW_T % cols4;
            int a4 = threadIdx.x / cols4, c4 = threadIdx.x % cols4;
            for (int e = threadIdx.x; e < total4; e += U * NW_T) {
                f32x4_t v[U], w[U];
                int64_t at[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const bool in = e + u * NW_T < total4;
                    const int ra = in ? a4 : 0, rc = in ? c4 * 4 : 0;
                    at[u] = (row0 + ra) * r.ldo + col0 + rc;
                    if (p.muon) w[u] = *reinterpret_cast<const f32x4_t*>((const float*)r.o + at[u]);
                    if (!r.turned) {
                        const char* o = x + ra * xs + rc * 2;
                        const uint2 h = *reinterpret_cast<const uint2*>(o), l = *reinterpret_cast<const uint2*>(o + xplane);
                        v[u] = f32x4_t{__uint_as_float((h.x << 16) | (l.x & 0xffffu)), __uint_as_float((h.x & 0xffff0000u) | (l.x >> 16)),
                                       __uint_as_float((h.y << 16) | (l.y & 0xffffu)), __uint_as_float((h.y & 0xffff0000u) | (l.y >> 16))};
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const char* o = x + (rc + q) * xs + ra * 2;
                            v[u][q] = __uint_as_float(((uint32_t)*reinterpret_cast<const uint16_t*>(o) << 16) | *reinterpret_cast<const uint16_t*>(o + xplane));
                        }
                    }
                    a4 += da4;
                    c4 += dc4;
                    if (c4 >= cols4) c4 -= cols4, ++a4;
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (e + u * NW_T < total4) put4(r, p, lr, at[u], v[u], w[u]);
            }
            return;
        }
        constexpr int U = 8;
        for (int e = threadIdx.x; e < total; e += U * NW_T) {
            float v[U], w[U];
            int64_t at[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool in = e + u * NW_T < total;
                const int ra = in ? a : 0, rc = in ? c : 0, o = (r.turned ? rc : ra) * xs + (r.turned ? ra : rc) * 2;
                at[u] = (row0 + ra) * r.ldo + col0 + rc;
                v[u] = __uint_as_float(((uint32_t)*reinterpret_cast<const uint16_t*>(x + o) << 16) | *reinterpret_cast<const uint16_t*>(x + xplane + o));
                if (p.muon) w[u] = ((const float*)r.o)[at[u]];
                a += da;
                c += dc;
                if (c >= cols) c -= cols, ++a;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (e + u * NW_T >= total) break;
                if (!p.muon) st_any(r.o, at[u], v[u], p.o_dtype);
                else {
                    const float nw = fmaf(-lr * r.out_scale, v[u], w[u] - lr * p.wd * w[u]);
                    ((float*)r.o)[at[u]] = nw;
                    if (r.p16) {
                        const bf16_t hi = f2bf(nw);
                        r.p16[at[u]] = hi;
                        if (r.p16lo) r.p16lo[at[u]] = f2bf(nw - bf2f(hi));
                    }
                }
            }
        }
    }
};

// the records of a long list of them
__global__ __launch_bounds__(NT) void muon_table_kernel(Rec* table, int count, const Recs recs) {
    for (int i = threadIdx.x; i < count * (int)(sizeof(Rec) / 4); i += NT) ((uint32_t*)table)[i] = ((const uint32_t*)recs.r)[i];
}
// one matrix per workgroup, start to end
template <int D> __global__ __launch_bounds__(NW_T, 2) void muon_narrow_kernel(const NarrowP p, const Recs recs) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ double red[NWAVES];
    const Rec r = p.s.table ? p.s.table[blockIdx.x] : recs.r[blockIdx.x];
    const StageP& sp = p.s;
    const Slab<D> L(smem, r.W);
    double s = L.template load<true>(r, sp, grad_scale_of(sp.gscale, sp.sqnorm, sp.max_norm), 0);
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.0;
#pragma unroll
    for (int i = 0; i < NWAVES; ++i) s += red[i];
    L.normalise(s < INFINITY ? (double)sp.out_exp / (sqrt(s) + (double)sp.eps) : (double)NAN);
    for (int k = 0; k < p.steps; ++k) {
        L.gram_planes(p.ascale[k]);
        L.square(p.a[k], p.b[k], p.c[k], p.qscale[k], r.d);
        if (k + 1 < p.steps) L.update(p.xscale[k]);
        else L.finish(r, sp, p.xscale[k], 0);
    }
}

// one slab per workgroup, one step per launch
template <int D> __global__ __launch_bounds__(NW_T, 2) void muon_slab_kernel(const NarrowP p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    typedef Narrow<D> N;
    const StageP& sp = p.s;
    const Rec r = find(sp.table, sp.firsts + SYM * sp.count, sp.count, blockIdx.x);
    const int slab = blockIdx.x - r.first[SYM], slabs = (r.n + r.W - 1) / r.W;
    const Slab<D> L(smem, r.W);
    char* xg = reinterpret_cast<char*>(sp.planes + r.x0) + (int64_t)slab * 2 * N::DP * r.W * 2;       // this slab's planes, rows of W columns
    const int cpr = r.W / 8;
    const float* part_in = reinterpret_cast<const float*>(sp.planes + (p.k & 1 ? r.bm : r.am));
    float* part_out = reinterpret_cast<float*>(sp.planes + (p.mode == N_INIT || (p.k & 1) ? r.am : r.bm));
    if (p.mode == N_INIT) {
        __shared__ double s_sum;
        if (threadIdx.x < 64) {
            double s = 0.0;
            for (int i = threadIdx.x; i < r.nb; i += 64) s += sp.part[r.part0 + i];
            for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, 64);
            if (threadIdx.x == 0) s_sum = s;
        }
        L.template load<false>(r, sp, grad_scale_of(sp.gscale, sp.sqnorm, sp.max_norm), slab * r.W);
        const double s = s_sum;                                               // (load has a barrier)
        L.normalise(s < INFINITY ? (double)sp.out_exp / (sqrt(s) + (double)sp.eps) : (double)NAN);
    } else {
        for (int c = threadIdx.x; c < 2 * N::DP * cpr; c += NW_T) {
            const int row = c / cpr, q = c - row * cpr;
            *reinterpret_cast<u32x4_t*>(L.x + row * L.xs + q * 16) = *reinterpret_cast<const u32x4_t*>(xg + (int64_t)c * 16);
        }
        L.fold(part_in, slabs, p.ascale[p.k], false);
        L.square(p.a[p.k], p.b[p.k], p.c[p.k], p.qscale[p.k], r.d);
        if (p.mode == N_LAST) return L.finish(r, sp, p.xscale[p.k], slab * r.W);
        L.update(p.xscale[p.k]);
    }
    typename Slab<D>::Tile acc[N::ROUNDS];
    L.gram(acc);
    part_out += (int64_t)slab * N::NM * 1024;
    float* to = N::PARTS > 1 ? reinterpret_cast<float*>(L.reg) : part_out;
#pragma unroll
    for (int u = 0; u < N::ROUNDS; ++u)
        if (L.wave + u * NWAVES < N::ITEMS) L.put_tile(to + (L.wave + u * NWAVES) * 1024, acc[u]);
    if constexpr (N::PARTS > 1) {
        __syncthreads();
        float v[2 * N::NM];
        L.sum_tiles(to, N::PARTS, v);
#pragma unroll
        for (int m = 0; m < 2 * N::NM; ++m) part_out[m * 512 + threadIdx.x] = v[m];
    }
    for (int c = threadIdx.x; c < 2 * N::DP * cpr; c += NW_T) {
        const int row = c / cpr, q = c - row * cpr;
        *reinterpret_cast<u32x4_t*>(xg + (int64_t)c * 16) = *reinterpret_cast<const u32x4_t*>(L.x + row * L.xs + q * 16);
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------
constexpr int CUS = 256;
struct Tiles { int sym, upd; };                // tile edges of the symmetric and the update products
struct Choice { Tiles large, small; };         // ... of the matrices with d > 256, and of the others
struct Layout {
    int64_t table, firsts, part, planes, total;      // byte offsets
    int64_t plane_elems;
    int count, parts, maxW, tiles[GRIDS];
};
int esize(int dt) { return dt == POET_F32 ? 4 : 2; }
int up(int v, int m) { return (v + m - 1) / m * m; }

// How a matrix is worked on, from its own shape alone (so that its result does not depend on what else is in the list):
// 0 = the chain, SMALL = the chain of small tiles (d <= 256), D = one workgroup (d <= 32 D), MAX_D + D = slabs
constexpr int SMALL = MAX_D + MAX_SLAB_D + 1, GROUPS = SMALL + 1;
int group_of(int rows, int cols, int& W) {
    const int d = rows < cols ? rows : cols, n = rows < cols ? cols : rows, D = cdiv(d, 32);
    W = 0;
    if (d > 256) return 0;
    if (D <= MAX_D && n <= W_MAX[D]) {                       // (66 x 256: 55 us against 70 with the chain; 60 x 300: 44 against 72; 120 x 150 would take 80 against 72)
        W = up(n, 32);
        return D;
    }
    // slabs of 256 columns (at most 8, wider then): 20 x 2000: 47 us against 123 with the chain, four 60 x 1500: 73 against 119; with three tiles
    // of rows and more the chain wins (90 x 400: 96 against 78, 131 x 257: 115 against 79)
    if (D > MAX_SLAB_D || n > MAX_SLABS * W_MAX[D]) return SMALL;
    const int slabs = cdiv(n, 256) < MAX_SLABS ? cdiv(n, 256) : MAX_SLABS;
    W = up(cdiv(n, slabs), 32);
    return MAX_D + D;
}

Choice tiles_of(const int* rows, const int* cols, int n) {
    // d > 256: 128 x 128 tiles halve the operand traffic per product, 64 x 64 tiles make (up to) four times as many workgroups.  The update takes the
    // large ones once they keep half of the CUs busy (1024 x 1024, 64 tiles: 302 us against 230, 1536 x 1536, 144 tiles: 402 against 419, 2048 x
    // 2048, 256 tiles: 763 against 822, 4 x 4096 x 1024: 1119 against 1476), the symmetric products
    // once they fill it (2048 x 2048, 136 tiles: 783 against 763, 6 x 1024 x 1024, 216 tiles: 549 against 531, 3000 x 3000, 300 tiles:
    // 2019 against 2066).  d <= 256: 32 x 32 tiles while they fit the chip once (twice in the update): four 256 x 256 83 us against
    // 110, seven 95 against 115; sixteen 144 against 111, ten 1024 x 256 231 against 169.
    int64_t sym = 0, upd = 0, ssym = 0, supd = 0;
    for (int i = 0; i < n; ++i) {
        int W;
        const int group = group_of(rows[i], cols[i], W), d = rows[i] < cols[i] ? rows[i] : cols[i];
        if (group == 0) {
            const int64_t td = cdiv(d, 128);
            sym += td * (td + 1) / 2;
            upd += (int64_t)cdiv(rows[i], 128) * cdiv(cols[i], 128);
        } else if (group == SMALL) {
            const int64_t td = cdiv(d, 32);
            ssym += td * (td + 1) / 2;
            supd += (int64_t)cdiv(rows[i], 32) * cdiv(cols[i], 32);
        }
    }
    return {{sym >= CUS ? 128 : 64, upd >= CUS / 2 ? 128 : 64}, {ssym > 256 ? 64 : 32, supd > 512 ? 64 : 32}};
}

// the records of one group among matrices [first, n) -- or among order[first .. n) -- (at most `most` of them): shape-dependent members into rec
// (when given), sizes into L; returns the index behind the last one taken, or -1: too large
int layout(const int* rows, const int* cols, const int* order, int first, int n, int group, const Choice& choice, int most, Layout& L, Rec* rec) {
    const Tiles T = group == SMALL ? choice.small : choice.large;
    const int P = T.sym == 128 || T.upd == 128 ? 128 : 64;   // planes hold whole tiles of every kind
    int64_t planes = 0, parts = 0, tiles[GRIDS] = {0, 0, 0};
    int i = first, count = 0;
    L.maxW = 0;
    for (; i < n && count < most; ++i) {
        Rec r = {};
        const int m = order ? order[i] : i;
        if (group_of(rows[m], cols[m], r.W) != group) continue;
        r.rows = rows[m];
        r.cols = cols[m];
        r.turned = r.rows > r.cols;
        r.d = r.turned ? r.cols : r.rows;
        r.n = r.turned ? r.rows : r.cols;
        const int64_t e = (int64_t)r.rows * r.cols;
        r.nb = (int)(e > 256ll * NORM_ELEMS ? 256 : cdiv(e, NORM_ELEMS));
        int64_t mine[GRIDS] = {0, 0, 0};
        r.x0 = planes;
        if (group == 0 || group == SMALL) {
            r.dp = up(r.d, P);
            r.np = up(r.n, P);
            r.x1 = r.x0 + 2 * (int64_t)r.dp * r.np;
            r.am = r.x1 + 2 * (int64_t)r.dp * r.np;
            r.bm = r.am + 2 * (int64_t)r.dp * r.dp;
            planes = r.bm + 2 * (int64_t)r.dp * r.dp;
            // Staged 64 x 64 tiles run k in steps of 64, so that next to 32 x 32 ones the rows up to a multiple of 64 must be there (as zeros):
            // one kind of product writes what the other reads
            const int rows_of_tiles = group == SMALL && (T.sym == 64 || T.upd == 64) ? r.dp : r.d;
            const int64_t td = cdiv(rows_of_tiles, T.sym);
            mine[SYM] = td * (td + 1) / 2;
            mine[UPD] = (int64_t)cdiv(rows_of_tiles, T.upd) * (r.np / T.upd);
            mine[PACK] = (int64_t)(r.dp / 64) * (r.np / 64);
        } else if (group > MAX_D) {           // slabs
            const int D = group - MAX_D, slabs = cdiv(r.n, r.W);
            const int64_t gram = (int64_t)slabs * D * (D + 1) / 2 * 2048;       // fp32 partial tiles, in 16-bit elements
            r.am = r.x0 + (int64_t)slabs * 2 * 32 * D * r.W;
            r.bm = r.am + gram;
            planes = r.bm + gram;
            mine[SYM] = slabs;
        }
        if (r.W > L.maxW) L.maxW = r.W;
        r.part0 = (int)parts;
        parts += r.nb;
        for (int k = 0; k < GRIDS; ++k) {
            if (tiles[k] + mine[k] > (1 << 29)) return -1;
            r.first[k] = (int)tiles[k];
            tiles[k] += mine[k];
        }
        if (rec) rec[count] = r;
        ++count;
    }
    if (group > 0 && group <= MAX_D && (int64_t)count * NW_T >= 1ll << 32) return -1;      // (a workgroup each: more threads than a launch can have)
    L.count = count;
    L.parts = (int)parts;
    L.plane_elems = planes;
    for (int k = 0; k < GRIDS; ++k) L.tiles[k] = (int)tiles[k];
    L.table = 0;
    L.firsts = ((int64_t)count * sizeof(Rec) + 15) / 16 * 16;
    L.part = (L.firsts + (int64_t)count * GRIDS * 4 + 15) / 16 * 16;
    L.planes = (L.part + parts * 8 + 255) / 256 * 256;
    L.total = (L.planes + planes * 2 + 255) / 256 * 256;
    if (group > 0 && group <= MAX_D) L.total = count > CHUNK ? L.firsts : 0;      // (all in LDS; the table of a long list)
    L.total = (L.total + 255) / 256 * 256;
    return i;
}

// The order of a group's matrices in the grids: as listed when they are of one length; else the long ones first, dealt to the 8 XCDs (each takes a
// contiguous eighth of a grid's tiles), so that no XCD is left with all the long sums of X X^T (15 matrices of 256 x 256, 5 of 512 x 256 and 10
// of 1024 x 256: 280 -> 249 us).  order: room for 3 n entries; returns their number.
int arrange(const int* rows, const int* cols, int n, int group, int* order) {
    int count = 0, W;
    bool same = true;
    auto length = [&](int i) { return rows[i] > cols[i] ? rows[i] : cols[i]; };
    for (int i = 0; i < n; ++i)
        if (group_of(rows[i], cols[i], W) == group) {
            order[count++] = i;
            same = same && length(i) == length(order[0]);
        }
    if (same) return count;
    int *sorted = order + n, *bin = sorted + n;
    int64_t load[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int k = 0; k < count; ++k) sorted[k] = order[k];
    std::sort(sorted, sorted + count, [&](int a, int b) { return length(a) != length(b) ? length(a) > length(b) : a < b; });
    for (int k = 0; k < count; ++k) {
        const int64_t t = cdiv(rows[sorted[k]] < cols[sorted[k]] ? rows[sorted[k]] : cols[sorted[k]], 32);
        bin[k] = (int)(std::min_element(load, load + 8) - load);
        load[bin[k]] += t * (t + 1) / 2;
    }
    int at = 0;
    for (int b = 0; b < 8; ++b)
        for (int k = 0; k < count; ++k)
            if (bin[k] == b) order[at++] = sorted[k];
    return count;
}

// exponents that keep X_k, A and q of every step within a quarter of fp16's range; false: the iteration leaves any useful range
struct Steps { int ex[MAX_STEPS + 1], ea[MAX_STEPS], eq[MAX_STEPS]; };
bool ranges(const double* coeffs, int steps, Steps& S) {
    auto exponent = [](double bound) { return 13 - (int)ceil(log2(bound > 1e-6 ? bound : 1e-6)); };
    double xb = 1.0001;
    for (int k = 0; k < steps; ++k) {
        const double a = coeffs[3 * k], b = coeffs[3 * k + 1], c = coeffs[3 * k + 2];
        if (!isfinite(a + b + c)) return false;
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

// split: d <= 256, where sums have four parts whichever tile is taken
template <int T, int BK, int SETS, int SLOTS, int Q> void sym_staged(const StageP& p, hipStream_t st) {
    static unsigned long long done = 0;
    constexpr int lds = Core<T, BK, false, SETS, SLOTS>::LDS;
    lds_attr_once((const void*)muon_sym_kernel<T, BK, SETS, SLOTS, Q>, lds, done);
    hipLaunchKernelGGL((muon_sym_kernel<T, BK, SETS, SLOTS, Q>), dim3(p.total), dim3(threads_of(T)), lds, st, p);
}
template <int T, int BK, int SETS, int SLOTS, bool LAST> void update_staged(const StageP& p, hipStream_t st) {
    static unsigned long long done = 0;
    constexpr int lds = Core<T, BK, true, SETS, SLOTS>::LDS;
    lds_attr_once((const void*)muon_update_kernel<T, BK, SETS, SLOTS, LAST>, lds, done);
    hipLaunchKernelGGL((muon_update_kernel<T, BK, SETS, SLOTS, LAST>), dim3(p.total), dim3(threads_of(T)), lds, st, p);
}
template <int Q> void sym_product(int T, bool split, const StageP& p, hipStream_t st) {
    if (T == 32) hipLaunchKernelGGL((muon_sym_split_kernel<Q>), dim3(p.total), dim3(NT), 0, st, p);
    else if (split && p.total > CUS) sym_staged<64, 64, 4, 2, Q>(p, st);
    else if (split) sym_staged<64, 64, 4, 4, Q>(p, st);
    else if (T == 64 && p.total > CUS) sym_staged<64, 64, 1, 2, Q>(p, st);
    else if (T == 64) sym_staged<64, 64, 1, 4, Q>(p, st);
    else if (p.total > CUS) sym_staged<128, 32, 1, 2, Q>(p, st);
    else sym_staged<128, 32, 1, 4, Q>(p, st);
}
template <bool LAST> void update_product(int T, bool split, const StageP& p, hipStream_t st) {
    if (T == 32) hipLaunchKernelGGL((muon_update_split_kernel<LAST>), dim3(p.total), dim3(NT), 0, st, p);
    else if (split && p.total > CUS) update_staged<64, 64, 4, 2, LAST>(p, st);
    else if (split) update_staged<64, 64, 4, 4, LAST>(p, st);
    else if (T == 64 && p.total > CUS) update_staged<64, 64, 1, 2, LAST>(p, st);
    else if (T == 64) update_staged<64, 64, 1, 4, LAST>(p, st);
    else if (p.total > CUS) update_staged<128, 32, 1, 2, LAST>(p, st);
    else update_staged<128, 32, 1, 4, LAST>(p, st);
}
StageP stage_params(const Layout& L, const Job& j, const Steps& S, char* ws) {
    StageP p = {};
    p.table = (const Rec*)(ws + L.table);
    p.firsts = (const int*)(ws + L.firsts);
    p.part = (const double*)(ws + L.part);
    p.planes = (_Float16*)(ws + L.planes);
    p.count = L.count;
    p.g_dtype = j.g_dtype; p.o_dtype = j.o_dtype; p.muon = j.muon; p.nesterov = j.nesterov;
    p.mu = (float)j.mu; p.omu = (float)(1.0 - j.mu); p.eps = j.eps; p.gscale = j.gscale; p.max_norm = j.max_norm; p.sqnorm = j.sqnorm;
    p.lr = j.lr; p.wd = j.wd;
    p.out_exp = pow2(S.ex[0]);
    return p;
}
void chain(Tiles T, bool split, const Rec& first, bool one_shape, const Layout& L, const Job& j, const Steps& S, char* ws, hipStream_t st) {
    StageP p = stage_params(L, j, S, ws);
    if (one_shape) {
        p.uniform = {first.x0, first.x1, first.am, first.bm, first.d, first.n, first.dp, first.np};
        p.stride = L.plane_elems / L.count;
        p.per[SYM] = L.tiles[SYM] / L.count;
        p.per[UPD] = L.tiles[UPD] / L.count;
    }
    hipLaunchKernelGGL(muon_pack_kernel, dim3(L.tiles[PACK]), dim3(NT), 0, st, p);
    for (int k = 0; k < j.steps; ++k) {
        p.flip = k & 1;
        p.total = L.tiles[SYM];
        p.in_scale = pow2(-2 * S.ex[k]);
        p.out_exp = pow2(S.ea[k]);
        sym_product<0>(T.sym, split, p, st);
        p.a = (float)j.coeffs[3 * k];
        p.b = (float)(j.coeffs[3 * k + 1] * pow2(-S.ea[k]));
        p.c = (float)j.coeffs[3 * k + 2];
        p.in_scale = pow2(-2 * S.ea[k]);
        p.out_exp = pow2(S.eq[k]);
        sym_product<1>(T.sym, split, p, st);
        p.total = L.tiles[UPD];
        p.in_scale = pow2(-S.eq[k] - S.ex[k]);
        p.out_exp = pow2(S.ex[k + 1]);
        if (k + 1 < j.steps) update_product<false>(T.upd, split, p, st);
        else update_product<true>(T.upd, split, p, st);
    }
}
NarrowP narrow_params(const Layout& L, const Job& j, const Steps& S, char* ws) {
    NarrowP p = {};
    p.s = stage_params(L, j, S, ws);
    p.steps = j.steps;
    for (int k = 0; k < j.steps; ++k) {
        p.a[k] = (float)j.coeffs[3 * k];
        p.b[k] = (float)(j.coeffs[3 * k + 1] * pow2(-S.ea[k]));
        p.c[k] = (float)(j.coeffs[3 * k + 2] * pow2(-2 * S.ea[k]));
        p.ascale[k] = pow2(S.ea[k] - 2 * S.ex[k]);
        p.qscale[k] = pow2(S.eq[k]);
        p.xscale[k] = pow2((k + 1 < j.steps ? S.ex[k + 1] : 0) - S.eq[k] - S.ex[k]);
    }
    return p;
}
template <int D> int narrow_lds(int W) { return Narrow<D>::REGION + 2 * Narrow<D>::DP * (W * 2 + 16); }
template <int D> void narrow_single(const NarrowP& p, const Recs& recs, int count, int W, hipStream_t st) {       // records: recs, or p.s.table
    static unsigned long long done = 0;
    static_assert(Narrow<D>::REGION + 2 * Narrow<D>::DP * (W_MAX[D] * 2 + 16) + 256 <= 160 * 1024, "LDS");
    lds_attr_once((const void*)muon_narrow_kernel<D>, narrow_lds<D>(W_MAX[D]), done);
    hipLaunchKernelGGL((muon_narrow_kernel<D>), dim3(count), dim3(NW_T), narrow_lds<D>(W), st, p, recs);
}
template <int D> void narrow_slabs(NarrowP p, const Layout& L, hipStream_t st) {
    static unsigned long long done = 0;
    lds_attr_once((const void*)muon_slab_kernel<D>, narrow_lds<D>(W_MAX[D]), done);
    for (int k = -1; k < p.steps; ++k) {
        p.mode = k < 0 ? N_INIT : k + 1 < p.steps ? N_STEP : N_LAST;
        p.k = k < 0 ? 0 : k;
        hipLaunchKernelGGL((muon_slab_kernel<D>), dim3(L.tiles[SYM]), dim3(NW_T), narrow_lds<D>(L.maxW), st, p);
    }
}

// bytes of all groups (at least one aligned block), -1: too large
int64_t workspace_of(const int* rows, const int* cols, int n, const Choice& T) {
    int64_t need = 0;
    for (int group = 0; group < GROUPS; ++group) {
        Layout L;
        if (layout(rows, cols, nullptr, 0, n, group, T, n, L, nullptr) < 0) return -1;
        need += L.total;
    }
    return need > 256 ? need : 256;
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
    const Choice T = tiles_of(j.rows, j.cols, j.n);
    const int64_t need = workspace_of(j.rows, j.cols, j.n, T);
    POET_CHECK(need >= 0, POET_ERR_UNSUPPORTED, "%s: too many matrices or tiles", what);
    POET_CHECK(ws && ((uintptr_t)ws % 256) == 0 && ws_bytes >= need, POET_ERR_ARG, "%s: workspace of %lld bytes needed (256-byte aligned), %lld given", what,
               (long long)need, (long long)ws_bytes);
    struct Ints {
        int* p;
        ~Ints() { delete[] p; }
    } order = {new (std::nothrow) int[3 * (size_t)j.n]};
    POET_CHECK(order.p, POET_ERR_ARG, "%s: no host memory for a list of %d", what, j.n);
    hipStream_t st = (hipStream_t)stream;
    char* base = (char*)ws;
    for (int group = 0; group < GROUPS; ++group) {
        Layout L;
        const int members = arrange(j.rows, j.cols, j.n, group, order.p);
        if (!members) continue;
        layout(j.rows, j.cols, order.p, 0, members, group, T, members, L, nullptr);
        const bool single = group > 0 && group <= MAX_D;
        NormP np = {};
        np.table = (Rec*)(base + L.table);
        np.firsts = (int*)(base + L.firsts);
        np.part = (double*)(base + L.part);
        np.n = L.count;
        np.g_dtype = j.g_dtype; np.muon = j.muon; np.nesterov = j.nesterov;
        np.mu = (float)j.mu; np.omu = (float)(1.0 - j.mu); np.gscale = j.gscale; np.max_norm = j.max_norm; np.sqnorm = j.sqnorm;
        NarrowP narrow = narrow_params(L, j, S, base);
        Recs short_list = {};
        int64_t planes = 0;                                   // of the chunks before this one
        int parts = 0, tiles[GRIDS] = {0, 0, 0};
        Rec shape = {};
        bool one_shape = true;
        for (int at = 0; np.first < L.count;) {
            Recs recs = {};
            Layout C;
            const int from = at;
            at = layout(j.rows, j.cols, order.p, from, members, group, T, CHUNK, C, recs.r);
            int blocks = 0;
            for (int c = 0; c < C.count; ++c) {
                const int i = order.p[from + c];
                Rec& r = recs.r[c];
                if (np.first + c == 0) shape = r;
                one_shape = one_shape && r.d == shape.d && r.n == shape.n;
                r.x0 += planes; r.x1 += planes; r.am += planes; r.bm += planes;
                r.part0 += parts;
                for (int k = 0; k < GRIDS; ++k) r.first[k] += tiles[k];
                r.g = j.g[i];
                r.o = j.o[i];
                r.mom = j.muon ? j.mom[i] : nullptr;
                r.p16 = j.p16 ? j.p16[i] : nullptr;
                r.p16lo = j.p16lo ? j.p16lo[i] : nullptr;
                r.lr_scale = j.lr_scale ? j.lr_scale[i] : nullptr;
                r.ldg = j.ldg ? j.ldg[i] : r.cols;
                r.ldo = j.ldo ? j.ldo[i] : r.cols;
                r.out_scale = j.out_scale ? j.out_scale[i] : 1.f;
                const int ge = esize(j.g_dtype), oe = esize(j.o_dtype), gw = 16 / ge;
                r.gvec = r.ldg == r.cols && (int64_t)r.rows * r.cols % gw == 0 && ((uintptr_t)r.g | (uintptr_t)r.mom) % 16 == 0;
                r.rows_vec = r.cols % 4 == 0 && r.ldg % 4 == 0 && (uintptr_t)r.g % (4 * ge) == 0 && (uintptr_t)r.mom % 16 == 0;
                r.ovec = r.cols % 4 == 0 && r.ldo % 4 == 0 && (uintptr_t)r.o % (4 * oe) == 0 && ((uintptr_t)r.p16 | (uintptr_t)r.p16lo) % 8 == 0;
                blocks += r.nb;
            }
            np.count = C.count;
            if (!single) hipLaunchKernelGGL(muon_norm_kernel, dim3(blocks), dim3(NT), 0, st, np, recs);
            else if (L.count > CHUNK) hipLaunchKernelGGL(muon_table_kernel, dim3(1), dim3(NT), 0, st, np.table + np.first, C.count, recs);
            else short_list = recs;
            planes += C.plane_elems;
            parts += C.parts;
            for (int k = 0; k < GRIDS; ++k) tiles[k] += C.tiles[k];
            np.first += C.count;
        }
        if (single) {                                         // (a hundred 66 x 256: 5 launches of 24 one after the other 258 us, 68 with the table)
            if (L.count <= CHUNK) narrow.s.table = nullptr;
            if (group == 1) narrow_single<1>(narrow, short_list, L.count, L.maxW, st);
            else if (group == 2) narrow_single<2>(narrow, short_list, L.count, L.maxW, st);
            else narrow_single<3>(narrow, short_list, L.count, L.maxW, st);
        } else if (group == 0) chain(T.large, false, shape, one_shape, L, j, S, base, st);
        else if (group == SMALL) chain(T.small, true, shape, one_shape, L, j, S, base, st);
        else if (group == MAX_D + 1) narrow_slabs<1>(narrow, L, st);
        else if (group == MAX_D + 2) narrow_slabs<2>(narrow, L, st);
        base += L.total;
    }
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
    const int64_t need = workspace_of(rows_host, cols_host, n, tiles_of(rows_host, cols_host, n));
    POET_CHECK(need >= 0, POET_ERR_UNSUPPORTED, "muon_workspace: too many matrices or tiles");
    return need;
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
