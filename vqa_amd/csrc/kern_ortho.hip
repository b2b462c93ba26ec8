// Orthogonalised updates: Newton-Schulz products that carry the singular values of a matrix towards 1, and the
// optimizer step around them (momentum, orthogonalisation, weight update).
//
// X0 = G / (|G|_F + eps), then `steps` times  A = X X^T,  X <- a X + (b A + c A A) X.  A singular value s of X goes to
// a s + b s^3 + c s^5 and the singular vectors stay, so the result is U p(S) V^T of G = U S V^T without an SVD.
// r = min(rows, cols), c = max: X is taken r x c (the transpose of a matrix with more rows than columns).
//
// Two forms:
// * r <= 64 and X fits the LDS of a CU: one workgroup carries a matrix through all steps (k_ns_small), in 64-bit or
//   32-bit matrix instructions.
// * else: three tiled products a step (k_ns_product), X, X^T, A and b A + c A A in device memory, all row-major with the
//   summed index contiguous, padded with zeros to whole tiles.  64-bit matrices use 64-bit matrix instructions; the
//   others hold every value as a sum of two 16-bit floats hi + lo (22 bits and a sign, scaled so that neither part
//   leaves its normal range) and take the three products hi hi + hi lo + lo hi with 32-bit sums: the left-out lo lo is
//   2^-22 of a product, the size of the roundings that 32-bit products make along a sum, at 5 times their rate.
#include <math.h>
#include <stdlib.h>

#include <algorithm>

#include "vqa_core.h"

namespace vqa {

namespace {

constexpr int kT = 256;
constexpr int kWaves = kT / 64;

typedef double double4v __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef _Float16 half4v __attribute__((ext_vector_type(4)));

// ---- stored types; C: the type of the state and of the products' sums --------------------------------------------
struct F64 { using S = double; using C = double;
    static __device__ C up(S v) { return v; } static __device__ S down(C v) { return v; } };
struct F32 { using S = float; using C = float;
    static __device__ C up(S v) { return v; } static __device__ S down(C v) { return v; } };
struct F16 { using S = _Float16; using C = float;
    static __device__ C up(S v) { return (float)v; } static __device__ S down(C v) { return (_Float16)v; } };
struct BF16 { using S = uint16_t; using C = float;
    static __device__ C up(S v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ S down(C v) {   // round to nearest even; NaN stays NaN
        const uint32_t u = __float_as_uint(v);
        if (v != v) return (uint16_t)((u >> 16) | 0x40);
        return (uint16_t)((u + 0x7fff + ((u >> 16) & 1)) >> 16);
    } };

// what a call does, by value to every kernel
template <class Ty>
struct Job {
    using S = typename Ty::S;
    using C = typename Ty::C;
    const S* g;
    int64_t g_row, g_batch;    // strides in elements
    S* out;                    // [batch, rows, cols], contiguous (null: an optimizer step)
    C* w;                      // optimizer step: weights and momentum, contiguous
    C* m;
    C mu, decay, rate;         // w <- decay w - rate O
    int nesterov;
    int batch, rows, cols, r, c, turned, steps;
    C ka, kb, kc;
    double eps;

    // element e of a matrix in row-major order as it enters the products; first: the momentum is brought up to date
    template <bool kFirst>
    __device__ __forceinline__ C enter(int b, int64_t row, int64_t col) const {
        const C v = Ty::up(g[b * g_batch + row * g_row + col]);
        if (!m) return v;
        const int64_t at = ((int64_t)b * rows + row) * cols + col;
        C mm = m[at];
        if (kFirst) m[at] = mm = mu * mm + v;
        return nesterov ? v + mu * mm : mm;
    }
    __device__ __forceinline__ void leave(int b, int64_t row, int64_t col, C o) const {
        const int64_t at = ((int64_t)b * rows + row) * cols + col;
        if (m) w[at] = decay * w[at] - rate * o;
        else out[at] = Ty::down(o);
    }
};

__device__ __forceinline__ double block_sum(double v, double* sh) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0;
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) s += sh[w];
    return s;
}

// ---- 16 x 16 x 4 matrix instruction: lane l holds A[l % 16][l / 16], B[l / 16][l % 16]; D[row(l, reg)][l % 16] ------
template <class C> struct Mma;
template <> struct Mma<double> {
    using Acc = double4v;
    static __device__ Acc go(double a, double b, Acc c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }
    static __device__ int row(int l, int reg) { return (l >> 4) + 4 * reg; }
};
template <> struct Mma<float> {
    using Acc = float4v;
    static __device__ Acc go(float a, float b, Acc c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
    static __device__ int row(int l, int reg) { return 4 * (l >> 4) + reg; }
};

// ---- one workgroup a matrix ---------------------------------------------------------------------------------------
constexpr int kSmallRows = 64;

int pad16(int v) { return (v + 15) / 16 * 16; }
size_t small_lds(int r, int c, size_t size) {
    const size_t rp = pad16(r), cp = pad16(c);
    return (rp * (cp + 4) + 2 * rp * (rp + 4) + 4 * 256) * size + 64;
}

template <class Ty>
__global__ __launch_bounds__(kT) void k_ns_small(Job<Ty> j) {
    using C = typename Ty::C;
    using Acc = typename Mma<C>::Acc;
    extern __shared__ char lds[];
    const int rp = (j.r + 15) / 16 * 16, cp = (j.c + 15) / 16 * 16, nt = rp / 16;
    const int ldx = cp + 4, lda = rp + 4;
    double* sh = (double*)lds;
    C* X = (C*)(lds + 64);
    C* A = X + rp * ldx;
    C* B = A + rp * lda;
    C* part = B + rp * lda;              // [4][256]: a single tile's product, its summed index in four parts
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, lk = lane >> 4;

    for (int b = blockIdx.x; b < j.batch; b += gridDim.x) {
        for (int i = threadIdx.x; i < rp * ldx; i += kT) X[i] = C(0);
        __syncthreads();
        double ss = 0;
        const int n = j.rows * j.cols;
        for (int e = threadIdx.x; e < n; e += kT) {
            const int row = e / j.cols, col = e - row * j.cols;
            const C v = j.template enter<true>(b, row, col);
            X[j.turned ? col * ldx + row : row * ldx + col] = v;
            ss += (double)v * (double)v;
        }
        const double norm = sqrt(block_sum(ss, sh)) + j.eps;
        for (int i = threadIdx.x; i < rp * ldx; i += kT) X[i] = (C)((double)X[i] / norm);
        __syncthreads();

        const int tiles = nt * (nt + 1) / 2, parts = nt == 1 ? kWaves : 1;
        for (int s = 0; s < j.steps; ++s) {
            // A = X X^T, its lower tiles
            for (int it = wave; it < tiles * parts; it += kWaves) {
                const int t = it / parts, p = it - t * parts;
                int ti = 0;
                while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
                const int tj = t - ti * (ti + 1) / 2, len = cp / parts;
                const C* xa = X + (ti * 16 + lr) * ldx + p * len + lk;
                const C* xb = X + (tj * 16 + lr) * ldx + p * len + lk;
                Acc acc = { 0, 0, 0, 0 };
                for (int k = 0; k < len; k += 4) acc = Mma<C>::go(xa[k], xb[k], acc);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int row = Mma<C>::row(lane, q);
                    if (parts > 1) part[p * 256 + row * 16 + lr] = acc[q];
                    else {
                        A[(ti * 16 + row) * lda + tj * 16 + lr] = acc[q];
                        A[(tj * 16 + lr) * lda + ti * 16 + row] = acc[q];
                    }
                }
            }
            __syncthreads();
            if (parts > 1) {
                const int e = threadIdx.x;
                A[(e >> 4) * lda + (e & 15)] = (part[e] + part[256 + e]) + (part[512 + e] + part[768 + e]);
                __syncthreads();
            }
            // B = b A + c A A
            for (int t = wave; t < tiles; t += kWaves) {
                int ti = 0;
                while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
                const int tj = t - ti * (ti + 1) / 2;
                const C* xa = A + (ti * 16 + lr) * lda + lk;
                const C* xb = A + (tj * 16 + lr) * lda + lk;
                Acc acc = { 0, 0, 0, 0 };
                for (int k = 0; k < rp; k += 4) acc = Mma<C>::go(xa[k], xb[k], acc);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int row = Mma<C>::row(lane, q);
                    const C v = j.kb * A[(ti * 16 + row) * lda + tj * 16 + lr] + j.kc * acc[q];
                    B[(ti * 16 + row) * lda + tj * 16 + lr] = v;
                    B[(tj * 16 + lr) * lda + ti * 16 + row] = v;
                }
            }
            __syncthreads();
            // X <- a X + B X, a strip of 16 columns by one wave: it reads all of the strip before it writes any
            for (int n0 = wave * 16; n0 < cp; n0 += kWaves * 16) {
                Acc acc[kSmallRows / 16];
#pragma unroll
                for (int i = 0; i < kSmallRows / 16; ++i) acc[i] = Acc{ 0, 0, 0, 0 };
                for (int k = 0; k < rp; k += 4) {
                    const C xb = X[(k + lk) * ldx + n0 + lr];
#pragma unroll
                    for (int i = 0; i < kSmallRows / 16; ++i)
                        if (i < nt) acc[i] = Mma<C>::go(B[(i * 16 + lr) * lda + k + lk], xb, acc[i]);
                }
#pragma unroll
                for (int i = 0; i < kSmallRows / 16; ++i)
                    if (i < nt)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            C* x = X + (i * 16 + Mma<C>::row(lane, q)) * ldx + n0 + lr;
                            *x = j.ka * *x + acc[i][q];
                        }
            }
            __syncthreads();
        }
        for (int e = threadIdx.x; e < n; e += kT) {
            const int row = e / j.cols, col = e - row * j.cols;
            j.leave(b, row, col, X[j.turned ? col * ldx + row : row * ldx + col]);
        }
        __syncthreads();
    }
}

// ---- tiled products -------------------------------------------------------------------------------------------------
constexpr int kTile = 64;
constexpr int kNormParts = 256;

// Scales of the 16-bit pairs (powers of two).  Entries of X are at most the largest singular value, below 4 by the
// caller's check, and 1 / sqrt(r c) at the start; of A below 16; of b A + c A A below 32.
constexpr float kSX = 4096.f, kSA = 1024.f, kSB = 1024.f;

// values of a padded matrix: 64-bit, or a 16-bit pair in two arrays
struct Pair {
    _Float16 *hi, *lo;
    __device__ __forceinline__ float get(size_t i, float scale) const { return ((float)hi[i] + (float)lo[i]) * (1.f / scale); }
    __device__ __forceinline__ void put(size_t i, float v, float scale) const {
        v *= scale;
        const _Float16 h = (_Float16)v;
        hi[i] = h;
        lo[i] = (_Float16)(v - (float)h);
    }
    // 16 neighbours, the first at a multiple of 16
    __device__ __forceinline__ void get16(size_t i, float scale, float* v) const {
        const half8v h0 = *(const half8v*)(hi + i), h1 = *(const half8v*)(hi + i + 8);
        const half8v l0 = *(const half8v*)(lo + i), l1 = *(const half8v*)(lo + i + 8);
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            v[n] = ((float)h0[n] + (float)l0[n]) * (1.f / scale);
            v[8 + n] = ((float)h1[n] + (float)l1[n]) * (1.f / scale);
        }
    }
    __device__ __forceinline__ void put16(size_t i, const float* v, float scale) const {
        half8v h[2], l[2];
#pragma unroll
        for (int n = 0; n < 16; ++n) {
            const float x = v[n] * scale;
            h[n >> 3][n & 7] = (_Float16)x;
            l[n >> 3][n & 7] = (_Float16)(x - (float)h[n >> 3][n & 7]);
        }
        *(half8v*)(hi + i) = h[0];
        *(half8v*)(hi + i + 8) = h[1];
        *(half8v*)(lo + i) = l[0];
        *(half8v*)(lo + i + 8) = l[1];
    }
    __device__ __forceinline__ Pair at(size_t bytes) const { return Pair{ (_Float16*)((char*)hi + bytes), (_Float16*)((char*)lo + bytes) }; }
};
struct Wide {
    double* v;
    __device__ __forceinline__ double get(size_t i, float) const { return v[i]; }
    __device__ __forceinline__ void put(size_t i, double x, float) const { v[i] = x; }
    __device__ __forceinline__ void get16(size_t i, float, double* x) const {
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const double2 d = *(const double2*)(v + i + 2 * n);
            x[2 * n] = d.x;
            x[2 * n + 1] = d.y;
        }
    }
    __device__ __forceinline__ void put16(size_t i, const double* x, float) const {
#pragma unroll
        for (int n = 0; n < 8; ++n) *(double2*)(v + i + 2 * n) = make_double2(x[2 * n], x[2 * n + 1]);
    }
    __device__ __forceinline__ Wide at(size_t bytes) const { return Wide{ (double*)((char*)v + bytes) }; }
};
template <class C> struct StoreOf { using T = Pair; };
template <> struct StoreOf<double> { using T = Wide; };

// a matrix's working memory: X and X^T twice (a step reads one and writes the other), A, b A + c A A, partial sums
template <class M>
struct Mats {
    M x[2], xt[2], a, b;
    double* part;
    size_t stride;    // bytes to the next matrix of the batch
    int rp, cp;
};

template <class Ty>
__global__ __launch_bounds__(kT) void k_ns_norm(Job<Ty> j, double* part, size_t stride) {
    __shared__ double sh[kWaves];
    const int b = blockIdx.y;
    const int64_t n = (int64_t)j.rows * j.cols;
    double ss = 0;
    for (int64_t e = (int64_t)blockIdx.x * kT + threadIdx.x; e < n; e += (int64_t)gridDim.x * kT) {
        const int64_t row = e / j.cols, col = e - row * j.cols;
        const double v = (double)j.template enter<true>(b, row, col);
        ss += v * v;
    }
    ss = block_sum(ss, sh);
    if (threadIdx.x == 0) ((double*)((char*)part + b * stride))[blockIdx.x] = ss;
}

// X0 and its transpose, a tile a workgroup
template <class Ty>
__global__ __launch_bounds__(kT) void k_ns_enter(Job<Ty> j, Mats<typename StoreOf<typename Ty::C>::T> w, int norm_parts) {
    using C = typename Ty::C;
    __shared__ double sh[kWaves];
    __shared__ C tile[kTile][kTile + 1];
    const int b = blockIdx.z;
    const size_t off = b * w.stride;
    const double* part = (const double*)((char*)w.part + off);
    const double norm = sqrt(block_sum((int)threadIdx.x < norm_parts ? part[threadIdx.x] : 0.0, sh)) + j.eps;
    // rows and columns of the caller's matrix
    const int64_t r0 = (int64_t)(j.turned ? blockIdx.x : blockIdx.y) * kTile, c0 = (int64_t)(j.turned ? blockIdx.y : blockIdx.x) * kTile;
    for (int e = threadIdx.x; e < kTile * kTile; e += kT) {
        const int y = e / kTile, x = e % kTile;
        tile[y][x] = r0 + y < j.rows && c0 + x < j.cols ? (C)((double)j.template enter<false>(b, r0 + y, c0 + x) / norm) : C(0);
    }
    __syncthreads();
    const auto xm = w.x[0].at(off), xt = w.xt[0].at(off);
    const size_t x0 = (size_t)blockIdx.y * kTile, y0 = (size_t)blockIdx.x * kTile;   // row and column of X
    for (int e = threadIdx.x; e < kTile * kTile; e += kT) {
        const int y = e / kTile, x = e % kTile;
        xm.put((x0 + y) * w.cp + y0 + x, j.turned ? tile[x][y] : tile[y][x], kSX);
        xt.put((y0 + y) * w.rp + x0 + x, j.turned ? tile[y][x] : tile[x][y], kSX);
    }
}

enum Kind { kGram, kPoly, kUpdate, kLast };

// 16 bytes of global memory straight to LDS, lane l's to base + 16 l (base: the same for the wave)
__device__ __forceinline__ void copy_to_lds(const void* from, void* base) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)base, 16, 0, 0);
}

// D[i][j] = sum_k P[i][k] Q[j][k] of one T x T tile
template <class C, int T> struct Tile;
template <int T> struct Tile<float, T> {
    // T = 256: 8 waves of 128 x 64;  128 and 64: 4 waves of T/2 x T/2
    static constexpr int kThreads = T == 256 ? 512 : 256, kWv = kThreads / 64;
    static constexpr int WJ = T == 256 ? 4 : 2;                     // waves side by side
    static constexpr int NI = T == 256 ? 4 : T / 64, NJ = T == 256 ? 2 : T / 64;   // 32 x 32 blocks of a wave
    static constexpr int BK = 32;
    float16v acc[NI][NJ];
    // A stage holds BK values of T rows of the four arrays; a row is 4 pieces of 16 bytes, whose order in the row is
    // turned by swz(row), so that the 16 rows a quarter of a wave reads at once lie in different banks.
    static __device__ __forceinline__ int swz(int row) { return (((row >> 1) ^ (row >> 3)) & 1) | ((row >> 2) & 1) << 1; }
    static constexpr int kArray = T * BK;                 // values of one array in a stage
    static constexpr int kStage = 4 * kArray;
    static constexpr size_t kBytes = 2 * kStage * sizeof(_Float16);
    static_assert(kBytes >= kWv * 32 * 33 * sizeof(float));

    static __device__ __forceinline__ int wave_i() { return (threadIdx.x >> 6) / WJ * (NI * 32); }
    static __device__ __forceinline__ int wave_j() { return (threadIdx.x >> 6) % WJ * (NJ * 32); }

    __device__ __forceinline__ void fetch(const Pair& p, const Pair& q, size_t i0, size_t j0, int ld, int k, _Float16* st) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
        for (int n = 0; n < T / (16 * kWv); ++n) {
            const int r0 = (n * kWv + wave) * 16, row = r0 + (lane >> 2);
            const size_t x = k + ((lane & 3) ^ swz(row)) * 8;
            const size_t ap = (i0 + row) * ld + x, aq = (j0 + row) * ld + x;
            copy_to_lds(p.hi + ap, st + r0 * BK);
            copy_to_lds(p.lo + ap, st + kArray + r0 * BK);
            copy_to_lds(q.hi + aq, st + 2 * kArray + r0 * BK);
            copy_to_lds(q.lo + aq, st + 3 * kArray + r0 * BK);
        }
    }
    __device__ __forceinline__ void run(const Pair& p, const Pair& q, size_t i0, size_t j0, int ld, int K, char* shared) {
        _Float16* lds = (_Float16*)shared;
        const int lane = threadIdx.x & 63, half = lane >> 5;
        const int wi = wave_i() + (lane & 31), wj = wave_j() + (lane & 31);
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) acc[i][j] = 0.f;
        fetch(p, q, i0, j0, ld, 0, lds);
        int at = 0;
        for (int k = 0; k < K; k += BK) {
            // this stage has arrived (each wave waits for its own copies, the barrier for the waves), the other one was read
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (k + BK < K) fetch(p, q, i0, j0, ld, k + BK, lds + (at ^ 1) * kStage);
            const _Float16* st = lds + at * kStage;
            at ^= 1;
#pragma unroll
            for (int kk = 0; kk < BK / 16; ++kk) {
                half8v ph[NI], pl[NI], qh[NJ], ql[NJ];
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const int r = wj + 32 * j, x = r * BK + ((2 * kk + half) ^ swz(r)) * 8;
                    qh[j] = *(const half8v*)(st + 2 * kArray + x);
                    ql[j] = *(const half8v*)(st + 3 * kArray + x);
                }
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const int r = wi + 32 * i, x = r * BK + ((2 * kk + half) ^ swz(r)) * 8;
                    ph[i] = *(const half8v*)(st + x);
                    pl[i] = *(const half8v*)(st + kArray + x);
                }
#pragma unroll
                for (int i = 0; i < NI; ++i) {
#pragma unroll
                    for (int j = 0; j < NJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(pl[i], qh[j], acc[i][j], 0, 0, 0);
#pragma unroll
                    for (int j = 0; j < NJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph[i], ql[j], acc[i][j], 0, 0, 0);
#pragma unroll
                    for (int j = 0; j < NJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph[i], qh[j], acc[i][j], 0, 0, 0);
                }
            }
        }
    }
    // The result block by block: a wave lays its 32 x 32 blocks one after another into its own part of the shared memory
    // (after the barrier: the stages are read) and hands each to f(row, column of the block, block).
    template <class F>
    __device__ __forceinline__ void blocks(char* shared, F f) {
        const int lane = threadIdx.x & 63;
        auto blk = (float(*)[33])shared + (threadIdx.x >> 6) * 32;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
#pragma unroll
                for (int q = 0; q < 16; ++q) blk[8 * (q >> 2) + 4 * (lane >> 5) + (q & 3)][lane & 31] = acc[i][j][q];
                f(wave_i() + 32 * i, wave_j() + 32 * j, blk);
            }
    }
};
template <> struct Tile<double, 64> {
    static constexpr int kThreads = 256;
    static constexpr int BK = 16;
    static constexpr size_t kBytes = kWaves * 32 * 33 * sizeof(double);   // of the result's blocks; the stages take less
    static_assert(kBytes >= 2 * 64 * (BK + 2) * sizeof(double));
    double4v acc[2][2];
    __device__ __forceinline__ void run(const Wide& p, const Wide& q, size_t i0, size_t j0, int ld, int K, char* shared) {
        double(*sp)[BK + 2] = (double(*)[BK + 2])shared, (*sq)[BK + 2] = sp + 64;
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const int wi = (wave >> 1) * 32, wj = (wave & 1) * 32;
        const int y = threadIdx.x >> 2, x = (threadIdx.x & 3) * 4;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int jj = 0; jj < 2; ++jj) acc[i][jj] = double4v{ 0, 0, 0, 0 };
        for (int k = 0; k < K; k += BK) {
            const double2* ap = (const double2*)(p.v + (i0 + y) * ld + k + x);
            const double2* aq = (const double2*)(q.v + (j0 + y) * ld + k + x);
            const double2 a = ap[0], b = ap[1], c = aq[0], d = aq[1];
            __syncthreads();
            *(double2*)&sp[y][x] = a;
            *(double2*)&sp[y][x + 2] = b;
            *(double2*)&sq[y][x] = c;
            *(double2*)&sq[y][x + 2] = d;
            __syncthreads();
#pragma unroll
            for (int kk = 0; kk < BK; kk += 4) {
                double pv[2], qv[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    pv[i] = sp[wi + 16 * i + (lane & 15)][kk + (lane >> 4)];
                    qv[i] = sq[wj + 16 * i + (lane & 15)][kk + (lane >> 4)];
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int jj = 0; jj < 2; ++jj) acc[i][jj] = Mma<double>::go(pv[i], qv[jj], acc[i][jj]);
            }
        }
    }
    template <class F>
    __device__ __forceinline__ void blocks(char* shared, F f) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        auto blk = (double(*)[33])shared + wave * 32;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int jj = 0; jj < 2; ++jj)
#pragma unroll
                for (int q = 0; q < 4; ++q) blk[16 * i + Mma<double>::row(lane, q)][16 * jj + (lane & 15)] = acc[i][jj][q];
        f((wave >> 1) * 32, (wave & 1) * 32, blk);
    }
};

// One product of a step.  kGram: A = X X^T;  kPoly: B = b A + c A A  (lower tiles, written to both sides of the
// diagonal);  kUpdate: X <- a X + B X as its transpose X^T B, both layouts written;  kLast: the same to the caller.
template <class Ty, Kind kind, int T>
__global__ __launch_bounds__((Tile<typename Ty::C, T>::kThreads)) void k_ns_product(Job<Ty> j, Mats<typename StoreOf<typename Ty::C>::T> w, int from) {
    using C = typename Ty::C;
    constexpr bool kSym = kind == kGram || kind == kPoly;
    extern __shared__ __attribute__((aligned(16))) char product_lds[];
    const size_t off = blockIdx.z * w.stride;
    size_t ti = blockIdx.y, tj = blockIdx.x;
    if (kSym) {
        ti = (size_t)((sqrtf(8.f * blockIdx.x + 1.f) - 1.f) * 0.5f);
        while (ti * (ti + 1) / 2 > blockIdx.x) --ti;
        while ((ti + 1) * (ti + 2) / 2 <= blockIdx.x) ++ti;
        tj = blockIdx.x - ti * (ti + 1) / 2;
    }
    const size_t i0 = ti * T, j0 = tj * T;
    const auto a = w.a.at(off), bm = w.b.at(off);
    Tile<C, T> t;
    // a lane's 16 neighbours of a block: half a row, or half a column
    const int lane = threadIdx.x & 63, line = lane >> 1, half = (lane & 1) * 16;
    if (kind == kGram || kind == kPoly) {
        const auto& src = kind == kGram ? w.x[from] : w.a;
        const auto m = src.at(off), out = kind == kGram ? a : bm;
        const int ld = kind == kGram ? w.cp : w.rp;
        t.run(m, m, i0, j0, ld, ld, product_lds);
        const float so = kind == kGram ? kSA : kSB;
        const C f = sizeof(C) == 8 ? C(1) : kind == kGram ? C(1.f / (kSX * kSX)) : C(1.f / (kSA * kSA));
        t.blocks(product_lds, [&](int bi, int bj, C(*blk)[33]) {
            const size_t y = i0 + bi + line, x = j0 + bj + half;
            C v[16];
            if (kind == kPoly) {
                a.get16(y * w.rp + x, kSA, v);
#pragma unroll
                for (int n = 0; n < 16; ++n) blk[line][half + n] = v[n] = j.kb * v[n] + j.kc * (f * blk[line][half + n]);
            } else {
#pragma unroll
                for (int n = 0; n < 16; ++n) blk[line][half + n] = v[n] = f * blk[line][half + n];
            }
            out.put16(y * w.rp + x, v, so);
            if (ti == tj) return;
#pragma unroll
            for (int n = 0; n < 16; ++n) v[n] = blk[half + n][line];
            out.put16((j0 + bj + line) * w.rp + i0 + bi + half, v, so);
        });
    } else {
        const auto xt = w.xt[from].at(off), nx = w.x[from ^ 1].at(off), nt = w.xt[from ^ 1].at(off);
        t.run(xt, bm, i0, j0, w.rp, w.rp, product_lds);   // rows: columns of X; columns: rows of X
        const C f = sizeof(C) == 8 ? C(1) : C(1.f / (kSX * kSB));
        t.blocks(product_lds, [&](int bi, int bj, C(*blk)[33]) {
            const size_t y = i0 + bi + line, x = j0 + bj + half;
            C v[16];
            xt.get16(y * w.rp + x, kSX, v);
#pragma unroll
            for (int n = 0; n < 16; ++n) blk[line][half + n] = v[n] = j.ka * v[n] + f * blk[line][half + n];
            if (kind == kUpdate) {
                nt.put16(y * w.rp + x, v, kSX);
#pragma unroll
                for (int n = 0; n < 16; ++n) v[n] = blk[half + n][line];
                nx.put16((j0 + bj + line) * w.cp + i0 + bi + half, v, kSX);
            } else {
                // the caller's rows are the block's rows (turned) or its columns: 32 neighbours of a row by half a wave
                const int64_t r0 = (j.turned ? i0 + bi : j0 + bj) + (lane >> 5), col = (j.turned ? j0 + bj : i0 + bi) + (lane & 31);
#pragma unroll
                for (int n = 0; n < 16; ++n) {
                    const int d = 2 * n + (lane >> 5);
                    const C o = j.turned ? blk[d][lane & 31] : blk[lane & 31][d];
                    if (r0 + 2 * n < j.rows && col < j.cols) j.leave(blockIdx.z, r0 + 2 * n, col, o);
                }
            }
        });
    }
}

// ---- launches -------------------------------------------------------------------------------------------------------
constexpr size_t kLds = 160 * 1024;

bool is_small(int dtype, int r, int c) {
    return r <= kSmallRows && c <= 32768 && small_lds(r, c, dtype == VQA_DTYPE_F64 ? 8 : 4) <= kLds;
}
// Side of a product's tile.  128 where the update has at least as many tiles as half the chip's CUs
int tile_of(int dtype, int batch, int r, int c) {
    if (dtype == VQA_DTYPE_F64) return 64;
    const int64_t n = (int64_t)((r + 127) / 128) * ((c + 127) / 128) * batch;
    static const int forced = getenv("NS_TILE") ? atoi(getenv("NS_TILE")) : 0;
    if (forced) return forced;
    return n >= 1024 ? 256 : n >= 128 ? 128 : 64;
}
int pad_to(int v, int t) { return (v + t - 1) / t * t; }
size_t up256(size_t v) { return (v + 255) / 256 * 256; }

template <class M>
size_t lay_out(char* base, int r, int c, int tile, Mats<M>* w);
template <>
size_t lay_out<Pair>(char* base, int r, int c, int tile, Mats<Pair>* w) {
    w->rp = pad_to(r, tile);
    w->cp = pad_to(c, tile);
    const size_t x = up256((size_t)w->rp * w->cp * 2), a = up256((size_t)w->rp * w->rp * 2);
    char* p = base;
    auto next = [&](size_t n) { char* q = p; p += n; return (_Float16*)q; };
    for (int i = 0; i < 2; ++i) {
        w->x[i].hi = next(x); w->x[i].lo = next(x);
        w->xt[i].hi = next(x); w->xt[i].lo = next(x);
    }
    w->a.hi = next(a); w->a.lo = next(a);
    w->b.hi = next(a); w->b.lo = next(a);
    w->part = (double*)p;
    p += kNormParts * 8;
    return w->stride = (size_t)(p - base);
}
template <>
size_t lay_out<Wide>(char* base, int r, int c, int tile, Mats<Wide>* w) {
    w->rp = pad_to(r, tile);
    w->cp = pad_to(c, tile);
    const size_t x = up256((size_t)w->rp * w->cp * 8), a = up256((size_t)w->rp * w->rp * 8);
    char* p = base;
    auto next = [&](size_t n) { char* q = p; p += n; return (double*)q; };
    for (int i = 0; i < 2; ++i) {
        w->x[i].v = next(x);
        w->xt[i].v = next(x);
    }
    w->a.v = next(a);
    w->b.v = next(a);
    w->part = (double*)p;
    p += kNormParts * 8;
    return w->stride = (size_t)(p - base);
}

// Dynamic shared memory beyond 64 KB is asked for once for each kernel and device
template <class F>
int allow_lds(F* fn, size_t bytes) {
    static uint64_t done = 0;   // a bit a device; asking twice does no harm
    int dev = 0;
    VQA_HIP(hipGetDevice(&dev));
    if (bytes > 65536 && !(done >> (dev & 63) & 1)) {
        VQA_HIP(hipFuncSetAttribute((const void*)fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)kLds));
        done |= (uint64_t)1 << (dev & 63);
    }
    return VQA_OK;
}

template <class Ty, Kind kind, int T>
int product(hipStream_t st, dim3 grid, const Job<Ty>& j, const Mats<typename StoreOf<typename Ty::C>::T>& w, int from) {
    using Tl = Tile<typename Ty::C, T>;
    if (int rc = allow_lds(k_ns_product<Ty, kind, T>, Tl::kBytes)) return rc;
    hipLaunchKernelGGL((k_ns_product<Ty, kind, T>), grid, dim3(Tl::kThreads), Tl::kBytes, st, j, w, from);
    return VQA_OK;
}

template <class Ty, int T>
int steps(hipStream_t st, const Job<Ty>& j, const Mats<typename StoreOf<typename Ty::C>::T>& w) {
    const unsigned tr = w.rp / T, tc = w.cp / T, sym = tr * (tr + 1) / 2, nb = (unsigned)j.batch;
    int rc = VQA_OK;
    for (int s = 0; s < j.steps && !rc; ++s) {
        const int from = s & 1;
        rc = product<Ty, kGram, T>(st, dim3(sym, 1, nb), j, w, from);
        if (!rc) rc = product<Ty, kPoly, T>(st, dim3(sym, 1, nb), j, w, from);
        if (!rc) rc = s + 1 < j.steps ? product<Ty, kUpdate, T>(st, dim3(tr, tc, nb), j, w, from) : product<Ty, kLast, T>(st, dim3(tr, tc, nb), j, w, from);
    }
    return rc;
}

template <class Ty>
int run(hipStream_t st, const OrthoCall& q) {
    using C = typename Ty::C;
    Job<Ty> j;
    j.g = (const typename Ty::S*)q.g;
    j.g_row = q.g_row_stride;
    j.g_batch = q.g_batch_stride;
    j.out = (typename Ty::S*)q.out;
    j.w = (C*)q.weight;
    j.m = (C*)q.momentum;
    j.mu = (C)q.mu;
    j.decay = (C)(1.0 - q.lr * q.weight_decay);
    j.rate = (C)(q.lr * sqrt(std::max(1.0, (double)q.rows / (double)q.cols)));
    j.nesterov = q.nesterov;
    j.batch = q.batch;
    j.rows = q.rows;
    j.cols = q.cols;
    j.r = std::min(q.rows, q.cols);
    j.c = std::max(q.rows, q.cols);
    j.turned = q.rows > q.cols;
    j.steps = q.steps;
    j.ka = (C)q.coefs[0];
    j.kb = (C)q.coefs[1];
    j.kc = (C)q.coefs[2];
    j.eps = q.eps;
    if (is_small(q.dtype, j.r, j.c)) {
        const size_t lds = small_lds(j.r, j.c, sizeof(C));
        if (int rc = allow_lds(k_ns_small<Ty>, lds)) return rc;
        hipLaunchKernelGGL((k_ns_small<Ty>), dim3((unsigned)q.batch), dim3(kT), lds, st, j);
        VQA_HIP(hipGetLastError());
        return VQA_OK;
    }
    Mats<typename StoreOf<C>::T> w;
    const int tile = tile_of(q.dtype, q.batch, j.r, j.c);
    lay_out((char*)q.workspace, j.r, j.c, tile, &w);
    const int64_t n = (int64_t)j.rows * j.cols;
    const int parts = (int)std::min<int64_t>(kNormParts, (n + 4 * kT - 1) / (4 * kT));
    const unsigned nb = (unsigned)q.batch;
    hipLaunchKernelGGL((k_ns_norm<Ty>), dim3(parts, nb), dim3(kT), 0, st, j, w.part, w.stride);
    hipLaunchKernelGGL((k_ns_enter<Ty>), dim3(w.cp / kTile, w.rp / kTile, nb), dim3(kT), 0, st, j, w, parts);
    int rc;
    if constexpr (sizeof(C) == 4) {
        rc = tile == 256 ? steps<Ty, 256>(st, j, w) : tile == 128 ? steps<Ty, 128>(st, j, w) : steps<Ty, 64>(st, j, w);
    } else rc = steps<Ty, 64>(st, j, w);
    if (rc) return rc;
    VQA_HIP(hipGetLastError());
    return VQA_OK;
}

}  // namespace

size_t ortho_workspace_bytes(int dtype, int batch, int rows, int cols) {
    const int r = std::min(rows, cols), c = std::max(rows, cols);
    if (is_small(dtype, r, c)) return 0;
    if (dtype == VQA_DTYPE_F64) {
        Mats<Wide> w;
        return lay_out<Wide>(nullptr, r, c, tile_of(dtype, batch, r, c), &w) * (size_t)batch;
    }
    Mats<Pair> w;
    return lay_out<Pair>(nullptr, r, c, tile_of(dtype, batch, r, c), &w) * (size_t)batch;
}

int ortho_launch(hipStream_t stream, const OrthoCall& q) {
    switch (q.dtype) {
        case VQA_DTYPE_F64: return run<F64>(stream, q);
        case VQA_DTYPE_F32: return run<F32>(stream, q);
        case VQA_DTYPE_BF16: return run<BF16>(stream, q);
        default: return run<F16>(stream, q);
    }
}

}  // namespace vqa
