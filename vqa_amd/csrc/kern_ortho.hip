// Orthogonalised updates: Newton-Schulz products that carry the singular values of a matrix towards 1, and the
// optimizer step around them (momentum, orthogonalisation, weight update).
//
// X0 = G / (|G|_F + eps), then `steps` times  A = X X^T,  X <- a X + (b A + c A A) X.  A singular value s of X goes to
// a s + b s^3 + c s^5 and the singular vectors stay, so the result is U p(S) V^T of G = U S V^T without an SVD.
// r = min(rows, cols), c = max: X is taken r x c (the transpose of a matrix with more rows than columns).
//
// Four forms:
// * r <= 16, short rows: one workgroup carries a matrix through all steps, X in the registers of its waves in strips of 16
//   columns (k_ns_strip), in 64-bit or 32-bit matrix instructions.  (64-bit rows beyond 1024, eight strips a wave: 64 of the
//   registers lie in scratch.)
// * r <= 64, short rows: the same with X in shared memory (k_ns_block).
// * r <= 64, long rows: the steps on X X^T alone, between two passes over the matrix (k_ns_gram, k_ns_poly, k_ns_apply).
// * else: three tiled products a step (k_ns_product), X, X^T, A and b A + c A A in device memory, all row-major with the
//   summed index contiguous, padded to whole tiles.  64-bit matrices use 64-bit matrix instructions; the others hold every
//   value as a sum of two 16-bit floats hi + lo (22 bits and a sign, scaled by powers of two that follow X's size) and
//   take the three products hi hi + hi lo + lo hi with 32-bit sums: the left-out lo lo is 2^-22 of a product, the size of
//   the roundings that 32-bit products make along a sum, at 5 times their rate.
#include <math.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

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

    // A thread's U elements as they enter the products, all loads under way before the first is used.  at(u, row, col) names
    // element u (false: there is none, 0).  kFirst: the momentum is brought up to date.
    template <bool kFirst, int U, class F>
    __device__ __forceinline__ void enter(int b, C* v, F at) const {
        const S* gb = g + b * g_batch;
        C* mb = m + (int64_t)b * rows * cols;
        S raw[U];
        C mm[U];
        bool ok[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            int row = 0, col = 0;
            ok[u] = at(u, row, col);
            raw[u] = gb[ok[u] ? row * g_row + col : 0];
        }
        if (m) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                int row = 0, col = 0;
                mm[u] = at(u, row, col) ? mb[(int64_t)row * cols + col] : C(0);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            v[u] = ok[u] ? Ty::up(raw[u]) : C(0);
            if (m) {
                int row = 0, col = 0;
                at(u, row, col);
                if (kFirst) {
                    mm[u] = mu * mm[u] + v[u];
                    if (ok[u]) mb[(int64_t)row * cols + col] = mm[u];
                }
                v[u] = nesterov ? v[u] + mu * mm[u] : mm[u];
            }
        }
    }
    // U elements of the result, in the same way
    template <int U, class F>
    __device__ __forceinline__ void leave(int b, const C* o, F at) const {
        const int64_t base = (int64_t)b * rows * cols;
        int64_t to[U];
        bool ok[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            int row = 0, col = 0;
            ok[u] = at(u, row, col);
            to[u] = base + (ok[u] ? (int64_t)row * cols + col : 0);
        }
        if (m) {
            C ww[U];
#pragma unroll
            for (int u = 0; u < U; ++u) ww[u] = w[to[u]];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (ok[u]) w[to[u]] = decay * ww[u] - rate * o[u];
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (ok[u]) out[to[u]] = Ty::down(o[u]);
        }
    }
    // N neighbours of a row of the result from (row, col) on; those outside the matrix are left out
    template <int N>
    __device__ __forceinline__ void leave_run(int b, const C* o, int row, int col) const {
        const int64_t to = ((int64_t)b * rows + row) * cols + col;
        if (row < rows && col + N <= cols) {
            if (m ? aligned<C, N>(w + to) : aligned<S, N>(out + to)) {
                if (m) {
                    alignas(16) C v[N];
                    move<C, N>(v, w + to);
#pragma unroll
                    for (int n = 0; n < N; ++n) v[n] = decay * v[n] - rate * o[n];
                    move<C, N>(w + to, v);
                } else {
                    alignas(16) S v[N];
#pragma unroll
                    for (int n = 0; n < N; ++n) v[n] = Ty::down(o[n]);
                    move<S, N>(out + to, v);
                }
                return;
            }
        }
#pragma unroll
        for (int k = 0; k < N; k += 4) {   // (a few at a time: their places take registers)
            leave<4>(b, o + k, [&](int n, int& r, int& c) { r = row; c = col + k + n; return row < rows && col + k + n < cols; });
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    template <class E, int N> static constexpr int kPiece = N * sizeof(E) < 16 ? (int)(N * sizeof(E)) : 16;
    template <class E, int N> static __device__ __forceinline__ bool aligned(const E* p) { return (uintptr_t)p % kPiece<E, N> == 0; }
    template <class E, int N>
    static __device__ __forceinline__ void move(E* to, const E* from) {   // (both aligned to a piece)
        using V = std::conditional_t<kPiece<E, N> == 16, uint4, uint2>;
        static_assert(N * sizeof(E) % sizeof(V) == 0);
#pragma unroll
        for (int n = 0; n < (int)(N * sizeof(E) / sizeof(V)); ++n) ((V*)to)[n] = ((const V*)from)[n];
    }
};

// the elements of a rows x cols matrix in row-major order, T threads apart, U at a time: next(row, col) steps T elements on
template <int T>
struct Walk {
    int row, col, dr, dc, cols;
    __device__ __forceinline__ Walk(int first, int cols_) : row(first / cols_), col(first % cols_), dr(T / cols_), dc(T % cols_), cols(cols_) {}
    __device__ __forceinline__ void step() {
        row += dr;
        col += dc;
        if (col >= cols) { col -= cols; ++row; }
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

// |G| + eps from the sum of squares; NaN where the squares leave 64 bits (a matrix divided by infinity would pass for zero)
__device__ __forceinline__ double size_of_matrix(double squares, double eps) {
    return squares < __builtin_inf() ? sqrt(squares) + eps : __builtin_nan("");
}

// What a wave's lanes wrote to shared memory before this is what its lanes read after it (and the other way round).  The
// hardware runs a wave's shared memory accesses in order; this keeps the compiler from moving one lane's accesses past each
// other that do not meet in that lane.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
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

// ---- one workgroup a matrix, r <= 16: X in registers -----------------------------------------------------------------
// A wave holds strips of 16 columns: lane l has X[row(l, q)][l % 16] of a strip in register q, which is at once
// * the second operand of a product B X (summed index row(l, q)), and its result's layout: X never leaves its registers;
// * for a symmetric matrix the first operand as well, so A A and B X take A and B as the products before left them.
// Only X X^T needs X with the columns as summed index: each wave turns its own strip through shared memory and sums over its
// own columns; the waves' parts of A are added in a fixed order (one barrier a step, two with 16 waves).
// Bound by the chain of 12 dependent matrix instructions a step (64 cycles each in 64 bits).  11 x 36 in 64 bits: 6.4 us, with
// X in shared memory and a barrier between the products 14.5; 256 of 9 x 60 (one a CU) 7.7.
template <class Ty, int NW, int S>
__global__ __launch_bounds__(NW * 64) void k_ns_strip(Job<Ty> j) {
    using C = typename Ty::C;
    using Acc = typename Mma<C>::Acc;
    __shared__ double sh[NW];
    __shared__ C turn[NW][16][17];
    __shared__ C part[2][NW][256];
    __shared__ C total[NW > 4 ? 256 : 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15;
    const int active = min(NW, (j.c + 15) / 16);          // waves with a strip

    const int b = blockIdx.x;
    C x[S][4];
    constexpr int SU = S < 4 ? S : 4;                  // strips whose loads are under way at once
    // (of: the thread's number, as one value for the way in and another for the way out, so that the places of 4 S
    // elements are worked out twice and not kept in registers through the steps)
    int of = threadIdx.x;
    auto at = [&](int s0, int u, int& row, int& col) {
        const int r = Mma<C>::row(of & 63, u & 3), c = ((s0 + (u >> 2)) * NW + (of >> 6)) * 16 + (of & 15);
        row = j.turned ? c : r;
        col = j.turned ? r : c;
        return r < j.r && c < j.c;
    };
#pragma unroll
    for (int s = 0; s < S; s += SU)
        j.template enter<true, 4 * SU>(b, x[s], [&](int u, int& row, int& col) { return at(s, u, row, col); });
    double ss = 0;
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
        for (int q = 0; q < 4; ++q) ss += (double)x[s][q] * (double)x[s][q];
    const double norm = size_of_matrix(block_sum(ss, sh), j.eps);
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
        for (int q = 0; q < 4; ++q) x[s][q] = (C)((double)x[s][q] / norm);

    for (int step = 0; step < j.steps; ++step) {
        Acc acc = { 0, 0, 0, 0 };
#pragma unroll
        for (int s = 0; s < S; ++s)
            if ((s * NW + wave) * 16 < j.c) {
#pragma unroll
                for (int q = 0; q < 4; ++q) turn[wave][Mma<C>::row(lane, q)][lr] = x[s][q];
                wave_fence();
                C a[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) a[q] = turn[wave][lr][Mma<C>::row(lane, q)];
                wave_fence();
#pragma unroll
                for (int q = 0; q < 4; ++q) acc = Mma<C>::go(a[q], a[q], acc);
            }
        auto& pt = part[step & 1];                     // (the other one may still be read)
#pragma unroll
        for (int q = 0; q < 4; ++q) pt[wave][q * 64 + lane] = acc[q];
        __syncthreads();
        C A[4];
        if constexpr (NW > 4) {
            if (threadIdx.x < 256) {
                C v = pt[0][threadIdx.x];
                for (int w = 1; w < active; ++w) v += pt[w][threadIdx.x];
                total[threadIdx.x] = v;
            }
            __syncthreads();
#pragma unroll
            for (int q = 0; q < 4; ++q) A[q] = total[q * 64 + lane];
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                A[q] = pt[0][q * 64 + lane];
#pragma unroll
                for (int w = 1; w < NW; ++w) A[q] += pt[w][q * 64 + lane];
            }
        }
        Acc aa = { 0, 0, 0, 0 };
#pragma unroll
        for (int q = 0; q < 4; ++q) aa = Mma<C>::go(A[q], A[q], aa);
        C B[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) B[q] = j.kb * A[q] + j.kc * aa[q];
#pragma unroll
        for (int s = 0; s < S; ++s)
            if ((s * NW + wave) * 16 < j.c) {
                Acc up = { 0, 0, 0, 0 };
#pragma unroll
                for (int q = 0; q < 4; ++q) up = Mma<C>::go(B[q], x[s][q], up);
#pragma unroll
                for (int q = 0; q < 4; ++q) x[s][q] = j.ka * x[s][q] + up[q];
            }
    }
    asm volatile("" : "+v"(of));
#pragma unroll
    for (int s = 0; s < S; s += SU)
        j.template leave<4 * SU>(b, x[s], [&](int u, int& row, int& col) { return at(s, u, row, col); });
}

// ---- one workgroup a matrix, 16 < r <= 64: X, A and b A + c A A in shared memory --------------------------------------
// NT = r / 16 tile rows.  X X^T is dealt as (lower tile, part of the columns) over the 16 waves, the parts added in a fixed
// order; X <- a X + B X by strips of 16 columns, each read whole by its wave before it is written.
constexpr int kBlockWaves = 16, kBlockThreads = 64 * kBlockWaves;
template <int NT>
struct Block {
    static constexpr int kRows = 16 * NT, kTiles = NT * (NT + 1) / 2, kParts = kBlockWaves / kTiles, LDA = kRows + 4;
    static size_t bytes(int c, size_t size) {
        const size_t cp = (c + 15) / 16 * 16;
        return (kRows * (cp + 4) + 2 * kRows * LDA + (kParts > 1 ? kTiles * kParts * 256 : 0)) * size + 128;
    }
};

// the tile row and column of lower tile t
__device__ __forceinline__ void lower(int t, int& ti, int& tj) {
    ti = t >= 6 ? 3 : t >= 3 ? 2 : t >= 1 ? 1 : 0;
    tj = t - ti * (ti + 1) / 2;
}

// sum over n4 groups of 4 of xa[4 k] xb[4 k]: operands of four instructions are read before the first is issued
template <class C>
__device__ __forceinline__ typename Mma<C>::Acc dot16(const C* xa, const C* xb, int n4) {
    typename Mma<C>::Acc a0 = { 0, 0, 0, 0 }, a1 = { 0, 0, 0, 0 };
    int k = 0;
    for (; k + 4 <= n4; k += 4) {
        C p[4], q[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) { p[u] = xa[4 * (k + u)]; q[u] = xb[4 * (k + u)]; }
        a0 = Mma<C>::go(p[0], q[0], a0);
        a1 = Mma<C>::go(p[1], q[1], a1);
        a0 = Mma<C>::go(p[2], q[2], a0);
        a1 = Mma<C>::go(p[3], q[3], a1);
    }
    for (; k < n4; ++k) a0 = Mma<C>::go(xa[4 * k], xb[4 * k], a0);
    return a0 + a1;
}

// Bound by the matrix instructions of one CU and the reading of their operands: 48 x 250 in 32 bits 38 us, 64 x 128 in 64 bits
// 70 us = 0.12 TFLOP/s of the CU's 0.28 (20 registers of a thread lie in scratch there).
template <class Ty, int NT>
__global__ __launch_bounds__(kBlockThreads) void k_ns_block(Job<Ty> j) {
    using C = typename Ty::C;
    using Acc = typename Mma<C>::Acc;
    using Bl = Block<NT>;
    constexpr int rp = Bl::kRows, lda = Bl::LDA, tiles = Bl::kTiles, parts = Bl::kParts;
    extern __shared__ __attribute__((aligned(16))) char block_lds[];
    const int cp = (j.c + 15) / 16 * 16, ldx = cp + 4;
    double* sh = (double*)block_lds;
    C* X = (C*)(block_lds + 128);
    C* A = X + rp * ldx;
    C* B = A + rp * lda;
    C* part = B + rp * lda;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, lk = lane >> 4;
    // this wave's share of X X^T and of A A
    const int g_part = wave / tiles, g_tile = wave - g_part * tiles;
    int gi, gj, pi, pj;
    lower(g_tile, gi, gj);
    lower(wave < tiles ? wave : 0, pi, pj);
    const int n4 = cp / 4, per = (n4 + parts - 1) / parts, k0 = g_part * per, kn = min(per, n4 - k0);

    const int b = blockIdx.x;
    for (int i = threadIdx.x; i < rp * ldx; i += kBlockThreads) X[i] = C(0);
    __syncthreads();
    double ss = 0;
    for (Walk<kBlockThreads> w(threadIdx.x, j.cols); w.row < j.rows;) {
        int row[8], col[8];
        C v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) { row[u] = w.row; col[u] = w.col; w.step(); }
        j.template enter<true, 8>(b, v, [&](int u, int& r, int& c) { r = row[u]; c = col[u]; return row[u] < j.rows; });
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (row[u] < j.rows) X[j.turned ? col[u] * ldx + row[u] : row[u] * ldx + col[u]] = v[u];
            ss += (double)v[u] * (double)v[u];
        }
    }
    const double norm = size_of_matrix(block_sum(ss, sh), j.eps);
    for (int i = threadIdx.x; i < rp * ldx; i += kBlockThreads) X[i] = (C)((double)X[i] / norm);
    __syncthreads();

    for (int s = 0; s < j.steps; ++s) {
        // A = X X^T, its lower tiles
        if (g_part < parts) {
            const Acc acc = dot16<C>(X + (gi * 16 + lr) * ldx + 4 * k0 + lk, X + (gj * 16 + lr) * ldx + 4 * k0 + lk, kn);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int row = Mma<C>::row(lane, q);
                if constexpr (parts > 1) part[(g_part * tiles + g_tile) * 256 + row * 16 + lr] = acc[q];
                else {
                    A[(gi * 16 + row) * lda + gj * 16 + lr] = acc[q];
                    A[(gj * 16 + lr) * lda + gi * 16 + row] = acc[q];
                }
            }
        }
        __syncthreads();
        if constexpr (parts > 1) {
            for (int e = threadIdx.x; e < tiles * 256; e += kBlockThreads) {
                C v = part[e];
#pragma unroll
                for (int p = 1; p < parts; ++p) v += part[p * tiles * 256 + e];
                int ti, tj;
                lower(e >> 8, ti, tj);
                const int row = e >> 4 & 15, col = e & 15;
                A[(ti * 16 + row) * lda + tj * 16 + col] = v;
                A[(tj * 16 + col) * lda + ti * 16 + row] = v;
            }
            __syncthreads();
        }
        // B = b A + c A A
        if (wave < tiles) {
            const Acc acc = dot16<C>(A + (pi * 16 + lr) * lda + lk, A + (pj * 16 + lr) * lda + lk, rp / 4);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int row = Mma<C>::row(lane, q);
                const C v = j.kb * A[(pi * 16 + row) * lda + pj * 16 + lr] + j.kc * acc[q];
                B[(pi * 16 + row) * lda + pj * 16 + lr] = v;
                B[(pj * 16 + lr) * lda + pi * 16 + row] = v;
            }
        }
        __syncthreads();
        // X <- a X + B X
        for (int n0 = wave * 16; n0 < cp; n0 += kBlockWaves * 16) {
            Acc acc[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i) acc[i] = Acc{ 0, 0, 0, 0 };
#pragma unroll
            for (int k = 0; k < rp; k += 16) {
                C xb[4], bv[NT][4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    xb[u] = X[(k + 4 * u + lk) * ldx + n0 + lr];
#pragma unroll
                    for (int i = 0; i < NT; ++i) bv[i][u] = B[(i * 16 + lr) * lda + k + 4 * u + lk];
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int i = 0; i < NT; ++i) acc[i] = Mma<C>::go(bv[i][u], xb[u], acc[i]);
            }
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    C* x = X + (i * 16 + Mma<C>::row(lane, q)) * ldx + n0 + lr;
                    *x = j.ka * *x + acc[i][q];
                }
        }
        __syncthreads();
    }
    for (Walk<kBlockThreads> w(threadIdx.x, j.cols); w.row < j.rows;) {
        int row[8], col[8];
        C v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            row[u] = w.row;
            col[u] = w.col;
            v[u] = row[u] < j.rows ? X[j.turned ? col[u] * ldx + row[u] : row[u] * ldx + col[u]] : C(0);
            w.step();
        }
        j.template leave<8>(b, v, [&](int u, int& r, int& c) { r = row[u]; c = col[u]; return row[u] < j.rows; });
    }
}

// ---- r <= 64 and long rows: the steps on X X^T -------------------------------------------------------------------------
// What the steps make of X is P X with P a polynomial of A = X X^T: with Q = a I + b A + c A A a step takes P to Q P and A to
// Q A Q, r x r all.  So a round of steps reads the matrix twice (A; P X), and the r x r products between are a workgroup's.
// A has the squares of the singular values: an error u of it moves P X by up to |a|^(2 steps) u.  For matrices of 32 and 16
// bits, with the products in 64 bits, a round is as many steps as keep |a|^steps <= 2^13 (u |a|^(2 steps) <= 2^-27), with the
// usual coefficients all of them; 64-bit matrices take a round a step, and X lies in the workspace between rounds.
// (For any coefficients: with s' = p(s) a step takes an error of s^2 times (s' / s) p'(s), a round times (s_n / s_0) prod p', so
// s_n is off by u prod p' / (2 s_0) where steps on s itself in 32 bits are off by 2^-24 prod p': less from s_0 = 2^-30 on, and
// a smaller s_0 stays where p(s) is a s, as |a|^steps <= 2^13 does not carry it out of there.)
// All r x r matrices are symmetric: a lower tile a wave, written to both sides of the diagonal.
template <int NT>
struct Long {
    static constexpr int kRows = 16 * NT, kTiles = NT * (NT + 1) / 2, LD = kRows + 2;
    static constexpr size_t kBytes = (size_t)4 * kRows * LD * 8 + 64;
};
constexpr int kMaxParts = 16;   // of the columns of a matrix
struct LongWs {
    double* part;      // A0 of a part of the columns: [part][lower tile][16 x 16]
    double* poly;      // P (in the first round / (|G| + eps)), [16 NT][16 NT]
    double* x;         // X^T between rounds, [c][16 NT]
    size_t stride;     // bytes of a matrix
    int parts;
    template <class T> __device__ T* at(T* p, int b) const { return (T*)((char*)p + b * stride); }
};

// A of a part of the columns: each wave sums its own, operands straight from memory (a column's elements in 16 lanes).
// 256 x 17 x 2048 in 32 bits, us: 27 here (36 MB), 12 for the polynomials, 41 for P X (71 MB); 64 x 4096: 17, 35 and 14.
template <class Ty, int NT, bool kEnter>
__global__ __launch_bounds__(kT) void k_ns_gram(Job<Ty> j, LongWs w) {
    using Lg = Long<NT>;
    constexpr int V = 4;                                    // instructions' columns under way at once
    __shared__ double sum[2][kWaves][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b = blockIdx.y;
    const int per = ((j.c + 15) / 16 + w.parts - 1) / w.parts * 16, c0 = blockIdx.x * per, c1 = min(j.c, c0 + per);
    double4v acc[Lg::kTiles];
#pragma unroll
    for (int t = 0; t < Lg::kTiles; ++t) acc[t] = double4v{ 0, 0, 0, 0 };
    for (int k0 = c0 + wave * 4 * V; k0 < c1; k0 += kWaves * 4 * V) {
        std::conditional_t<kEnter, typename Ty::C, double> x[NT * V];
        if constexpr (kEnter) {
            j.template enter<true, NT * V>(b, x, [&](int u, int& row, int& col) {
                const int i = u / V * 16 + (lane & 15), k = k0 + u % V * 4 + (lane >> 4);
                row = j.turned ? k : i;
                col = j.turned ? i : k;
                return i < j.r && k < c1;
            });
        } else {
            const double* xt = w.at(w.x, b);
#pragma unroll
            for (int u = 0; u < NT * V; ++u) {
                const int k = k0 + u % V * 4 + (lane >> 4);
                x[u] = k < c1 ? xt[(size_t)k * Lg::kRows + u / V * 16 + (lane & 15)] : 0.0;
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int t = 0; t < Lg::kTiles; ++t) {
                int ti = 0, tj = 0;
                lower(t, ti, tj);
                acc[t] = Mma<double>::go((double)x[ti * V + v], (double)x[tj * V + v], acc[t]);
            }
    }
    double* out = w.at(w.part, b) + (size_t)blockIdx.x * Lg::kTiles * 256;
#pragma unroll
    for (int t = 0; t < Lg::kTiles; ++t) {
#pragma unroll
        for (int q = 0; q < 4; ++q) sum[t & 1][wave][Mma<double>::row(lane, q) * 16 + (lane & 15)] = acc[t][q];
        __syncthreads();
        double v = 0;
#pragma unroll
        for (int u = 0; u < kWaves; ++u) v += sum[t & 1][u][threadIdx.x];
        out[t * 256 + threadIdx.x] = v;
    }
}

// The steps of a round on A: three phases a step, each a barrier and N4 dependent matrix instructions (64 rows: 16 of them,
// 2.3 us a phase with the reading of the operands).
template <int NT>
__global__ __launch_bounds__(64 * Long<NT>::kTiles) void k_ns_poly(LongWs w, int r, int steps, double ka, double kb, double kc, double eps,
                                                                      bool first) {
    using Lg = Long<NT>;
    constexpr int R = Lg::kRows, LD = Lg::LD, T = 64 * Lg::kTiles, N4 = R / 4;
    extern __shared__ __attribute__((aligned(16))) char poly_lds[];
    double* A = (double*)poly_lds;
    double *Q = A + R * LD, *P = Q + R * LD, *W = P + R * LD, *inv = W + R * LD;
    const int lane = threadIdx.x & 63, b = blockIdx.x;
    int ti, tj;
    lower(threadIdx.x >> 6, ti, tj);
    const int row0 = ti * 16, col0 = tj * 16 + (lane & 15);
    // operands of the wave's tile of a product of symmetric matrices, and its elements of the result
    const int left = (row0 + (lane & 15)) * LD + (lane >> 4), right = col0 * LD + (lane >> 4);
    auto put = [&](double* m, const double4v& v) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int row = row0 + Mma<double>::row(lane, q);
            m[row * LD + col0] = v[q];
            if (ti != tj) m[col0 * LD + row] = v[q];
        }
    };
    auto get = [&](const double* m) {
        double4v v;
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = m[(row0 + Mma<double>::row(lane, q)) * LD + col0];
        return v;
    };
    {
        double4v v = { 0, 0, 0, 0 };
        const double* part = w.at(w.part, b) + (threadIdx.x >> 6) * 256 + (lane & 15);
#pragma unroll 4
        for (int p = 0; p < w.parts; ++p)
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] += part[(size_t)p * Lg::kTiles * 256 + Mma<double>::row(lane, q) * 16];
        put(A, v);
    }
    __syncthreads();
    double scale = 1;
    if (first) {
        if (threadIdx.x < 64) {
            double d = lane < r ? A[lane * LD + lane] : 0.0;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) d += __shfl_xor(d, o);
            if (lane == 0) *inv = 1.0 / size_of_matrix(d, eps);
        }
        __syncthreads();
        scale = *inv;
        double4v v = get(A);
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = v[q] * scale * scale;
        __syncthreads();
        put(A, v);
        __syncthreads();
    }
    for (int s = 0; s < steps; ++s) {
        double4v q = dot16<double>(A + left, A + right, N4);
        const double4v a = get(A);
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = kb * a[e] + kc * q[e] + (row0 + Mma<double>::row(lane, e) == col0 ? ka : 0.0);
        put(Q, q);
        if (s == 0) put(P, q);
        __syncthreads();
        double4v p, v;
        if (s > 0) p = dot16<double>(Q + left, P + right, N4);
        if (s + 1 < steps) {
            v = dot16<double>(Q + left, A + right, N4);
            put(W, v);
        }
        __syncthreads();
        if (s > 0) put(P, p);
        if (s + 1 < steps) {
            v = dot16<double>(W + left, Q + right, N4);
            put(A, v);
        }
        __syncthreads();
    }
    double* out = w.at(w.poly, b);
    for (int e = threadIdx.x; e < R * R; e += T) out[e] = P[e / R * LD + e % R] * scale;
}

// P X, P in shared memory, 16 columns a wave at a time
template <class Ty, int NT, bool kEnter, bool kLeave>
__global__ __launch_bounds__(kT) void k_ns_apply(Job<Ty> j, LongWs w) {
    using C = typename Ty::C;
    using Lg = Long<NT>;
    constexpr int R = Lg::kRows, LD = Lg::LD, N4 = R / 4;
    __shared__ double P[R * LD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, lk = lane >> 4, b = blockIdx.y;
    const double* from = w.at(w.poly, b);
    double* xt = w.at(w.x, b);
    for (int e = threadIdx.x; e < R * R; e += kT) P[e / R * LD + e % R] = from[e];
    __syncthreads();
    // 16 columns of X a wave, read whole before they are written
    for (int k0 = (blockIdx.x * kWaves + wave) * 16; k0 < j.c; k0 += gridDim.x * kWaves * 16) {
        std::conditional_t<kEnter, C, double> x[N4];
        if constexpr (kEnter) {
            j.template enter<false, N4>(b, x, [&](int u, int& row, int& col) {
                const int i = 4 * u + lk, k = k0 + lr;
                row = j.turned ? k : i;
                col = j.turned ? i : k;
                return i < j.r && k < j.c;
            });
        } else {
#pragma unroll
            for (int u = 0; u < N4; ++u) x[u] = k0 + lr < j.c ? xt[(size_t)(k0 + lr) * R + 4 * u + lk] : 0.0;
        }
        // (P is symmetric: the same operands give the result's transpose when they change places)
        const bool turned = !kLeave || j.turned;
        double4v o[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            o[t] = double4v{ 0, 0, 0, 0 };
#pragma unroll
            for (int u = 0; u < N4; ++u) {
                const double p = P[(t * 16 + lr) * LD + 4 * u + lk];
                o[t] = turned ? Mma<double>::go((double)x[u], p, o[t]) : Mma<double>::go(p, (double)x[u], o[t]);
            }
        }
        if constexpr (kLeave) {
            C v[4 * NT];
#pragma unroll
            for (int u = 0; u < 4 * NT; ++u) v[u] = (C)o[u >> 2][u & 3];
            j.template leave<4 * NT>(b, v, [&](int u, int& row, int& col) {
                const int d = Mma<double>::row(lane, u & 3), t = u >> 2;
                row = j.turned ? k0 + d : t * 16 + d;
                col = j.turned ? t * 16 + lr : k0 + lr;
                return row < j.rows && col < j.cols;
            });
        } else {
#pragma unroll
            for (int u = 0; u < 4 * NT; ++u) {
                const int k = k0 + Mma<double>::row(lane, u & 3);
                if (k < j.c) xt[(size_t)k * R + (u >> 2) * 16 + lr] = o[u >> 2][u & 3];
            }
        }
    }
}

// ---- tiled products -------------------------------------------------------------------------------------------------
constexpr int kTile = 64;
constexpr int kNormParts = 256;
constexpr int kMaxCount = 128;        // tiles of a product whose sum is split: at most half of the CUs

// Scales of the 16-bit pairs (powers of two).  Entries of X are at most the largest singular value, below 4 by the
// caller's check, and 1 / sqrt(r c) at the start; of A below 16; of b A + c A A below 32.
// Where |G| is far below eps, X starts small and grows by about |a| a step: it is held as 2^k X, and A and b A + c A A as
// 4^k times themselves, k of each matrix and step such that 2^k |X| <= 1 (b + c, so 4^k |b A + c A A|, at most 32 by the
// caller's check).  k = 0 from |X| = 1 / 2 on, which is where a matrix far above eps starts; with |a| >= 1, which the entry
// points ask for, X then stays of that size but for what cancels (a smaller |a| shrinks small singular values without bound,
// and only the size of X itself, not its bound, could be followed: 150 x 70 with (0, 1.5, -0.9), three steps, was 2e-4 off).
constexpr float kSX = 4096.f, kSA = 1024.f, kSB = 1024.f;
constexpr int kMostSteps = 100, kMostLift = 110;      // (2^-110 is left in the last product: its values stay normal numbers)
__device__ __forceinline__ int lift_of(float size) { return min(kMostLift, max(0, -1 - ilogbf(fmaxf(size, 1e-36f)))); }

// values of a padded matrix: 64-bit, or a 16-bit pair in two arrays
struct Pair {
    _Float16 *hi, *lo;
    // N neighbours, the first at a multiple of N; as they are stored (the load is under way), and their values
    template <int N>
    struct Raw {
        static constexpr int V = N < 8 ? N : 8;
        typedef _Float16 halves __attribute__((ext_vector_type(V)));
        halves h[N / V], l[N / V];
        __device__ __forceinline__ void values(float scale, float* v) const {
#pragma unroll
            for (int m = 0; m < N / V; ++m)
#pragma unroll
                for (int n = 0; n < V; ++n) v[m * V + n] = ((float)h[m][n] + (float)l[m][n]) * (1.f / scale);
        }
    };
    template <int N>
    __device__ __forceinline__ Raw<N> get(size_t i) const {
        using halves = typename Raw<N>::halves;
        Raw<N> r;
#pragma unroll
        for (int m = 0; m < N / Raw<N>::V; ++m) {
            r.h[m] = *(const halves*)(hi + i + m * Raw<N>::V);
            r.l[m] = *(const halves*)(lo + i + m * Raw<N>::V);
        }
        return r;
    }
    template <int N>
    __device__ __forceinline__ void put(size_t i, const float* v, float scale) const {
        constexpr int V = N < 8 ? N : 8;
        typedef _Float16 halves __attribute__((ext_vector_type(V)));
#pragma unroll
        for (int m = 0; m < N / V; ++m) {
            halves h, l;
#pragma unroll
            for (int n = 0; n < V; ++n) {
                const float x = v[m * V + n] * scale;
                h[n] = (_Float16)x;
                l[n] = (_Float16)(x - (float)h[n]);
            }
            *(halves*)(hi + i + m * V) = h;
            *(halves*)(lo + i + m * V) = l;
        }
    }
    __device__ __forceinline__ Pair at(size_t bytes) const { return Pair{ (_Float16*)((char*)hi + bytes), (_Float16*)((char*)lo + bytes) }; }
};
struct Wide {
    double* v;
    template <int N>
    struct Raw {
        double2 d[N / 2];
        __device__ __forceinline__ void values(float, double* x) const {
#pragma unroll
            for (int n = 0; n < N / 2; ++n) {
                x[2 * n] = d[n].x;
                x[2 * n + 1] = d[n].y;
            }
        }
    };
    template <int N>
    __device__ __forceinline__ Raw<N> get(size_t i) const {
        Raw<N> r;
#pragma unroll
        for (int n = 0; n < N / 2; ++n) r.d[n] = *(const double2*)(v + i + 2 * n);
        return r;
    }
    template <int N>
    __device__ __forceinline__ void put(size_t i, const double* x, float) const {
#pragma unroll
        for (int n = 0; n < N / 2; ++n) *(double2*)(v + i + 2 * n) = make_double2(x[2 * n], x[2 * n + 1]);
    }
    __device__ __forceinline__ Wide at(size_t bytes) const { return Wide{ (double*)((char*)v + bytes) }; }
};
template <class C> struct StoreOf { using T = Pair; };
template <> struct StoreOf<double> { using T = Wide; };

// a matrix's working memory: X and X^T twice (a step reads one and writes the other), A, b A + c A A, partial sums
template <class M>
struct Mats {
    M x[2], xt[2], a, b;
    double* part;     // of the norm
    void* sum;        // X X^T in parts: [tile][part][T x T], in C
    unsigned* count;  // parts of a tile that are there (0 between the kernels)
    int* lift;        // of 16-bit pairs: k of each step's X, and 0 for the result
    int splits;
    size_t stride;    // bytes to the next matrix of the batch
    // rows of X (and its columns) as they are stored, and as the products sum over them (r and c to whole stages).  Rows from
    // rk on, which the tiles of one product cover and those of another may not, hold anything: they are never summed over.
    int rp, cp, rk, ck;
};

// Parts of the sum of squares (and the momentum): a workgroup takes whole rows in turn, or, of few long rows, pieces of them.
// 16 loads of a thread are under way at once.  4096 x 4096 bfloat16: 21 us = 1.6 TB/s (with 4 under way 127).
template <class Ty>
__global__ __launch_bounds__(kT) void k_ns_norm(Job<Ty> j, double* part, size_t stride, int pieces) {
    using C = typename Ty::C;
    constexpr int U = 16;
    __shared__ double sh[kWaves];
    const int b = blockIdx.y;
    double ss = 0;
    for (int it = blockIdx.x; it < j.rows * pieces; it += gridDim.x) {
        const int row = it / pieces, per = (j.cols + pieces - 1) / pieces, c0 = (it - row * pieces) * per, c1 = min(j.cols, c0 + per);
        for (int c = c0 + threadIdx.x; c < c1; c += kT * U) {
            C v[U];
            j.template enter<true, U>(b, v, [&](int u, int& r, int& cc) { r = row; cc = c + u * kT; return c + u * kT < c1; });
#pragma unroll
            for (int u = 0; u < U; ++u) ss += (double)v[u] * (double)v[u];
        }
    }
    ss = block_sum(ss, sh);
    if (threadIdx.x == 0) ((double*)((char*)part + b * stride))[blockIdx.x] = ss;
}

// X0 and its transpose, a tile a workgroup, and the scales of the steps.  4096 x 4096 bfloat16: 43 to 46 us = 3.7 to 3.9 TB/s of the
// reading and of the four arrays written.
template <class Ty>
__global__ __launch_bounds__(kT) void k_ns_enter(Job<Ty> j, Mats<typename StoreOf<typename Ty::C>::T> w, int norm_parts) {
    using C = typename Ty::C;
    __shared__ double sh[kWaves];
    __shared__ C tile[kTile][kTile + 1];
    const int b = blockIdx.z;
    const size_t off = b * w.stride;
    const double* part = (const double*)((char*)w.part + off);
    const double squares = block_sum((int)threadIdx.x < norm_parts ? part[threadIdx.x] : 0.0, sh), norm = size_of_matrix(squares, j.eps);
    const bool one = blockIdx.x == 0 && blockIdx.y == 0;      // of the matrix's workgroups
    if (one && threadIdx.x < kMaxCount) ((unsigned*)((char*)w.count + off))[threadIdx.x] = 0;
    double by = norm;
    if constexpr (sizeof(C) == 4) {
        const double root = sqrt(squares);
        int first = 0;
        if (root < j.eps) {                                   // (else |X| is 1 / 2 or more)
            first = lift_of((float)(root / norm));
            by = ldexp(norm, -first);
        }
        if (one && threadIdx.x == 0) {
            float size = (float)(root / norm);                // |X|, NaN with the norm
            int* lift = (int*)((char*)w.lift + off);
            lift[0] = first;
            for (int s = 1; s <= j.steps; ++s) {              // (a singular value grows by |a + b y + c y^2| at most, and to 4)
                const float y = size * size;
                size = fminf(4.f, 1.01f * size * (fabsf(j.ka) + y * (fabsf(j.kb) + y * fabsf(j.kc))));
                lift[s] = s < j.steps ? lift_of(size) : 0;
            }
        }
    }
    // rows and columns of the caller's matrix
    const int64_t r0 = (int64_t)(j.turned ? blockIdx.x : blockIdx.y) * kTile, c0 = (int64_t)(j.turned ? blockIdx.y : blockIdx.x) * kTile;
    constexpr int U = kTile * kTile / kT;
    C v[U];
    j.template enter<false, U>(b, v, [&](int u, int& row, int& col) {
        const int e = threadIdx.x + u * kT;
        row = (int)r0 + e / kTile;
        col = (int)c0 + e % kTile;
        return row < j.rows && col < j.cols;
    });
#pragma unroll
    for (int u = 0; u < U; ++u) tile[(threadIdx.x + u * kT) / kTile][threadIdx.x % kTile] = (C)((double)v[u] / by);
    __syncthreads();
    const auto xm = w.x[0].at(off), xt = w.xt[0].at(off);
    const size_t x0 = (size_t)blockIdx.y * kTile, y0 = (size_t)blockIdx.x * kTile;   // row and column of X
    // a lane's 16 neighbours of a row of X, and of X^T
    const int y = threadIdx.x >> 2, x = (threadIdx.x & 3) * 16;
    C p[16], q[16];
#pragma unroll
    for (int n = 0; n < 16; ++n) {
        p[n] = j.turned ? tile[x + n][y] : tile[y][x + n];
        q[n] = j.turned ? tile[y][x + n] : tile[x + n][y];
    }
    xm.template put<16>((x0 + y) * w.cp + y0 + x, p, kSX);
    xt.template put<16>((y0 + y) * w.rp + x0 + x, q, kSX);
}

enum Kind { kGram, kPoly, kUpdate, kLast };

// 16 bytes of global memory straight to LDS, lane l's to base + 16 l (base: the same for the wave)
__device__ __forceinline__ void copy_to_lds(const void* from, void* base) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)base, 16, 0, 0);
}

// waits until at most N of the wave's copies are under way and its reads of shared memory are done, then for the other waves
template <int N>
__device__ __forceinline__ void wait_and_meet() {
    static_assert(N < 64);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// D[i][j] = sum_k P[i][k] Q[j][k] of one T x T tile.  WI x WJ waves lie over the tile, KG times: group g of the waves takes
// every KG-th piece of the summed index of a stage, so that small tiles still have two or more waves a SIMD to hide the
// way from shared memory; the groups' sums are added at the end.
// A stage holds BK values of T rows of each array; a row is Q pieces of 16 bytes, whose order in the row is turned by
// swz(row), so that the 8 or 16 rows that a part of a wave reads at once lie in different banks.
template <class C, int T> struct Shape;
// Stages in flight: a stage's way from memory takes about 0.5 us, longer than tiles of 32 and 64 compute on it, so three are
// under way while one is read (with two 1000 x 777 takes 213 us, with four 174);  larger tiles compute longer than that on one,
// and do better with fewer, longer stages (2048 x 2048: 781 us with two of 64, 822 with four of 32).
template <> struct Shape<float, 32> { static constexpr int WI = 1, WJ = 1, KG = 4, BK = 64, S = 4; };
template <> struct Shape<float, 64> { static constexpr int WI = 2, WJ = 2, KG = 4, BK = 64, S = 4; };
template <> struct Shape<float, 128> { static constexpr int WI = 2, WJ = 2, KG = 2, BK = 64, S = 2; };
template <> struct Shape<float, 256> { static constexpr int WI = 2, WJ = 4, KG = 1, BK = 32, S = 2; };
// 64 bits: several workgroups a CU hide each other's barriers and ends (8 x 1024 x 1024 3620 us = 47 TFLOP/s, with four shorter
// stages 3820; 1000 x 1000 823 | 996).  Tiles of 32 read twice as much for a product, but the last round is fuller and fewer
// of its rows are padding (1000 x 1000 717 us; 29 x 276 x 160 270 | 370; 8 x 1024 x 1024 4070).
template <> struct Shape<double, 64> { static constexpr int WI = 2, WJ = 2, KG = 2, BK = 32, S = 2; };
template <> struct Shape<double, 32> { static constexpr int WI = 1, WJ = 1, KG = 4, BK = 32, S = 2; };

template <class C> struct Frag;   // what a wave reads of one 32-row (16 for 64 bits) block at once, and its products
template <> struct Frag<float> {
    using M = Pair;
    using Acc = float16v;
    static constexpr int kSide = 32, kRegs = 16;
    static __device__ __forceinline__ int row(int lane, int q) { return 8 * (q >> 2) + 4 * (lane >> 5) + (q & 3); }
};
template <> struct Frag<double> {
    using M = Wide;
    using Acc = double4v;
    static constexpr int kSide = 16, kRegs = 4;
    static __device__ __forceinline__ int row(int lane, int q) { return Mma<double>::row(lane, q); }
};

// All parts of a value are multiplied, also where the result has 16 bits: without the low parts of X (11 bits) a bfloat16 result
// of 4096 x 4096 is off by 1.0e-3 of its norm before it is rounded, with them by 1e-6.
template <class C, int T>
struct Tile : Shape<C, T> {
    using Sh = Shape<C, T>;
    using Fr = Frag<C>;
    using M = typename Fr::M;
    static constexpr int WI = Sh::WI, WJ = Sh::WJ, KG = Sh::KG, BK = Sh::BK;
    static constexpr int NP = sizeof(C) == 4 ? 2 : 1, NQ = NP;         // parts of a value (16-bit pairs: 2)
    static constexpr int kArrays = NP + NQ, S = Sh::S;
    static constexpr int kWv = WI * WJ * KG, kThreads = 64 * kWv;
    static constexpr int kSize = sizeof(C) == 8 ? 8 : 2;              // of a stored value
    static constexpr int Q = BK * kSize / 16;                         // pieces of a row
    static constexpr int kArray = T * Q * 16, kStage = kArrays * kArray;   // bytes
    static constexpr int kCopies = kStage / 1024 / kWv;               // a wave's copies (1 KB each) of a stage
    static constexpr int NI = T / WI / Fr::kSide, NJ = T / WJ / Fr::kSide;     // blocks of a wave
    static constexpr int BI = T / WI / 32, BJ = T / WJ / 32;          // its 32 x 32 blocks as they leave
    static constexpr int kBlock = 32 * 33;
    static constexpr size_t kOut = (size_t)kWv * BJ * kBlock * sizeof(C);
    static constexpr size_t kBytes = (size_t)S * kStage > kOut ? (size_t)S * kStage : kOut;
    static constexpr int N = 16 / KG;                                 // neighbours of a block's row that a lane takes
    static_assert(kStage % (1024 * kWv) == 0 && (Q == 4 || Q == 8 || Q == 16) && kBytes <= 160 * 1024);

    typename Fr::Acc acc[NI][NJ];

    static __device__ __forceinline__ int swz(int row) {
        return Q == 16 ? row & 15 : Q == 4 ? (((row >> 1) ^ (row >> 3)) & 1) | ((row >> 2) & 1) << 1 : ((row ^ (row >> 3)) & 1) | (row & 6);
    }
    static __device__ __forceinline__ int wave() { return threadIdx.x >> 6; }
    static __device__ __forceinline__ int group() { return wave() / (WI * WJ); }
    static __device__ __forceinline__ int wave_i() { return wave() % (WI * WJ) / WJ * (T / WI); }
    static __device__ __forceinline__ int wave_j() { return wave() % WJ * (T / WJ); }

    static __device__ __forceinline__ const char* base(const Pair& p, const Pair& q, int arr) {
        return (const char*)(arr < NP ? arr == 0 ? p.hi : p.lo : arr == NP ? q.hi : q.lo);
    }
    static __device__ __forceinline__ const char* base(const Wide& p, const Wide& q, int arr) { return (const char*)(arr ? q.v : p.v); }

    // where the wave's copies of a stage come from (a lane's 16 bytes, at the first stage) and go to
    struct Copies {
        const char* from[kCopies];
        int to[kCopies];
    };
    __device__ __forceinline__ void aim(const M& p, const M& q, size_t i0, size_t j0, int ld, int k0, Copies& c) {
        const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(wave());
        constexpr int kRows = 64 / Q, kChunks = T / kRows;            // rows of a copy, copies of an array
#pragma unroll
        for (int n = 0; n < kCopies; ++n) {
            const int id = n * kWv + w, arr = id / kChunks, r0 = id % kChunks * kRows, row = r0 + lane / Q;
            c.from[n] = base(p, q, arr) + ((arr >= NP ? j0 : i0) + row) * (size_t)ld * kSize + (size_t)k0 * kSize + ((lane % Q) ^ swz(row)) * 16;
            c.to[n] = arr * kArray + r0 * Q * 16;
        }
    }
    __device__ __forceinline__ void fetch(const Copies& c, int t, char* st) {
#pragma unroll
        for (int n = 0; n < kCopies; ++n) copy_to_lds(c.from[n] + (size_t)t * (BK * kSize), st + c.to[n]);
    }

    // the products of one piece pair of the summed index
    __device__ __forceinline__ void multiply(const char* st, int kk) {
        const int lane = threadIdx.x & 63;
        if constexpr (sizeof(C) == 4) {
            const int piece = 2 * kk + (lane >> 5);
            half8v pv[NI][NP], qv[NJ][NQ];
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int r = wave_j() + 32 * j + (lane & 31);
#pragma unroll
                for (int x = 0; x < NQ; ++x) qv[j][x] = *(const half8v*)(st + (r * Q + (piece ^ swz(r))) * 16 + (NP + x) * kArray);
            }
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int r = wave_i() + 32 * i + (lane & 31);
#pragma unroll
                for (int x = 0; x < NP; ++x) pv[i][x] = *(const half8v*)(st + (r * Q + (piece ^ swz(r))) * 16 + x * kArray);
            }
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                auto go = [&](int x, int y) {
#pragma unroll
                    for (int j = 0; j < NJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(pv[i][x], qv[j][y], acc[i][j], 0, 0, 0);
                };
                go(1, 0);     // lo hi
                go(0, 1);     // hi lo
                go(0, 0);     // hi hi
            }
        } else {
            // a lane's piece holds two neighbours of the summed index; the first ones of the four pieces make one matrix
            // instruction, the second ones another (the order of a sum's terms is free, as long as P's and Q's agree)
            const int piece = 4 * kk + (lane >> 4);
            double2 pv[NI], qv[NJ];
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int r = wave_j() + 16 * j + (lane & 15);
                qv[j] = *(const double2*)(st + kArray + (r * Q + (piece ^ swz(r))) * 16);
            }
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int r = wave_i() + 16 * i + (lane & 15);
                pv[i] = *(const double2*)(st + (r * Q + (piece ^ swz(r))) * 16);
            }
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < NJ; ++j) acc[i][j] = Mma<double>::go(pv[i].x, qv[j].x, acc[i][j]);
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < NJ; ++j) acc[i][j] = Mma<double>::go(pv[i].y, qv[j].y, acc[i][j]);
        }
    }

    // summed over k0 .. k0 + K, K a multiple of BK
    __device__ __forceinline__ void run(const M& p, const M& q, size_t i0, size_t j0, int ld, int k0, int K, char* lds) {
        constexpr int kSteps = Q / (sizeof(C) == 4 ? 2 : 4);
        static_assert(kSteps % KG == 0);
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int r = 0; r < Fr::kRegs; ++r) acc[i][j][r] = 0;
        const int n = K / BK;
        Copies c;
        aim(p, q, i0, j0, ld, k0, c);
#pragma unroll
        for (int t = 0; t < S - 1; ++t)
            if (t < n) fetch(c, t, lds + t * kStage);
        for (int t = 0; t < n; ++t) {
            // Stage t has arrived: each wave waits for its own copies (those of the later stages may be under way), the
            // barrier for the waves'.  The wave has also read what it needs of stage t - 1, which the next copies replace.
            if (t + S - 1 <= n) wait_and_meet<kCopies * (S - 2)>();
            else wait_and_meet<0>();
            if (t + S - 1 < n) fetch(c, t + S - 1, lds + (t + S - 1) % S * kStage);
            const char* st = lds + t % S * kStage;
#pragma unroll
            for (int kk = 0; kk < kSteps / KG; ++kk) multiply(st, kk * KG + group());
        }
        __syncthreads();   // the stages are read: the shared memory takes the result
    }

    // The result, a row of 32 x 32 blocks of each wave at a time, through shared memory:  first(y, x, raw, v) gets N
    // neighbours D[y][x ..] and may change them, second(y, x, v) then N neighbours D[y ..][x] of the changed result.
    // raw: what load(y, x) fetched for them while the blocks before were on their way.
    template <class L, class F, class G>
    __device__ __forceinline__ void leave(char* lds, L load, F first, G second) {
        const int lane = threadIdx.x & 63, w = wave() % (WI * WJ), at = group() * 64 + lane, line = at / (2 * KG), seg = at % (2 * KG) * N;
        auto blk = [&](int g, int j) { return (C(*)[33])lds + ((g * WI * WJ + w) * BJ + j) * 32; };
        auto meet = [] { if (KG > 1) __syncthreads(); else wave_fence(); };
        constexpr int kPer = 32 / Fr::kSide;
        using Raw = decltype(load(0, 0));
        Raw raw[BJ];
#pragma unroll
        for (int j = 0; j < BJ; ++j) raw[j] = load(wave_i() + line, wave_j() + 32 * j + seg);
#pragma unroll
        for (int i = 0; i < BI; ++i) {
            Raw next[BJ];
#pragma unroll
            for (int j = 0; j < BJ; ++j)
                if (i + 1 < BI) next[j] = load(wave_i() + 32 * (i + 1) + line, wave_j() + 32 * j + seg);
#pragma unroll
            for (int j = 0; j < BJ; ++j) {
                auto mine = blk(group(), j);
#pragma unroll
                for (int a = 0; a < kPer; ++a)
#pragma unroll
                    for (int b = 0; b < kPer; ++b)
#pragma unroll
                        for (int q = 0; q < Fr::kRegs; ++q)
                            mine[a * Fr::kSide + Fr::row(lane, q)][b * Fr::kSide + lane % Fr::kSide] = acc[i * kPer + a][j * kPer + b][q];
            }
            meet();
#pragma unroll
            for (int j = 0; j < BJ; ++j) {
                C v[N];
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    v[n] = blk(0, j)[line][seg + n];
#pragma unroll
                    for (int g = 1; g < KG; ++g) v[n] += blk(g, j)[line][seg + n];
                }
                first(wave_i() + 32 * i + line, wave_j() + 32 * j + seg, raw[j], v);
#pragma unroll
                for (int n = 0; n < N; ++n) blk(0, j)[line][seg + n] = v[n];
            }
            meet();
#pragma unroll
            for (int j = 0; j < BJ; ++j) {
                C v[N];
#pragma unroll
                for (int n = 0; n < N; ++n) v[n] = blk(0, j)[seg + n][line];
                second(wave_i() + 32 * i + seg, wave_j() + 32 * j + line, v);
            }
#pragma unroll
            for (int j = 0; j < BJ; ++j)
                if (i + 1 < BI) raw[j] = next[j];
            meet();
        }
    }
};

// Values that workgroups on other XCDs read while this kernel runs: the loads and stores go past the XCD's own L2.
template <int N, class C>
__device__ __forceinline__ void give(C* to, const C* v) {
    static_assert(N * sizeof(C) % 8 == 0);
#pragma unroll
    for (int n = 0; n < (int)(N * sizeof(C) / 8); ++n) {
        uint64_t u;
        __builtin_memcpy(&u, (const char*)v + 8 * n, 8);
        __hip_atomic_store((uint64_t*)to + n, u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}
template <int N, class C>
__device__ __forceinline__ void take(C* from, C* v) {
    uint64_t u[N * sizeof(C) / 8];
    C x[N];
#pragma unroll
    for (int n = 0; n < (int)(N * sizeof(C) / 8); ++n) u[n] = __hip_atomic_load((uint64_t*)from + n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __builtin_memcpy(x, u, sizeof(x));
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] += x[n];
}
// Whether this workgroup is the last of n to come here with what it gave.  Each wave waits for its stores to be where all XCDs
// see them, so that the count needs no fence: a fence writes the whole L2 back, 30 us with 200 workgroups at it.  The language's
// memory model orders relaxed atomics of different addresses in no way; that the wait does is this hardware's: stores of agent
// scope go past the L2 and are counted until they are there, loads of agent scope read past it, and both stay in program order
// around the wait and the barriers (volatile assembly with a memory clobber, __syncthreads).
__device__ __forceinline__ bool last_to_arrive(unsigned* count, int n, unsigned* sh) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        const unsigned before = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (before == (unsigned)n - 1) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *sh = before;
    }
    __syncthreads();
    const unsigned before = *sh;
    __syncthreads();
    return before == (unsigned)n - 1;
}

// One product of a step.  kGram: A = X X^T;  kPoly: B = b A + c A A  (lower tiles, written to both sides of the
// diagonal);  kUpdate: X <- a X + B X as its transpose X^T B, both layouts written;  kLast: the same to the caller.
// Time of X X^T | b A + c A A | update, us:  4096 x 4096 280 | 287 | 390 (of 16- and 32-bit matrices alike; the last update of 16
// bits keeps 8 registers of a thread in scratch): the symmetric products are 528 tiles of 128 in 3 rounds of 256, the third nearly
// empty;  2048 x 2048 float32  54 | 57 | 65;  1000 x 777  10 | 8 | 12 (with tiles of 64 12 | 10 | 12): bound by the 3 to 5 us that a
// launch, the way of the first stage, the epilogue and the last stores take;  1024 x 4096  31 | 11 | 40: 136 tiles for 256
// CUs, and an update that writes 34 MB in one round, after its products.
template <class Ty, Kind kind, int T>
__global__ __launch_bounds__((Tile<typename Ty::C, T>::kThreads)) void k_ns_product(Job<Ty> j, Mats<typename StoreOf<typename Ty::C>::T> w, int step) {
    using C = typename Ty::C;
    const int from = step & 1;
    constexpr bool kSym = kind == kGram || kind == kPoly;
    extern __shared__ __attribute__((aligned(16))) char product_lds[];
    const size_t off = blockIdx.z * w.stride;
    size_t ti = blockIdx.y, tj = blockIdx.x;
    const int splits = kind == kGram && T <= 64 ? w.splits : 1, tile_id = blockIdx.x / splits, split = blockIdx.x - tile_id * splits;
    if (kSym) {
        ti = (size_t)((sqrtf(8.f * tile_id + 1.f) - 1.f) * 0.5f);
        while (ti * (ti + 1) / 2 > (size_t)tile_id) --ti;
        while ((ti + 1) * (ti + 2) / 2 <= (size_t)tile_id) ++ti;
        tj = tile_id - ti * (ti + 1) / 2;
    }
    const size_t i0 = ti * T, j0 = tj * T;
    const auto a = w.a.at(off), bm = w.b.at(off);
    using Tl = Tile<C, T>;
    Tl t;
    constexpr int N = Tl::N;
    int lift = 0, next = 0;
    if constexpr (sizeof(C) == 4 && kind != kGram) {
        const int* of = (const int*)((const char*)w.lift + off) + step;
        lift = of[0];
        next = of[1];
    }
    const C square = sizeof(C) == 4 ? (C)ldexpf(1.f, -2 * lift) : C(1);     // (0 where b A + c A A is nothing beside a)
    if (kind == kGram || kind == kPoly) {
        const auto m = (kind == kGram ? w.x[from] : w.a).at(off), out = kind == kGram ? a : bm;
        const float so = kind == kGram ? kSA : kSB;
        const C f = sizeof(C) == 8 ? C(1) : kind == kGram ? C(1.f / (kSX * kSX)) : C(1.f / (kSA * kSA)) * square;
        if constexpr (kind == kGram && T <= 64) {
            if (w.splits > 1) {
                const int per = ((w.ck + 63) / 64 + w.splits - 1) / w.splits * 64, k0 = split * per;
                t.run(m, m, i0, j0, w.cp, k0, min(per, w.ck - k0), product_lds);
                C* sum = (C*)((char*)w.sum + off) + (size_t)tile_id * w.splits * (T * T);
                t.leave(product_lds, [](int, int) { return 0; },
                    [&](int y, int x, int, C* v) { give<N>(sum + (size_t)split * (T * T) + y * T + x, v); },
                    [](int, int, const C*) {});
                if (!last_to_arrive((unsigned*)((char*)w.count + off) + tile_id, w.splits, (unsigned*)product_lds)) return;
                // The last part to arrive adds all of them, in their order.  (No part waits for another.)
                struct Sum { C v[N]; };
                t.leave(product_lds,
                    [&](int y, int x) {
                        Sum all;
#pragma unroll
                        for (int n = 0; n < N; ++n) all.v[n] = C(0);
                        for (int q = 0; q < w.splits; ++q) take<N>(sum + (size_t)q * (T * T) + y * T + x, all.v);
                        return all;
                    },
                    [&](int y, int x, const Sum& all, C* v) {
#pragma unroll
                        for (int n = 0; n < N; ++n) v[n] = f * all.v[n];
                        out.template put<N>((i0 + y) * w.rp + j0 + x, v, so);
                    },
                    [&](int y, int x, const C* v) {
                        if (ti != tj) out.template put<N>((j0 + x) * w.rp + i0 + y, v, so);
                    });
                return;
            }
        }
        t.run(m, m, i0, j0, kind == kGram ? w.cp : w.rp, 0, kind == kGram ? w.ck : w.rk, product_lds);
        t.leave(product_lds,
            [&](int y, int x) {
                if constexpr (kind == kPoly) return a.template get<N>((i0 + y) * w.rp + j0 + x);
                else return 0;
            },
            [&](int y, int x, const auto& raw, C* v) {
                const size_t at = (i0 + y) * w.rp + j0 + x;
                if constexpr (kind == kPoly) {
                    C av[N];
                    raw.values(kSA, av);
#pragma unroll
                    for (int n = 0; n < N; ++n) v[n] = j.kb * av[n] + j.kc * (f * v[n]);
                } else {
#pragma unroll
                    for (int n = 0; n < N; ++n) v[n] *= f;
                }
                out.template put<N>(at, v, so);
            },
            [&](int y, int x, const C* v) {
                if (ti != tj) out.template put<N>((j0 + x) * w.rp + i0 + y, v, so);
            });
    } else {
        const auto xt = w.xt[from].at(off), nx = w.x[from ^ 1].at(off), nt = w.xt[from ^ 1].at(off);
        t.run(xt, bm, i0, j0, w.rp, 0, w.rk, product_lds);   // rows: columns of X; columns: rows of X
        const C f = sizeof(C) == 8 ? C(1) : C(1.f / (kSX * kSB)) * square, grow = sizeof(C) == 4 ? (C)ldexpf(1.f, next - lift) : C(1);
        t.leave(product_lds,
            [&](int y, int x) { return xt.template get<N>((i0 + y) * w.rp + j0 + x); },
            [&](int y, int x, const auto& raw, C* v) {
                const size_t at = (i0 + y) * w.rp + j0 + x;
                C xv[N];
                raw.values(kSX, xv);
#pragma unroll
                for (int n = 0; n < N; ++n) v[n] = (j.ka * xv[n] + f * v[n]) * grow;
                if (kind == kUpdate) nt.template put<N>(at, v, kSX);
                else if (j.turned)
                    j.template leave_run<N>(blockIdx.z, v, (int)i0 + y, (int)j0 + x);
            },
            [&](int y, int x, const C* v) {
                if (kind == kUpdate) nx.template put<N>((j0 + x) * w.cp + i0 + y, v, kSX);
                else if (!j.turned)
                    j.template leave_run<N>(blockIdx.z, v, (int)j0 + x, (int)i0 + y);
            });
    }
}

// ---- launches -------------------------------------------------------------------------------------------------------
constexpr size_t kLds = 160 * 1024;

// Which form carries a matrix.  Measured, us, long | strip or block (batch x r x c):  32 bits  1 x 11 x 512  17 | 18,  256 x 16 x
// 512  23 | 21,  1 x 16 x 4096  18 | 73,  1 x 32 x 512  25 | 39,  1 x 64 x 256  61 | 57,  256 x 48 x 256  56 | 44;  64 bits, where
// the long form takes three launches a step,  1 x 16 x 1024  51 | 35,  1 x 11 x 2048  52 | 64,  256 x 11 x
// 2048  189 | 79,  1 x 64 x 128  115 | 72.
// Against the tiles of 64 x 64:  256 x 17 x 2048 of 32 bits  79 | 2710,  1 x 64 x 4096  66 | 110.
enum Form { kTiled, kStrip, kBlock, kLong };
Form form_of(int dtype, int batch, int r, int c) {
    const size_t size = dtype == VQA_DTYPE_F64 ? 8 : 4;
    if (r > 64) return kTiled;
    if (size == 4 && c >= 512) return kLong;
    if (r <= 16) return c <= (batch > 32 ? 2048 : 1024) ? kStrip : kLong;   // (2048: the registers of 16 waves)
    return (r <= 32 ? Block<2>::bytes(c, size) : r <= 48 ? Block<3>::bytes(c, size) : Block<4>::bytes(c, size)) <= kLds ? kBlock : kLong;
}
// Parts of the columns: enough workgroups for the chip, each with 256 columns or more
LongWs long_ws(char* base, int batch, int r, int c) {
    LongWs w;
    const size_t nt = (r + 15) / 16, tile = 256;
    w.parts = std::max(1, std::min({ kMaxParts, (c + 255) / 256, (1024 + batch - 1) / std::max(batch, 1) }));
    w.part = (double*)base;
    w.poly = w.part + w.parts * (nt * (nt + 1) / 2) * tile;
    w.x = w.poly + nt * nt * tile;
    w.stride = (w.parts * (nt * (nt + 1) / 2) * tile + nt * nt * tile + (size_t)c * nt * 16) * 8;
    return w;
}
// How the products are cut: sides of the tiles of X X^T, of b A + c A A and of the update, and into how many parts the sum of
// X X^T is split.
struct Cut { int gram, poly, up, splits; };
struct Side { int side, splits; };

// The tile and the parts whose rounds of 256 workgroups (one a CU) take least.  In us: what a round takes at its ends, and for
// a summed index of 64 with the chip filled.  Of tiles of 32 a CU holds several workgroups, so the last round's share counts.
// Measured for the tile so chosen | the next best, us a product of 32 bits:
//   update      of 4096 x 4096  420 (256) | 504 (128)    of 2048 x 2048  62 (128) | 85 (64)    of 1024 x 4096  37 (128) | 46 (64)
//   b A + c A A of 3000         148 (128) | 230 (256)    of 2048          53 (128) | 58 (64)    of 1024         12 (64) | 26 (128)
// (Of 4096 the symmetric products' 528 tiles of 128, paid as 3 rounds, and 136 of 256 come out alike here, 303.0 and 303.7; measured,
// the whole operator takes 4780 | 4950, so the choice that the sums make by little is the right one.)
// and the whole operator with tiles of 32 | 64:  512 x 512  92 | 133,  300 x 300  77 | 105,  1000 x 1000  233 | 196.
// (Tiles of 192 take 288 us for A A of 4096 by itself, those of 256 331, but the whole operator then takes 3% longer.)
// A split sum (few tiles and a long sum: X X^T of a wide matrix) also takes the giving and taking of its parts, 4.5 us and 0.35
// a part.  Whole operator, split | not, tiles of 64:  100 x 4000  123 us (8 parts) | 218;  512 x 4096  231 (3) | 306.  Tiles of
// 128 lose what splitting gains to that (1024 x 4096: 588 us with 5 parts, 449 with tiles of 64 unsplit).
struct Round { int side; double ends, sum; };
constexpr Round kRounds32[] = { { 256, 8, 4.62 }, { 128, 5, 1.5 }, { 64, 5, 0.45 }, { 32, 3, 0.33 } }, kRounds64[] = { { 64, 5, 2.1 }, { 32, 1.5, 0.68 } };
template <int N>
Side side_of(const Round (&rounds)[N], int64_t batch, int rows, int cols, int sum, bool symmetric, bool split) {
    Side best = { 64, 1 };
    double least = 1e30;
    for (const Round& k : rounds) {
        const int64_t a = (rows + k.side - 1) / k.side, b = (cols + k.side - 1) / k.side, n = (symmetric ? a * (a + 1) / 2 : a * b) * batch;
        const int stages = (sum + 63) / 64, most = split && k.side <= 64 ? (int)std::min<int64_t>(256 / n, stages / 4) : 1;
        for (int p = 1; p <= std::max(1, most); ++p) {
            const int per = (stages + p - 1) / p;
            if ((stages + per - 1) / per != p) continue;   // (the last parts would be empty)
            const double full = k.side == 32 ? std::max(1.0, (double)(n * p) / 256) : (double)((n * p + 255) / 256);
            const double us = full * (k.ends + per * k.sum) + (p > 1 ? 4.5 + p * 0.35 : 0);
            if (us < least) { least = us; best = { k.side, p }; }
        }
    }
    return best;
}
int pad_to(int v, int t) { return (v + t - 1) / t * t; }
template <int N>
Cut cut_of(const Round (&rounds)[N], int batch, int r, int c) {
    const Side x = side_of(rounds, batch, r, r, c, true, true);
    return { x.side, side_of(rounds, batch, r, r, r, true, false).side, side_of(rounds, batch, c, r, r, false, false).side, x.splits };
}
// whole stages, of which a tile's summed index is made up: what is summed over, and what tiles cover at the least
int least_pad(int dtype) { return dtype == VQA_DTYPE_F64 ? 32 : 64; }
Cut cut_of(int dtype, int batch, int r, int c) {
    r = pad_to(r, least_pad(dtype));
    c = pad_to(c, least_pad(dtype));
    return dtype == VQA_DTYPE_F64 ? cut_of(kRounds64, batch, r, c) : cut_of(kRounds32, batch, r, c);
}
size_t up256(size_t v) { return (v + 255) / 256 * 256; }

size_t sum_bytes(int rk, Cut t, size_t size) {
    const size_t a = (rk + t.gram - 1) / t.gram;
    return a * (a + 1) / 2 * t.splits * t.gram * t.gram * size;
}
template <class M>
void extents(int r, int c, Cut t, Mats<M>* w) {
    const int least = least_pad(std::is_same_v<M, Wide> ? VQA_DTYPE_F64 : VQA_DTYPE_F32);
    w->rk = pad_to(r, least);
    w->ck = pad_to(c, least);
    w->rp = pad_to(std::max({ pad_to(r, t.gram), pad_to(r, t.poly), pad_to(r, t.up) }), kTile);
    w->cp = pad_to(pad_to(c, t.up), kTile);
}

template <class M>
size_t lay_out(char* base, int r, int c, Cut t, Mats<M>* w);
template <>
size_t lay_out<Pair>(char* base, int r, int c, Cut t, Mats<Pair>* w) {
    extents(r, c, t, w);
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
    w->count = (unsigned*)p;
    p += kMaxCount * 4;
    w->lift = (int*)p;
    p += up256((kMostSteps + 1) * 4);
    w->sum = p;
    w->splits = t.splits;
    if (t.splits > 1) p += sum_bytes(w->rk, t, 4);
    return w->stride = (size_t)(p - base);
}
template <>
size_t lay_out<Wide>(char* base, int r, int c, Cut t, Mats<Wide>* w) {
    extents(r, c, t, w);
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
    w->count = (unsigned*)p;
    p += kMaxCount * 4;
    w->lift = nullptr;
    w->sum = p;
    w->splits = t.splits;
    if (t.splits > 1) p += sum_bytes(w->rk, t, 8);
    return w->stride = (size_t)(p - base);
}

// Dynamic shared memory beyond 64 KB is asked for once for each kernel and device
template <auto kKernel>
int allow_lds(size_t bytes) {
    static std::atomic<uint64_t> done{ 0 };   // a bit a device; asking twice does no harm
    int dev = 0;
    VQA_HIP(hipGetDevice(&dev));
    if (bytes > 65536 && !(done >> (dev & 63) & 1)) {
        VQA_HIP(hipFuncSetAttribute((const void*)kKernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)kLds));
        done |= (uint64_t)1 << (dev & 63);
    }
    return VQA_OK;
}

template <class Ty, int NT>
int long_rows(hipStream_t st, const Job<Ty>& j, const LongWs& w) {
    if (int rc = allow_lds<k_ns_poly<NT>>(Long<NT>::kBytes)) return rc;
    int round = 1;
    if (sizeof(typename Ty::C) == 4)
        for (double a = fabs((double)j.ka), p = a * a; round < j.steps && p <= 8192.0; p *= a) ++round;
    const dim3 parts(w.parts, (unsigned)j.batch), one((unsigned)j.batch), wide((unsigned)std::max(1, std::min((j.c + 63) / 64, 2048 / j.batch)), (unsigned)j.batch);
    for (int s = 0; s < j.steps; s += round) {
        const bool first = s == 0, last = s + round >= j.steps;
        if (first) hipLaunchKernelGGL((k_ns_gram<Ty, NT, true>), parts, dim3(kT), 0, st, j, w);
        else hipLaunchKernelGGL((k_ns_gram<Ty, NT, false>), parts, dim3(kT), 0, st, j, w);
        hipLaunchKernelGGL((k_ns_poly<NT>), one, dim3(64 * Long<NT>::kTiles), Long<NT>::kBytes, st, w, j.r, std::min(round, j.steps - s),
                           (double)j.ka, (double)j.kb, (double)j.kc, j.eps, first);
        if (first && last) hipLaunchKernelGGL((k_ns_apply<Ty, NT, true, true>), wide, dim3(kT), 0, st, j, w);
        else if (first) hipLaunchKernelGGL((k_ns_apply<Ty, NT, true, false>), wide, dim3(kT), 0, st, j, w);
        else if (last) hipLaunchKernelGGL((k_ns_apply<Ty, NT, false, true>), wide, dim3(kT), 0, st, j, w);
        else hipLaunchKernelGGL((k_ns_apply<Ty, NT, false, false>), wide, dim3(kT), 0, st, j, w);
    }
    VQA_HIP(hipGetLastError());
    return VQA_OK;
}

template <class Ty, int NT>
int block(hipStream_t st, const Job<Ty>& j) {
    const size_t lds = Block<NT>::bytes(j.c, sizeof(typename Ty::C));
    if (int rc = (allow_lds<k_ns_block<Ty, NT>>(lds))) return rc;
    hipLaunchKernelGGL((k_ns_block<Ty, NT>), dim3((unsigned)j.batch), dim3(kBlockThreads), lds, st, j);
    return VQA_OK;
}

template <class Ty, Kind kind, int T>
int product(hipStream_t st, dim3 grid, const Job<Ty>& j, const Mats<typename StoreOf<typename Ty::C>::T>& w, int step) {
    using Tl = Tile<typename Ty::C, T>;
    if (int rc = allow_lds<k_ns_product<Ty, kind, T>>(Tl::kBytes)) return rc;
    hipLaunchKernelGGL((k_ns_product<Ty, kind, T>), grid, dim3(Tl::kThreads), Tl::kBytes, st, j, w, step);
    return VQA_OK;
}

template <class Ty, Kind kind>
int product(hipStream_t st, int tile, const Job<Ty>& j, const Mats<typename StoreOf<typename Ty::C>::T>& w, int step) {
    const unsigned tr = (w.rk + tile - 1) / tile, tc = (w.ck + tile - 1) / tile;   // (all that is summed over is written)
    const dim3 grid = kind == kGram || kind == kPoly ? dim3(tr * (tr + 1) / 2 * (kind == kGram ? w.splits : 1), 1, (unsigned)j.batch) : dim3(tr, tc, (unsigned)j.batch);
    if constexpr (sizeof(typename Ty::C) == 4) {
        if (tile == 256) return product<Ty, kind, 256>(st, grid, j, w, step);
        if (tile == 128) return product<Ty, kind, 128>(st, grid, j, w, step);
    }
    if (tile == 32) return product<Ty, kind, 32>(st, grid, j, w, step);
    if (tile != 64) VQA_FAIL(VQA_EINVAL, "no tile of %d", tile);
    return product<Ty, kind, 64>(st, grid, j, w, step);
}

template <class Ty>
int steps(hipStream_t st, const Job<Ty>& j, const Mats<typename StoreOf<typename Ty::C>::T>& w, Cut t) {
    int rc = VQA_OK;
    for (int s = 0; s < j.steps && !rc; ++s) {
        rc = product<Ty, kGram>(st, t.gram, j, w, s);
        if (!rc) rc = product<Ty, kPoly>(st, t.poly, j, w, s);
        if (!rc) rc = s + 1 < j.steps ? product<Ty, kUpdate>(st, t.up, j, w, s) : product<Ty, kLast>(st, t.up, j, w, s);
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
    const Form form = form_of(q.dtype, q.batch, j.r, j.c);
    if (form == kLong) {
        const LongWs w = long_ws((char*)q.workspace, q.batch, j.r, j.c);
        return j.r <= 16 ? long_rows<Ty, 1>(st, j, w) : j.r <= 32 ? long_rows<Ty, 2>(st, j, w) : j.r <= 48 ? long_rows<Ty, 3>(st, j, w) : long_rows<Ty, 4>(st, j, w);
    }
    if (form == kStrip) {
        const int strips = (j.c + 15) / 16;
        const dim3 grid((unsigned)q.batch);
        if (strips <= 4) hipLaunchKernelGGL((k_ns_strip<Ty, 4, 1>), grid, dim3(256), 0, st, j);
        else if (strips <= 16) hipLaunchKernelGGL((k_ns_strip<Ty, 4, 4>), grid, dim3(256), 0, st, j);
        else if (strips <= 64) hipLaunchKernelGGL((k_ns_strip<Ty, 16, 4>), grid, dim3(1024), 0, st, j);
        else if constexpr (sizeof(C) == 8) hipLaunchKernelGGL((k_ns_strip<Ty, 16, 8>), grid, dim3(1024), 0, st, j);
        VQA_HIP(hipGetLastError());
        return VQA_OK;
    }
    if (form == kBlock) {
        const int rc = j.r <= 32 ? block<Ty, 2>(st, j) : j.r <= 48 ? block<Ty, 3>(st, j) : block<Ty, 4>(st, j);
        if (rc) return rc;
        VQA_HIP(hipGetLastError());
        return VQA_OK;
    }
    if (q.steps > kMostSteps) VQA_FAIL(VQA_EINVAL, "more than %d steps", kMostSteps);
    Mats<typename StoreOf<C>::T> w;
    const Cut cut = cut_of(q.dtype, q.batch, j.r, j.c);
    lay_out((char*)q.workspace, j.r, j.c, cut, &w);
    const unsigned nb = (unsigned)q.batch;
    const int pieces = std::max(1, std::min((j.cols + 4 * kT - 1) / (4 * kT), (2 * kNormParts + j.rows - 1) / j.rows));
    const int parts = std::min(kNormParts, j.rows * pieces);
    hipLaunchKernelGGL((k_ns_norm<Ty>), dim3(parts, nb), dim3(kT), 0, st, j, w.part, w.stride, pieces);
    hipLaunchKernelGGL((k_ns_enter<Ty>), dim3(w.cp / kTile, w.rp / kTile, nb), dim3(kT), 0, st, j, w, parts);
    if (const int rc = steps(st, j, w, cut)) return rc;
    VQA_HIP(hipGetLastError());
    return VQA_OK;
}

}  // namespace

bool ortho_in_pairs(int dtype, int rows, int cols) { return dtype != VQA_DTYPE_F64 && std::min(rows, cols) > 64; }

size_t ortho_workspace_bytes(int dtype, int batch, int rows, int cols) {
    const int r = std::min(rows, cols), c = std::max(rows, cols);
    switch (form_of(dtype, batch, r, c)) {
        case kStrip: case kBlock: return 0;
        case kLong: return long_ws(nullptr, batch, r, c).stride * (size_t)batch;
        default: break;
    }
    if (dtype == VQA_DTYPE_F64) {
        Mats<Wide> w;
        return lay_out<Wide>(nullptr, r, c, cut_of(dtype, batch, r, c), &w) * (size_t)batch;
    }
    Mats<Pair> w;
    return lay_out<Pair>(nullptr, r, c, cut_of(dtype, batch, r, c), &w) * (size_t)batch;
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
