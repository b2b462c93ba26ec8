// Softmax read-out of rows of scores: log probabilities of given outcomes, the rows' entropies and most probable
// outcomes, and the gradient of a loss that weighs them.
//
// With x = scale * z and the row's maximum m:  s = sum over the row of exp(x - m), WITHOUT the one term 1 of the first
// element that attains m, and t = sum exp(x - m) (x - m).  Then log p_c = (x_c - m) - log1p(s) and the entropy is
// log1p(s) - t / (1 + s); both keep their relative accuracy for a row whose probability sits in one outcome, where
// log(1 + s) would lose s.  (m, s, t) of two parts of a row join exactly like running maximum and sum of a softmax,
// so a row is read once, by lanes, waves and workgroups that each take a part (Part, join).
// m is kept as the stored score z: (z - m) * scale rounds the small difference and not the large product.
#include <algorithm>
#include <type_traits>

#include "vqa_core.h"

namespace vqa {

namespace {

typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr int kT = 256;
constexpr int kWaves = kT / 64;

// ---- stored types: A is the type of the sums (64 bits for double, else 32) --------------------------------------
struct F64 { using S = double; using A = double; static constexpr bool kFast = false;
    static __device__ A up(S v) { return v; } static __device__ S down(A v) { return v; } };
struct F32 { using S = float; using A = float; static constexpr bool kFast = false;
    static __device__ A up(S v) { return v; } static __device__ S down(A v) { return v; } };
struct F16 { using S = _Float16; using A = float; static constexpr bool kFast = true;
    static __device__ A up(S v) { return (float)v; } static __device__ S down(A v) { return (_Float16)v; } };
struct BF16 { using S = uint16_t; using A = float; static constexpr bool kFast = true;
    static __device__ A up(S v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ S down(A v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }   // to nearest even
    };

__device__ __forceinline__ double neg_inf(double) { return -__builtin_inf(); }
__device__ __forceinline__ float neg_inf(float) { return -__builtin_inff(); }
__device__ __forceinline__ double nan_of(double) { return __builtin_nan(""); }
__device__ __forceinline__ float nan_of(float) { return __builtin_nanf(""); }
__device__ __forceinline__ double max_of(double a, double b) { return fmax(a, b); }
__device__ __forceinline__ float max_of(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double exp_of(double d) { return exp(d); }
// exp(d), d <= 0, as 2^h (1 + l ln 2) with d log2 e = h + l: the hardware's 2^h (1 step off) with the rounding of the product
// brought back, 7 instructions beside it; the library's expf takes about 15.  l is taken of a bounded d (-inf - -inf is NaN).
__device__ __forceinline__ float exp_of(float d) {
    constexpr float kLog2e = 1.442695041f, kRest = 1.925963033e-8f;     // log2 e = kLog2e + kRest
    const float b = fmaxf(d, -16000.f), l = __builtin_fmaf(b, kRest, __builtin_fmaf(b, kLog2e, -(b * kLog2e)));
    const float e = __builtin_amdgcn_exp2f(d * kLog2e);
    return __builtin_fmaf(e, l * 0.693147181f, e);
}
__device__ __forceinline__ double log1p_of(double d) { return log1p(d); }
__device__ __forceinline__ float log1p_of(float d) { return log1pf(d); }

// exp(d) for d <= 0.  Scores of 16 bits: the hardware's exp2 of the rounded product.  scale * log2 e and the product are each
// rounded, so a term is off by up to |d| 2^-23 of itself, and terms at one distance in one direction: a sum by the mean of
// |d| under p, which is the entropy less log S and so at most log V, times 2^-23, and log p and the entropy with it.  For a
// 16-bit gradient that is far below its own rounding.
template <class Ty>
__device__ __forceinline__ typename Ty::A exp_neg(typename Ty::A d) {
    if constexpr (Ty::kFast) return __builtin_amdgcn_exp2f(d * 1.44269504088896340736f);
    else return exp_of(d);
}

// below this difference a term is 0 in every type; sums take it in place of -inf, whose product with 0 is NaN
template <class A>
__device__ __forceinline__ A floor_of(A d) { return max_of(d, A(-16000)); }

// In a row's inner loop differences are multiplied by scale * unit and raised by raise(): the fast types work in powers of
// two, so that the multiplication by log2 e is the scale's, and their t is brought back at the end.
template <class Ty>
__device__ __forceinline__ typename Ty::A unit() { return Ty::kFast ? typename Ty::A(1.4426950408889634) : typename Ty::A(1); }
template <class Ty>
__device__ __forceinline__ typename Ty::A raise(typename Ty::A d) {
    if constexpr (Ty::kFast) return __builtin_amdgcn_exp2f(d);
    else return exp_of(d);
}

template <class A>
struct Part {
    A m, s, t;   // m = -inf: nothing seen but masked places (s is then 0, or NaN once a NaN was seen)
};

// Nothing read yet.  m goes through a register that the compiler cannot see into: where it knew this m to be the same for a
// wave and -infinity in 64 bits, it moved it with one scalar instruction whose constant holds 32 bits, and it became 0.  (The
// build searches the assembly of every object for such moves and fails where it finds one: other constants may meet it too.)
template <class A>
__device__ __forceinline__ Part<A> nothing() {
    A m = neg_inf(A(0));
    asm volatile("" : "+v"(m));
    return Part<A>{ m, A(0), A(0) };
}

template <class A>
__device__ __forceinline__ Part<A> join(const Part<A>& a, const Part<A>& b, A scale) {
    const A ni = neg_inf(A(0));
    const bool a_first = a.m >= b.m;
    const Part<A>&hi = a_first ? a : b, &lo = a_first ? b : a;
    if (lo.m == ni) return Part<A>{ hi.m, hi.s + lo.s, hi.t };   // lo.s: 0, or NaN
    const A d = floor_of((lo.m - hi.m) * scale), f = exp_of(d), all = lo.s + A(1);
    return Part<A>{ hi.m, hi.s + f * all, hi.t + f * (lo.t + d * all) };
}

// the finished row; a NaN or +inf among the scores makes everything NaN
template <class A>
struct Row {
    A m, ls, entropy;   // log p = (z - m) * scale - ls
    bool bad, empty;
};
template <class A>
__device__ __forceinline__ Row<A> finish(const Part<A>& p) {
    Row<A> r;
    r.m = p.m;
    r.bad = p.s != p.s || p.m == -neg_inf(A(0));
    r.empty = !r.bad && p.m == neg_inf(A(0));
    r.ls = log1p_of(p.s);
    r.entropy = r.bad ? nan_of(A(0)) : (r.empty ? A(0) : r.ls - p.t / (A(1) + p.s));
    return r;
}
template <class A>
__device__ __forceinline__ A log_p(const Row<A>& r, A z, A scale) {
    if (r.bad) return nan_of(A(0));
    if (r.empty || z == neg_inf(A(0))) return neg_inf(A(0));
    return (z - r.m) * scale - r.ls;
}
// a target of a row: < 0 none, >= width does not exist (the row's outputs become NaN)
template <class A>
__device__ __forceinline__ void given(Row<A>& r, int target, int64_t width) {
    if (target >= 0 && (int64_t)target >= width) {
        r.bad = true;
        r.empty = false;
        r.entropy = nan_of(A(0));
    }
}

template <class A>
__device__ __forceinline__ bool before(A v, int i, A w, int j) { return v > w || (v == w && i < j); }

template <class A>
struct Grad {   // weights of a row's log probability and entropy in the loss
    A g, h;
};
// d loss / d z_c = scale (g (delta - p) - h p (log p + H))
template <class Ty>
__device__ __forceinline__ typename Ty::A slope(const Row<typename Ty::A>& r, typename Ty::A z, typename Ty::A scale, bool hit,
                                                const Grad<typename Ty::A>& w) {
    using A = typename Ty::A;
    if (r.bad) return nan_of(A(0));
    if (r.empty) return A(0);
    A v = hit ? w.g : A(0);
    const A lp = (z - r.m) * scale - r.ls;
    const A p = exp_neg<Ty>(lp);
    if (p > A(0)) v -= p * (w.g + w.h * (lp + r.entropy));
    return v * scale;
}

// ---- lanes ---------------------------------------------------------------------------------------------------------
// a value of one lane (the lane's number is the same for the whole wave) for all
__device__ __forceinline__ int lane_of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ float lane_of(float v, int lane) { return __int_as_float(lane_of(__float_as_int(v), lane)); }
__device__ __forceinline__ double lane_of(double v, int lane) {
    return __hiloint2double(lane_of(__double2hiint(v), lane), lane_of(__double2loint(v), lane));
}
template <int kCtrl>
__device__ __forceinline__ int dpp(int old, int v) { return __builtin_amdgcn_update_dpp(old, v, kCtrl, 0xf, 0xf, false); }
template <int kCtrl>
__device__ __forceinline__ float dpp(float old, float v) { return __int_as_float(dpp<kCtrl>(__float_as_int(old), __float_as_int(v))); }
template <int kCtrl>
__device__ __forceinline__ double dpp(double old, double v) {
    return __hiloint2double(dpp<kCtrl>(__double2hiint(old), __double2hiint(v)), dpp<kCtrl>(__double2loint(old), __double2loint(v)));
}
constexpr int kShr1 = 0x111, kShr2 = 0x112, kShr4 = 0x114, kShr8 = 0x118, kBcast15 = 0x142, kBcast31 = 0x143;
// the largest of a wave's values, for all lanes
template <class A>
__device__ __forceinline__ A wave_max(A v) {
    v = max_of(v, dpp<kShr1>(v, v));
    v = max_of(v, dpp<kShr2>(v, v));
    v = max_of(v, dpp<kShr4>(v, v));
    v = max_of(v, dpp<kShr8>(v, v));
    v = max_of(v, dpp<kBcast15>(v, v));
    v = max_of(v, dpp<kBcast31>(v, v));
    return lane_of(v, 63);
}
// an exchange with the lane 2^o away, without shared memory up to 16 lanes (within groups that are uniform already, which
// is what a reduction over all smaller distances leaves)
template <int o, class A>
__device__ __forceinline__ A across(A v) {
    if constexpr (o == 1) return dpp<0xB1>(v, v);        // pairs
    else if constexpr (o == 2) return dpp<0x4E>(v, v);   // halves of four
    else if constexpr (o == 4) return dpp<0x141>(v, v);  // eight, mirrored
    else if constexpr (o == 8) return dpp<0x140>(v, v);  // sixteen, mirrored
    else return __shfl_xor(v, o);
}
// f(value of the other half) for distances 1, 2 .. G / 2
template <int G, int o = 1, class F>
__device__ __forceinline__ void reduce(F f) {
    if constexpr (o < G) {
        f(std::integral_constant<int, o>());
        reduce<G, 2 * o>(f);
    }
}

// ---- short rows: G lanes of a wave hold a row, E elements each ----------------------------------------------------
// Everything stays in registers; the best outcomes are taken one by one (an argmax over the lanes' own best).  65536 rows of
// 12 in 64 bits, top 2: 7.3 us, with the gradient 9.6 (6.3 and 12.6 MB are 1.3 and 2.6 us at the rate of a copy); what is
// left is the launch and the chain load, maximum, exponentials, logarithm, of which 1024 workgroups each make one.
template <class Ty, int G, int E, bool kGrad>
__global__ __launch_bounds__(kT) void k_lp_short(const typename Ty::S* __restrict__ z, int64_t rows, int width, int64_t ld,
                                                 typename Ty::A scale, const int32_t* __restrict__ target, int top_k,
                                                 const typename Ty::A* __restrict__ dg, const typename Ty::A* __restrict__ dh,
                                                 typename Ty::A* lp_out, typename Ty::A* ent_out, typename Ty::A* top_lp,
                                                 int32_t* top_ix, typename Ty::S* dz, int64_t ld_dz) {
    using A = typename Ty::A;
    constexpr int kRows = kT / G;
    const int lane = threadIdx.x % G;
    for (int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / G; row < rows; row += (int64_t)gridDim.x * kRows) {
        const typename Ty::S* zr = z + row * ld;
        A v[E];
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int c = lane + G * i;
            v[i] = c < width ? Ty::up(zr[c]) : neg_inf(A(0));
        }
        A m = v[0];
        bool nan = v[0] != v[0];
#pragma unroll
        for (int i = 1; i < E; ++i) {
            m = max_of(m, v[i]);
            nan |= v[i] != v[i];
        }
        if (nan) m = neg_inf(A(0));
        reduce<G>([&](auto o) { m = max_of(m, across<o.value>(m)); });
        const A base = m == neg_inf(A(0)) ? A(0) : m;
        // which element is the one whose term is left out: the first at the maximum
        int first = 0x7fffffff;
#pragma unroll
        for (int i = E - 1; i >= 0; --i)
            if (v[i] == m) first = lane + G * i;
        reduce<G>([&](auto o) { first = min(first, across<o.value>(first)); });
        A s = nan ? nan_of(A(0)) : A(0), t = A(0);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const A d = (v[i] - base) * scale;
            const bool skip = v[i] == neg_inf(A(0)) || lane + G * i == first;
            const A e = skip ? A(0) : exp_neg<Ty>(d);
            s += e;
            t += skip ? A(0) : e * floor_of(d);
        }
        reduce<G>([&](auto o) {
            s += across<o.value>(s);
            t += across<o.value>(t);
        });
        Row<A> r = finish(Part<A>{ m, s, t });
        const int tg = target ? target[row] : -1;
        given(r, tg, width);
        if (lane == 0) {
            if (ent_out) ent_out[row] = r.entropy;
            if (lp_out) lp_out[row] = r.bad ? nan_of(A(0)) : (tg < 0 ? A(0) : log_p(r, Ty::up(zr[tg]), scale));
        }
        if constexpr (kGrad) {
            const Grad<A> w = { tg < 0 ? A(0) : (dg ? dg[row] : A(0)), dh ? dh[row] : A(0) };
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const int c = lane + G * i;
                if (c < width) dz[row * ld_dz + c] = Ty::down(slope<Ty>(r, v[i], scale, c == tg, w));
            }
        } else {
            uint32_t used = 0;
            for (int k = 0; k < top_k; ++k) {
                A bv = neg_inf(A(0));
                int bi = 0x7fffffff, at = -1;
#pragma unroll
                for (int i = 0; i < E; ++i)
                    if (!(used >> i & 1) && v[i] > bv) { bv = v[i]; bi = lane + G * i; at = i; }
                const int mine = bi;
                reduce<G>([&](auto o) {
                    const A ov = across<o.value>(bv);
                    const int oi = across<o.value>(bi);
                    if (before(ov, oi, bv, bi)) { bv = ov; bi = oi; }
                });
                if (at >= 0 && mine == bi) used |= 1u << at;
                if (lane == 0) {
                    const bool none = r.bad || bi == 0x7fffffff;
                    top_lp[row * top_k + k] = r.bad ? nan_of(A(0)) : (none ? neg_inf(A(0)) : log_p(r, bv, scale));
                    top_ix[row * top_k + k] = none ? -1 : bi;
                }
            }
        }
    }
}

// ---- long rows ----------------------------------------------------------------------------------------------------
// A workgroup reads one of `splits` equal parts of a row, in 16-byte pieces; part boundaries and the first piece are
// aligned in memory, elements outside the row count as masked (-inf).
template <class Ty>
struct Piece {
    static constexpr int N = 16 / sizeof(typename Ty::S);
    int64_t off, pieces;            // elements before the row in its first piece; pieces of the whole row
    __device__ Piece(const typename Ty::S* row, int64_t width) {
        off = (int64_t)(((uintptr_t)row & 15) / sizeof(typename Ty::S));
        pieces = (off + width + N - 1) / N;
    }
};

template <class Ty>
__device__ __forceinline__ void load_piece(const typename Ty::S* zr, int64_t e0, int64_t width, typename Ty::A* v) {
    constexpr int N = Piece<Ty>::N;
    if (e0 >= 0 && e0 + N <= width) {
        alignas(16) typename Ty::S raw[N];
        *reinterpret_cast<uint4*>(raw) = *reinterpret_cast<const uint4*>(zr + e0);
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = Ty::up(raw[j]);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = e0 + j >= 0 && e0 + j < width ? Ty::up(zr[e0 + j]) : neg_inf(typename Ty::A(0));
    }
}

__device__ __forceinline__ float lowest(float) { return -3.402823466e38f; }
__device__ __forceinline__ double lowest(double) { return -1.7976931348623157e308; }
template <class A>
struct Best {
    A v;
    int i;
};
template <class A>
__device__ __forceinline__ Best<A> nobody() { return Best<A>{ neg_inf(A(0)), 0x7fffffff }; }

// orders a wave's own writes to and reads of shared memory
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A bound below the k-th best of a wave's first elements, from the lanes' own best mx: k lanes or more reach it.  It keeps
// the first pieces from offering each element that is better than those before it (about k log(elements / k) of them).
template <class A>
__device__ __forceinline__ A first_bound(A mx, int top_k) {
    if (__popcll(__ballot(mx > neg_inf(A(0)))) < top_k) return neg_inf(A(0));
    A hi = wave_max(mx), lo = -wave_max(mx > neg_inf(A(0)) ? -mx : neg_inf(A(0)));
    for (int n = 0; n < 12; ++n) {
        const A mid = A(0.5) * lo + A(0.5) * hi;
        const int reach = __popcll(__ballot(mx >= mid));
        if (reach >= top_k) lo = mid;
        else hi = mid;
        if (reach == top_k) break;
    }
    return lo;
}

// A wave's candidates for its top_k best outcomes, in shared memory and in no order: all that it has seen above a bound which
// top_k of them reach.  Candidates are only written down, which many lanes do at once; when there are too many the bound is
// raised, and the order is found at the end by counting.  (Kept in order by inserting them one by one, each took 0.19 us of
// its wave: a row of 131072, top 20, in 32 workgroups 15.8 us where the read-out without outcomes takes 5.5, and the joining
// of the lists as long again.)
constexpr int kPool = 128;
template <class A>
struct Store {
    A v[kPool];
    int i[kPool];
};
__device__ __forceinline__ float next_up(float v) {
    const int b = __float_as_int(v);
    return v == 0.f ? __int_as_float(1) : __int_as_float(b < 0 ? b - 1 : b + 1);
}
__device__ __forceinline__ double next_up(double v) {
    const long long b = __double_as_longlong(v);
    return v == 0.0 ? __longlong_as_double(1) : __longlong_as_double(b < 0 ? b - 1 : b + 1);
}
template <class A>
struct Pool {
    Store<A>* of;
    int n, top_k;      // the same for the wave, as the rest:
    A bound;           // top_k of what was seen reach it
    A least;           // the least value that counts: the bound, or above it what reaches it was there before, at lower indices

    __device__ __forceinline__ Pool(Store<A>* s, int k) : of(s), n(0), top_k(k), bound(neg_inf(A(0))), least(lowest(A(0))) {}
    __device__ __forceinline__ void raise_to(A b) {
        if (b > bound) bound = least = b;
    }
    // Values v[0 .. B) of each lane, id(j) the index of v[j]; possible(j): whether any lane's v[j ..] up to a multiple of N may
    // count.  ordered: what is offered has lower indices than all that follows.
    template <int B, int N, class F, class G>
    __device__ __forceinline__ void offer(const A* v, F id, G possible, bool ordered, int lane) {
        int from = 0;      // those before it are written down
        for (;;) {
            int stop = B;  // the first that there is no room for
#pragma unroll
            for (int j0 = 0; j0 < B; j0 += N) {
                if (j0 + N <= from || stop < B || !possible(j0)) continue;
#pragma unroll
                for (int j = j0; j < j0 + N; ++j) {
                    const uint64_t want = __ballot(v[j] >= least);
                    if (!want || j < from || stop < B) continue;
                    const int c = __popcll(want);
                    if (n + c > kPool) {
                        stop = j;
                        continue;
                    }
                    if (want >> lane & 1) {
                        const int at = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(want >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)want, 0));
                        of->v[at] = v[j];
                        of->i[at] = id(j);
                    }
                    n += c;
                }
            }
            wave_fence();
            if (n > min(kPool / 2, max(8, 2 * top_k))) prune(lane);
            if (stop == B) break;
            from = stop;
        }
        if (ordered) least = next_up(bound);
    }
    // at most 64 of them, or top_k, with all that are among the best
    __device__ __forceinline__ void prune(int lane) {
        if (n <= top_k) return;
        const A v0 = lane < n ? of->v[lane] : neg_inf(A(0)), v1 = 64 + lane < n ? of->v[64 + lane] : neg_inf(A(0));
        const int i0 = of->i[lane], i1 = of->i[64 + lane];
        wave_fence();
        const A inf = -neg_inf(A(0));
        A lo = -wave_max(max_of(lane < n ? -v0 : -inf, 64 + lane < n ? -v1 : -inf)), hi = wave_max(max_of(v0, v1));
        int reach = n;
        for (int s = 0; s < 14 && reach > top_k; ++s) {
            const A mid = A(0.5) * lo + A(0.5) * hi;
            const int r = __popcll(__ballot(v0 >= mid)) + __popcll(__ballot(v1 >= mid));
            if (r >= top_k) {
                lo = mid;
                reach = r;
            } else {
                hi = mid;
            }
        }
        if (reach > kPool / 2 || reach > top_k + 8) {     // close together or equal: by their ranks
            rank(lane);
            return;
        }
        const uint64_t w0 = __ballot(lane < n && v0 >= lo), w1 = __ballot(64 + lane < n && v1 >= lo);
        const int n0 = __popcll(w0);
        if (w0 >> lane & 1) {
            const int at = __builtin_amdgcn_mbcnt_hi((uint32_t)(w0 >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)w0, 0));
            of->v[at] = v0;
            of->i[at] = i0;
        }
        if (w1 >> lane & 1) {
            const int at = n0 + __builtin_amdgcn_mbcnt_hi((uint32_t)(w1 >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)w1, 0));
            of->v[at] = v1;
            of->i[at] = i1;
        }
        wave_fence();
        n = reach;
        raise_to(lo);
    }
    // the best top_k of them (or all), best first
    __device__ __forceinline__ void rank(int lane) {
        const bool two = n > 64;
        const Best<A> a = lane < n ? Best<A>{ of->v[lane], of->i[lane] } : nobody<A>();
        const Best<A> b = 64 + lane < n ? Best<A>{ of->v[64 + lane], of->i[64 + lane] } : nobody<A>();
        int ra = 0, rb = 0;
        if (two) {
            for (int e = 0; e < n; ++e) {
                ra += before(of->v[e], of->i[e], a.v, a.i);
                rb += before(of->v[e], of->i[e], b.v, b.i);
            }
        } else {
#pragma unroll 4
            for (int e = 0; e < n; ++e) ra += before(of->v[e], of->i[e], a.v, a.i);
        }
        wave_fence();
        if (lane < n && ra < top_k) {
            of->v[ra] = a.v;
            of->i[ra] = a.i;
        }
        if (64 + lane < n && rb < top_k) {
            of->v[rb] = b.v;
            of->i[rb] = b.i;
        }
        wave_fence();
        if (n >= top_k) {
            n = top_k;
            raise_to(lane_of(of->v[top_k - 1], 0));
        }
    }
    __device__ __forceinline__ void finish(int lane) {
        if (n > top_k + 16) prune(lane);
        rank(lane);
    }
    __device__ __forceinline__ Best<A> best(int lane) const { return lane < n ? Best<A>{ of->v[lane], of->i[lane] } : nobody<A>(); }
    // how many of a finished pool's outcomes come before one of another pool
    static __device__ __forceinline__ int ahead(const Store<A>& s, int n, const Best<A>& b) {
        int at = 0;
#pragma unroll
        for (int step = 64; step; step >>= 1)
            if (at + step <= n && before(s.v[at + step - 1], s.i[at + step - 1], b.v, b.i)) at += step;
        return at;
    }
};

// U pieces a lane into the wave's running state.  m is the wave's (the same in all lanes), s and t are the lane's.
template <class Ty, int U, bool kTop>
__device__ __forceinline__ void take(const typename Ty::A* v, const int* at, Part<typename Ty::A>& p, Pool<typename Ty::A>& pool,
                                     typename Ty::A k, int lane) {
    using A = typename Ty::A;
    constexpr int N = Piece<Ty>::N, B = U * N;
    A piece_max[U], mx = neg_inf(A(0));
#pragma unroll
    for (int u = 0; u < U; ++u) {
        piece_max[u] = v[u * N];
#pragma unroll
        for (int j = 1; j < N; ++j) piece_max[u] = max_of(piece_max[u], v[u * N + j]);
        mx = max_of(mx, piece_max[u]);
    }
    if constexpr (kTop) {
        if (__ballot(mx >= pool.least)) {
            if (pool.bound == neg_inf(A(0))) pool.raise_to(first_bound(mx, pool.top_k));
            const auto id = [&](int j) {
                int i = at[j / N];
                asm volatile("" : "+v"(i));   // (added where it is needed: B sums kept for the loop cost B registers)
                return i + j % N;
            };
            pool.template offer<B, N>(v, id, [&](int j) { return __ballot(piece_max[j / N] >= pool.least) != 0; },
                                      true, lane);
        }
    }
    if (__ballot(mx > p.m)) {                     // a new maximum (a NaN is not taken as one, it shows in s)
        const A m = wave_max(max_of(mx, p.m));
        const uint64_t holders = __ballot(mx == m);
        if (p.m > neg_inf(A(0))) {                // the old one's term comes in, in lane 0's sums
            const A d = floor_of((p.m - m) * k), f = raise<Ty>(d), all = p.s + (lane == 0 ? A(1) : A(0));
            p.s = f * all;
            p.t = f * (p.t + d * all);
        }
        p.m = m;
        bool left_out = lane != __builtin_ctzll(holders);     // one of the lanes that have it leaves its first one out
#pragma unroll
        for (int j = 0; j < B; ++j) {
            const A d = (v[j] - m) * k;
            const bool out = !left_out && v[j] == m;
            left_out |= out;
            const A e = out ? A(0) : raise<Ty>(d);
            p.s += e;
            p.t += e * floor_of(d);
        }
    } else {
        const A m = p.m == neg_inf(A(0)) ? A(0) : p.m;
#pragma unroll
        for (int j = 0; j < B; ++j) {
            const A d = (v[j] - m) * k;
            const A e = raise<Ty>(d);
            p.s += e;
            p.t += e * floor_of(d);
        }
    }
}

// pieces p0 + first + lane, + step .. of a row by one wave; all lanes hold the result
template <class Ty, bool kTop>
__device__ __forceinline__ Part<typename Ty::A> read_pieces(const typename Ty::S* zr, int64_t width, const Piece<Ty>& pc, int64_t p0,
                                                            int64_t p1, int step, typename Ty::A scale, Pool<typename Ty::A>& pool) {
    using A = typename Ty::A;
    constexpr int N = Piece<Ty>::N, U = 2;
    const int lane = threadIdx.x & 63;
    Part<A> p = nothing<A>();
    const A k = scale * unit<Ty>();
    for (int64_t q = p0; q < p1; q += step * U) {    // the same count for a wave's lanes
        A v[U * N];
        int at[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t piece = q + u * step + lane, e0 = piece < p1 ? piece * N - pc.off : width;
            at[u] = (int)e0;
            load_piece<Ty>(zr, e0, width, v + u * N);
        }
        take<Ty, U, kTop>(v, at, p, pool, k, lane);
    }
    reduce<64>([&](auto o) {
        p.s += across<o.value>(p.s);
        p.t += across<o.value>(p.t);
    });
    p.t *= A(1) / unit<Ty>();
    if constexpr (kTop) pool.finish(lane);
    return p;
}

// a part of a row by one workgroup; the result is complete in wave 0 (all lanes)
template <class Ty, bool kTop>
__device__ __forceinline__ Part<typename Ty::A> read_part(const typename Ty::S* zr, int64_t width, int split, int splits,
                                                          typename Ty::A scale, int top_k, Best<typename Ty::A>& best) {
    using A = typename Ty::A;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Piece<Ty> pc(zr, width);
    const int64_t per = (pc.pieces + splits - 1) / splits, p0 = split * per, p1 = min(pc.pieces, p0 + per);
    __shared__ Part<A> sp[kWaves];
    __shared__ Store<A> store[kTop ? kWaves : 1];
    __shared__ Best<A> sb[64];
    __shared__ int sn[kWaves];
    Pool<A> pool(&store[kTop ? wave : 0], top_k);
    Part<A> p = read_pieces<Ty, kTop>(zr, width, pc, p0 + wave * 64, p1, kT, scale, pool);
    if (lane == 0) {
        sp[wave] = p;
        sn[wave] = pool.n;
    }
    __syncthreads();
    if constexpr (kTop) {
        // an outcome's place among all waves': those before it in its own pool and in the others
        const Best<A> mine = pool.best(lane);
        int at = lane, all = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            all += sn[w];
            if (w != wave) at += Pool<A>::ahead(store[w], sn[w], mine);
        }
        if (lane < pool.n && at < top_k) sb[at] = mine;
        __syncthreads();
        best = lane < min(all, top_k) ? sb[lane] : nobody<A>();
    }
    if (wave == 0) {
#pragma unroll
        for (int w = 1; w < kWaves; ++w) p = join(p, sp[w], scale);
    }
    return p;
}

template <class A>
struct Ws {   // the parts of the rows, and the parts' best outcomes
    Part<A>* part;
    Best<A>* best;
};

// what a row's call returns, by the lanes of one wave that all hold the row's state
template <class Ty>
struct Out {
    using A = typename Ty::A;
    const int32_t* target;
    A *lp, *ent, *top_lp;
    int32_t* top_ix;
    int top_k;
    __device__ __forceinline__ void write(int64_t row, const typename Ty::S* zr, int64_t width, const Part<A>& p, const Best<A>& best,
                                          A scale, int lane) const {
        Row<A> r = finish(p);
        const int tg = target ? target[row] : -1;
        given(r, tg, width);
        if (lane == 0) {
            if (ent) ent[row] = r.entropy;
            if (lp) lp[row] = r.bad ? nan_of(A(0)) : (tg < 0 ? A(0) : log_p(r, Ty::up(zr[tg]), scale));
        }
        if (lane < top_k) {
            const bool none = r.bad || best.i == 0x7fffffff;
            top_lp[row * top_k + lane] = r.bad ? nan_of(A(0)) : (none ? neg_inf(A(0)) : log_p(r, best.v, scale));
            top_ix[row * top_k + lane] = none ? -1 : best.i;
        }
    }
};

// splits = 1: the workgroup writes the row's results, else its part of them.
// Eight waves a SIMD hide the way from memory (64 registers, with outcomes of 16 bits 4 more in scratch; two pieces of 16 bytes a
// lane at once): 2048 rows of 100003
// bfloat16, top 8, 114 us = 3.6 TB/s, 151 with 5 waves and four pieces; without outcomes 96 us = 4.3 TB/s.
template <class Ty, bool kTop>
__global__ __launch_bounds__(kT, sizeof(typename Ty::A) == 4 ? 8 : 4) void k_lp_parts(const typename Ty::S* __restrict__ z, int64_t rows, int64_t width, int64_t ld,
                                                 typename Ty::A scale, int top_k, int splits, Ws<typename Ty::A> ws, Out<Ty> out) {
    using A = typename Ty::A;
    for (int64_t it = blockIdx.x; it < rows * splits; it += gridDim.x) {
        const int64_t row = it / splits;
        const int split = (int)(it - row * splits);
        Best<A> best;
        const Part<A> p = read_part<Ty, kTop>(z + row * ld, width, split, splits, scale, top_k, best);
        if (threadIdx.x < 64) {
            if (splits == 1 && !ws.part) {
                out.write(row, z + row * ld, width, p, best, scale, threadIdx.x);
            } else {
                if (threadIdx.x == 0) ws.part[it] = p;
                if constexpr (kTop)
                    if ((int)threadIdx.x < top_k) ws.best[it * top_k + threadIdx.x] = best;
            }
        }
        __syncthreads();   // the shared arrays are written again
    }
}

// One wave a row.  65536 rows of 1024 bfloat16, top 4, 63 us (the way of short rows, an argmax an outcome: 125), 20000 of 2000
// float32, top 5, 47;  bound by instructions: the bound, the places and the order of a row's candidates are its wave's own.
template <class Ty, bool kTop>
__global__ __launch_bounds__(kT) void k_lp_wave(const typename Ty::S* __restrict__ z, int64_t rows, int64_t width, int64_t ld,
                                                typename Ty::A scale, int top_k, Out<Ty> out) {
    using A = typename Ty::A;
    __shared__ Store<A> store[kTop ? kWaves : 1];
    for (int64_t row = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6); row < rows; row += (int64_t)gridDim.x * kWaves) {
        const typename Ty::S* zr = z + row * ld;
        const Piece<Ty> pc(zr, width);
        Pool<A> pool(&store[kTop ? threadIdx.x >> 6 : 0], top_k);
        const Part<A> p = read_pieces<Ty, kTop>(zr, width, pc, 0, pc.pieces, 64, scale, pool);
        const Best<A> best = kTop ? pool.best(threadIdx.x & 63) : nobody<A>();
        out.write(row, zr, width, p, best, scale, threadIdx.x & 63);
    }
}

// a row's parts (at most 64), joined in a fixed tree by a wave
template <class A>
__device__ __forceinline__ Part<A> join_parts(const Part<A>* part, int splits, A scale, int lane) {
    Part<A> p = nothing<A>();
    if (lane < splits) p = part[lane];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) p = join(p, Part<A>{ __shfl_xor(p.m, o), __shfl_xor(p.s, o), __shfl_xor(p.t, o) }, scale);
    return p;
}

// One wave a row: joins its parts and their lists of best outcomes.  32 parts, top 20: 6.8 us, 2.8 without outcomes, 15.5 with
// the lists merged one outcome after the other.
template <class Ty>
__global__ __launch_bounds__(64) void k_lp_join(const typename Ty::S* __restrict__ z, int64_t rows, int64_t width, int64_t ld,
                                                typename Ty::A scale, int top_k, int splits, Ws<typename Ty::A> ws, Out<Ty> out) {
    using A = typename Ty::A;
    const int lane = threadIdx.x;
    __shared__ Store<A> store;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        Pool<A> pool(&store, top_k);
        if (top_k > 0) {
            constexpr int U = 16;
            const Best<A>* from = ws.best + row * splits * top_k;
            const int all = splits * top_k;
            for (int e0 = 0; e0 < all; e0 += 64 * U) {
                A v[U], mx = neg_inf(A(0));
                int ix[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const Best<A> c = e0 + u * 64 + lane < all ? from[e0 + u * 64 + lane] : nobody<A>();
                    v[u] = c.v;
                    ix[u] = c.i;
                    mx = max_of(mx, c.v);
                }
                if (pool.bound == neg_inf(A(0))) pool.raise_to(first_bound(mx, top_k));
                pool.template offer<U, U>(v, [&](int j) { return ix[j]; }, [](int) { return true; }, false, lane);
            }
            pool.finish(lane);
        }
        const Best<A> best = pool.best(lane);
        out.write(row, z + row * ld, width, join_parts(ws.part + row * splits, splits, scale, lane), best, scale, lane);
    }
}

// one piece of the gradient: 16 bytes at once where both rows allow it
template <class Ty>
__device__ __forceinline__ void store_piece(typename Ty::S* dr, int64_t e0, int64_t width, bool whole, const typename Ty::A* v) {
    constexpr int N = Piece<Ty>::N;
    if (whole && e0 >= 0 && e0 + N <= width) {
        alignas(16) typename Ty::S raw[N];
#pragma unroll
        for (int j = 0; j < N; ++j) raw[j] = Ty::down(v[j]);
        *reinterpret_cast<uint4*>(dr + e0) = *reinterpret_cast<const uint4*>(raw);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (e0 + j >= 0 && e0 + j < width) dr[e0 + j] = Ty::down(v[j]);
    }
}

// The gradient of pieces first, + T .. below `past` of a row whose state is known.
template <class Ty, int T>
__device__ __forceinline__ void write_slopes(const typename Ty::S* zr, typename Ty::S* dr, int64_t width, const Piece<Ty>& pc, int64_t first,
                                             int64_t past, const Row<typename Ty::A>& r, int tg, const Grad<typename Ty::A>& w,
                                             typename Ty::A scale) {
    using A = typename Ty::A;
    constexpr int N = Piece<Ty>::N, U = 2;
    const bool whole = (((uintptr_t)zr ^ (uintptr_t)dr) & 15) == 0, plain = !r.bad && !r.empty;
    const A k = scale * unit<Ty>(), w0 = -scale * (w.g + w.h * r.entropy), w1 = -scale * w.h / unit<Ty>(), ls = r.ls * unit<Ty>();
    for (int64_t q = first; q < past; q += T * U) {
        A v[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u) load_piece<Ty>(zr, q + u * T < past ? (q + u * T) * N - pc.off : width, width, v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (q + u * T >= past) break;
            const int64_t e0 = (q + u * T) * N - pc.off;
            if (plain) {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const A lp = floor_of((v[u][j] - r.m) * k - ls);     // masked: p is 0, and 0 times a number
                    v[u][j] = raise<Ty>(lp) * (lp * w1 + w0);
                }
                if (tg >= e0 && tg < e0 + N) {
#pragma unroll
                    for (int j = 0; j < N; ++j) v[u][j] += tg == e0 + j ? scale * w.g : A(0);
                }
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) v[u][j] = r.bad ? nan_of(A(0)) : A(0);
            }
            store_piece<Ty>(dr, e0, width, whole, v[u]);
        }
    }
}

// the row's log probability and entropy beside its gradient, by one thread; returns the state for the gradient
template <class Ty>
struct LossOut {
    using A = typename Ty::A;
    const int32_t* target;
    const A *dg, *dh;
    A *lp, *ent;
    typename Ty::S* dz;
    int64_t ld_dz;
    __device__ __forceinline__ Row<A> row(int64_t r, const typename Ty::S* zr, int64_t width, const Part<A>& p, A scale, bool write,
                                          int& tg, Grad<A>& w) const {
        Row<A> s = finish(p);
        tg = target ? target[r] : -1;
        given(s, tg, width);
        if (write) {
            if (ent) ent[r] = s.entropy;
            if (lp) lp[r] = s.bad ? nan_of(A(0)) : (tg < 0 ? A(0) : log_p(s, Ty::up(zr[tg]), scale));
        }
        w = Grad<A>{ tg < 0 ? A(0) : (dg ? dg[r] : A(0)), dh ? dh[r] : A(0) };
        return s;
    }
};

// The gradient of one part of a row, from the joined parts (few rows: the row is read again).  16 rows of 50000 float32: 8.8 us
// for the parts and 8.6 here, both launch and latency.
template <class Ty>
__global__ __launch_bounds__(kT) void k_lp_slope(const typename Ty::S* __restrict__ z, int64_t rows, int64_t width, int64_t ld,
                                                 typename Ty::A scale, int splits, Ws<typename Ty::A> ws, LossOut<Ty> out) {
    using A = typename Ty::A;
    for (int64_t it = blockIdx.x; it < rows * splits; it += gridDim.x) {
        const int64_t row = it / splits;
        const int split = (int)(it - row * splits);
        const typename Ty::S* zr = z + row * ld;
        typename Ty::S* dr = out.dz + row * out.ld_dz;
        int tg;
        Grad<A> w;
        const Row<A> r = out.row(row, zr, width, join_parts(ws.part + row * splits, splits, scale, threadIdx.x & 63), scale,
                                 split == 0 && threadIdx.x == 0, tg, w);
        const Piece<Ty> pc(zr, width);
        const int64_t per = (pc.pieces + splits - 1) / splits, p1 = min(pc.pieces, (split + 1) * per);
        write_slopes<Ty, kT>(zr, dr, width, pc, split * per + threadIdx.x, p1, r, tg, w, scale);
    }
}

// Waves a SIMD that the registers shall leave room for: as many as do without the compiler's moving parts of the row out, but for
// 16-bit rows of 512 threads, of whose 16 pieces 18 (bfloat16) and 27 registers (float16) lie in scratch.
constexpr int waves_a_simd(int T, int NP, size_t size) { return size == 8 ? 2 : NP <= 8 || T > 256 ? 4 : 3; }

// A row's loss with the row in the registers of one workgroup (NP pieces of 16 bytes a thread): read once, written once.
// Three passes over the registers: the maximum; the sums; the gradient p (w0 + w1 log p), w0 = -scale (g + h H), w1 = -scale h.
// Bound by HBM as long as the passes' arithmetic (about 30 instruction slots an element of 32 bits, 22 of 16) hides under it:
// 4000 rows of 32001 float32 199 us = 5.1 TB/s read and written, as fast as a copy; of 8000 bfloat16 35 us = 3.7 TB/s, bound by
// the arithmetic.
template <class Ty, int T, int NP>
__global__ __launch_bounds__(T, waves_a_simd(T, NP, sizeof(typename Ty::S))) void k_lp_loss(const typename Ty::S* __restrict__ z, int64_t rows,
                                                                                          int64_t width, int64_t ld, typename Ty::A scale,
                                                                                          LossOut<Ty> out) {
    using A = typename Ty::A;
    using S = typename Ty::S;
    constexpr int N = Piece<Ty>::N, W = T / 64;
    __shared__ A sm[W], ss[W], st[W];
    __shared__ int sc[W];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const S* zr = z + row * ld;
        const int off = (int)Piece<Ty>(zr, width).off, end = (int)width + off;      // elements from the first piece on
        const int first = (int)threadIdx.x * N;                                       // the thread's, of its piece 0
        // pieces lo <= n < hi of the thread lie whole in the row, those from past on outside it
        int lo = first < off ? 1 : 0, hi = end - N < first ? 0 : (end - N - first) / (T * N) + 1, past = end <= first ? 0 : (end - 1 - first) / (T * N) + 1;
        // element j of a piece that does not lie whole in the row
        auto inside = [&](int n, int j) { return first + n * (T * N) + j >= off && first + n * (T * N) + j < end; };
        auto edge = [&](int n) {      // a piece that the row begins or ends in
            alignas(16) S v[N];
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = inside(n, j) ? zr[n * (T * N) + first - off + j] : Ty::down(neg_inf(A(0)));
            return *reinterpret_cast<const uint4v*>(v);
        };
        alignas(16) S masked[N];
#pragma unroll
        for (int j = 0; j < N; ++j) masked[j] = Ty::down(neg_inf(A(0)));
        uint4v raw[NP];
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            raw[n] = *reinterpret_cast<const uint4v*>(masked);
            if (n >= lo && n < hi) raw[n] = *reinterpret_cast<const uint4v*>(zr - off + n * (T * N) + first);
        }
        if (lo > 0) raw[0] = edge(0);
        if (__ballot(past > hi && past > lo)) {
            const int last = past > hi && past > lo ? past - 1 : -1;
            uint4v e = *reinterpret_cast<const uint4v*>(masked);
            if (last >= 0) e = edge(last);
#pragma unroll
            for (int n = 0; n < NP; ++n) raw[n] = n == last ? e : raw[n];
        }
        // the stored 16 bits are unpacked anew in each pass (twice the registers would not do), so the compiler may not
        // know that they are the same
        auto anew = [&] {
            if constexpr (sizeof(S) == 2) {
#pragma unroll
                for (int n = 0; n < NP; ++n) asm volatile("" : "+v"(raw[n]));
            }
        };
        auto piece = [&](int n, A* v) {
            alignas(16) S x[N];
            __builtin_amdgcn_sched_barrier(0);     // a piece at a time: many at once take more registers than the row
            *reinterpret_cast<uint4v*>(x) = raw[n];
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = Ty::up(x[j]);
        };
        A mine_max = neg_inf(A(0));
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            A v[N];
            piece(n, v);
#pragma unroll
            for (int j = 0; j < N; ++j) mine_max = max_of(mine_max, v[j]);
        }
        A m = wave_max(mine_max);
        if (W > 1) {
            if (lane == 0) sm[wave] = m;
            __syncthreads();
            m = sm[0];
#pragma unroll
            for (int w = 1; w < W; ++w) m = max_of(m, sm[w]);
        }
        const A from = m == neg_inf(A(0)) ? A(0) : m, k = scale * unit<Ty>();
        // s: the terms below the maximum; the elements at the maximum are counted, and one of them is left out
        A s = A(0), t = A(0);
        int top = 0;
        anew();
        if (__ballot(mine_max == m)) {
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                A v[N];
                piece(n, v);
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const A d = (v[j] - from) * k, e = raise<Ty>(d);
                    const bool at = v[j] == m;              // (everything masked: counted, and not used)
                    top += at;
                    s += at ? A(0) : e;
                    t += e * floor_of(d);
                }
            }
        } else {
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                A v[N];
                piece(n, v);
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const A d = (v[j] - from) * k, e = raise<Ty>(d);
                    s += e;
                    t += e * floor_of(d);
                }
            }
        }
        reduce<64>([&](auto o) {
            s += across<o.value>(s);
            t += across<o.value>(t);
            top += across<o.value>(top);
        });
        if (W > 1) {
            if (lane == 0) { ss[wave] = s; st[wave] = t; sc[wave] = top; }
            __syncthreads();
            s = A(0);
            t = A(0);
            top = 0;
            for (int w = 0; w < W; ++w) { s += ss[w]; t += st[w]; top += sc[w]; }
        }
        if (m > neg_inf(A(0)) && top > 1) s += (A)(top - 1);
        t *= A(1) / unit<Ty>();
        int tg;
        Grad<A> w;
        const Row<A> r = out.row(row, zr, width, Part<A>{ m, s, t }, scale, threadIdx.x == 0, tg, w);
        S* dr = out.dz + row * out.ld_dz;
        if (((uintptr_t)zr ^ (uintptr_t)dr) & 15) hi = 0;      // pieces of the gradient are not aligned as the scores' are
        const A w0 = -scale * (w.g + w.h * r.entropy), w1 = -scale * w.h / unit<Ty>(), ls = r.ls * unit<Ty>();
        const bool plain = !r.bad && !r.empty;
        const int hit = tg < 0 ? -1 : tg + off - first;          // the target, counted from the thread's piece 0
        anew();
        asm volatile("" : "+v"(lo), "+v"(hi), "+v"(past));       // (compared again, not kept as NP masks)
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            A v[N];
            piece(n, v);
            if (plain) {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const A lp = floor_of((v[j] - m) * k - ls);     // masked: p is 0, and 0 times a number
                    v[j] = raise<Ty>(lp) * (lp * w1 + w0);
                }
                if ((unsigned)(hit - n * (T * N)) < (unsigned)N) {
#pragma unroll
                    for (int j = 0; j < N; ++j) v[j] += hit == n * (T * N) + j ? scale * w.g : A(0);
                }
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) v[j] = r.bad ? nan_of(A(0)) : A(0);
            }
            S* to = dr - off + n * (T * N) + first;
            if (n >= lo && n < hi) {
                alignas(16) S x[N];
#pragma unroll
                for (int j = 0; j < N; ++j) x[j] = Ty::down(v[j]);
                // (a gradient of this size is not read again from the caches: written past them)
                __builtin_nontemporal_store(*reinterpret_cast<const uint4v*>(x), reinterpret_cast<uint4v*>(to));
            } else if (n < past) {
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (inside(n, j)) to[j] = Ty::down(v[j]);
            }
        }
        if (W > 1) __syncthreads();   // the shared arrays are written again
    }
}

// A row a workgroup, read a second time for its gradient: rows whose registers would leave one workgroup on a CU, which
// cannot read the next row while it works on this one.  The second reading comes from the memory-side cache.  2000 rows of
// 200001 bfloat16: 516 us = 3.1 TB/s of the first reading and the writing.
template <class Ty, int T>
__global__ __launch_bounds__(T) void k_lp_twice(const typename Ty::S* __restrict__ z, int64_t rows, int64_t width, int64_t ld,
                                                typename Ty::A scale, LossOut<Ty> out) {
    using A = typename Ty::A;
    constexpr int W = T / 64;
    __shared__ Part<A> sp[W];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const typename Ty::S* zr = z + row * ld;
        const Piece<Ty> pc(zr, width);
        Pool<A> none(nullptr, 0);
        const Part<A> p = read_pieces<Ty, false>(zr, width, pc, wave * 64, pc.pieces, T, scale, none);
        if (lane == 0) sp[wave] = p;
        __syncthreads();
        int tg;
        Grad<A> w;
        const Row<A> r = out.row(row, zr, width, join_parts(sp, W, scale, lane), scale, threadIdx.x == 0, tg, w);
        write_slopes<Ty, T>(zr, out.dz + row * out.ld_dz, width, pc, threadIdx.x, pc.pieces, r, tg, w, scale);
        __syncthreads();   // the shared array is written again
    }
}

// ---- the chain into circuit parameters ------------------------------------------------------------------------------
// part[chunk][i] = sum over the chunk's samples b and observables o of d[b][o] (E[b][1 + 2 i][o] - E[b][2 + 2 i][o]):
// a lane a parameter (neighbouring lanes read neighbouring rows of the sweep), a wave a quarter of the chunk.
constexpr int kChainRows = 64;

__global__ __launch_bounds__(kT) void k_psr_chain(const double* __restrict__ e, int64_t B, int P, int n_obs,
                                                  const double* __restrict__ d, double* __restrict__ part) {
    __shared__ double sh[kWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t i = (int64_t)blockIdx.y * 64 + lane, K = 2 * (int64_t)P + 1;
    const int64_t b0 = (int64_t)blockIdx.x * kChainRows, b1 = min(B, b0 + kChainRows);
    double s = 0.0;
    if (i < P)
        for (int64_t b = b0 + wave; b < b1; b += kWaves) {
            const double* up = e + (b * K + 1 + 2 * i) * n_obs;
            const double* db = d + b * n_obs;
            for (int o = 0; o < n_obs; ++o) s += db[o] * (up[o] - up[n_obs + o]);
        }
    sh[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && i < P) part[blockIdx.x * (int64_t)P + i] = (sh[0][lane] + sh[1][lane]) + (sh[2][lane] + sh[3][lane]);
}
// 16 parameters a workgroup, the chunks over 64 threads each, added in a fixed order.  (65536 samples of 20 parameters and 3
// observables: 20 us for the parts, 64 MB at 3.2 TB/s, and 4.7 for their sum; with a thread a parameter the sum took 248.)
constexpr int kSumRows = 16, kSumParts = 64;
__global__ __launch_bounds__(kSumRows * kSumParts) void k_psr_chain_sum(const double* __restrict__ part, int64_t chunks, int P, double factor,
                                                                       double* __restrict__ out) {
    __shared__ double sh[kSumParts][kSumRows];
    const int x = threadIdx.x % kSumRows, y = threadIdx.x / kSumRows, i = blockIdx.x * kSumRows + x;
    double s = 0.0;
    if (i < P) {
#pragma unroll 8
        for (int64_t c = y; c < chunks; c += kSumParts) s += part[c * P + i];
    }
    sh[y][x] = s;
    __syncthreads();
#pragma unroll
    for (int n = kSumParts / 2; n; n /= 2) {
        if (y < n) sh[y][x] += sh[y + n][x];
        __syncthreads();
    }
    if (y == 0 && i < P) out[i] = factor * sh[0][x];
}

// ---- launches -----------------------------------------------------------------------------------------------------
constexpr int kLaneWidth = 64, kShortWidth = 1024;
constexpr int kWaveRows = 512, kWaveWidth = 8192;
// One workgroup a row needs rows enough for half of the CUs; of fewer rows the gradient is split, and reads them a second time.
constexpr int kWholeRows = 128;
constexpr int64_t kMaxGrid = 1 << 20;

// Parts of a row: enough workgroups for the chip (about 4 a CU) while a part keeps 4096 elements, at most one a lane of
// the joining wave.
int splits_of(int64_t rows, int64_t width) {
    int64_t s = (1024 + rows - 1) / rows;
    const int64_t most = width / 4096;
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : (s > 64 ? 64 : s));
}

bool wave_a_row(int64_t rows, int64_t width) { return width <= kShortWidth || (rows >= kWaveRows && width <= kWaveWidth); }
// Parts of a row whose states lie in the workspace, in the outputs alone and in the gradient; 0: the workspace is not touched.
// Both the size of the workspace and the launches go by this.
struct Dealt { int score, loss; };
Dealt dealt(int64_t rows, int64_t width) {
    const int splits = rows > 0 ? splits_of(rows, width) : 0;
    return { splits > 1 && !wave_a_row(rows, width) ? splits : 0, rows < kWholeRows && width > kShortWidth ? splits : 0 };
}

template <class Ty, bool kGrad>
void launch_short(hipStream_t st, const typename Ty::S* z, int64_t rows, int width, int64_t ld, double scale, const int32_t* target,
                  int top_k, const typename Ty::A* dg, const typename Ty::A* dh, typename Ty::A* lp, typename Ty::A* ent,
                  typename Ty::A* top_lp, int32_t* top_ix, typename Ty::S* dz, int64_t ld_dz) {
#define VQA_SHORT(G, E)                                                                                                      \
    hipLaunchKernelGGL((k_lp_short<Ty, G, E, kGrad>), dim3((unsigned)std::min<int64_t>(kMaxGrid, (rows + kT / G - 1) / (kT / G))), \
                       dim3(kT), 0, st, z, rows, width, ld, (typename Ty::A)scale, target, top_k, dg, dh, lp, ent, top_lp,   \
                       top_ix, dz, ld_dz)
    if (width <= 4) VQA_SHORT(4, 1);
    else if (width <= 16) VQA_SHORT(4, 4);
    else if (width <= 64) VQA_SHORT(16, 4);
    else if (width <= 256) VQA_SHORT(64, 4);
    else if constexpr (kGrad) VQA_SHORT(64, 16);
#undef VQA_SHORT
}

template <class A>
Ws<A> ws_of(void* p, int64_t parts) {
    return Ws<A>{ (Part<A>*)p, (Best<A>*)((char*)p + (parts * sizeof(Part<A>) + 15) / 16 * 16) };
}

template <class Ty>
int score(hipStream_t st, const void* z, int64_t rows, int64_t width, int64_t ld, double scale, const int32_t* target, int top_k,
          void* ws, void* lp, void* ent, void* top_lp, int32_t* top_ix) {
    using A = typename Ty::A;
    const auto* zz = (const typename Ty::S*)z;
    // A row in a part of a wave or with four elements a lane: registers alone, the best outcomes one by one, 5 us each for
    // 65536 rows;  else candidates are gathered.  65536 rows, us, so | the other way:  256 float32, top 4  57 | 51, none 30 | 35;
    // top 20  64 | 165;  400 float32, top 4  55 | 98;  1024 bfloat16, none  41 | 87.
    if (width <= kLaneWidth || (width <= 4 * kLaneWidth && top_k <= 4)) {
        launch_short<Ty, false>(st, zz, rows, (int)width, ld, scale, target, top_k, nullptr, nullptr, (A*)lp, (A*)ent, (A*)top_lp,
                                top_ix, nullptr, 0);
    } else {
        const Out<Ty> out = { target, (A*)lp, (A*)ent, (A*)top_lp, top_ix, top_k };
        if (wave_a_row(rows, width)) {
            const dim3 waves((unsigned)std::min<int64_t>(kMaxGrid, (rows + kWaves - 1) / kWaves));
            if (top_k > 0) hipLaunchKernelGGL((k_lp_wave<Ty, true>), waves, dim3(kT), 0, st, zz, rows, width, ld, (A)scale, top_k, out);
            else hipLaunchKernelGGL((k_lp_wave<Ty, false>), waves, dim3(kT), 0, st, zz, rows, width, ld, (A)scale, top_k, out);
            VQA_HIP(hipGetLastError());
            return VQA_OK;
        }
        const int splits = std::max(1, dealt(rows, width).score);
        if (splits > 1 && !ws) VQA_FAIL(VQA_EINVAL, "workspace is NULL");
        const Ws<A> w = splits > 1 ? ws_of<A>(ws, rows * splits) : Ws<A>{ nullptr, nullptr };
        const dim3 grid((unsigned)std::min<int64_t>(kMaxGrid, rows * splits)), grid2((unsigned)std::min<int64_t>(kMaxGrid, rows));
        if (top_k > 0) hipLaunchKernelGGL((k_lp_parts<Ty, true>), grid, dim3(kT), 0, st, zz, rows, width, ld, (A)scale, top_k, splits, w, out);
        else hipLaunchKernelGGL((k_lp_parts<Ty, false>), grid, dim3(kT), 0, st, zz, rows, width, ld, (A)scale, top_k, splits, w, out);
        if (splits > 1) hipLaunchKernelGGL((k_lp_join<Ty>), grid2, dim3(64), 0, st, zz, rows, width, ld, (A)scale, top_k, splits, w, out);
    }
    VQA_HIP(hipGetLastError());
    return VQA_OK;
}

template <class Ty>
int loss(hipStream_t st, const void* z, int64_t rows, int64_t width, int64_t ld, double scale, const int32_t* target, const void* dg,
         const void* dh, void* ws, void* lp, void* ent, void* dz, int64_t ld_dz) {
    using A = typename Ty::A;
    using S = typename Ty::S;
    const auto* zz = (const S*)z;
    if (width <= kShortWidth) {
        launch_short<Ty, true>(st, zz, rows, (int)width, ld, scale, target, 0, (const A*)dg, (const A*)dh, (A*)lp, (A*)ent, nullptr,
                               nullptr, (S*)dz, ld_dz);
        VQA_HIP(hipGetLastError());
        return VQA_OK;
    }
    const LossOut<Ty> out = { target, (const A*)dg, (const A*)dh, (A*)lp, (A*)ent, (S*)dz, ld_dz };
    const int64_t pieces = (width + 2 * Piece<Ty>::N - 2) / Piece<Ty>::N;    // of a row that begins anywhere
    const dim3 grid((unsigned)std::min<int64_t>(kMaxGrid, rows));
    const int splits = dealt(rows, width).loss;
    if (!splits) {
        if (pieces <= 8 * 64) hipLaunchKernelGGL((k_lp_loss<Ty, 64, 8>), grid, dim3(64), 0, st, zz, rows, width, ld, (A)scale, out);
        else if (pieces <= 16 * 64) hipLaunchKernelGGL((k_lp_loss<Ty, 64, 16>), grid, dim3(64), 0, st, zz, rows, width, ld, (A)scale, out);
        else if (pieces <= 16 * 256) hipLaunchKernelGGL((k_lp_loss<Ty, 256, 16>), grid, dim3(256), 0, st, zz, rows, width, ld, (A)scale, out);
        else if (pieces <= 16 * 512) hipLaunchKernelGGL((k_lp_loss<Ty, 512, 16>), grid, dim3(512), 0, st, zz, rows, width, ld, (A)scale, out);
        else hipLaunchKernelGGL((k_lp_twice<Ty, 512>), grid, dim3(512), 0, st, zz, rows, width, ld, (A)scale, out);
    } else {
        if (!ws) VQA_FAIL(VQA_EINVAL, "workspace is NULL");
        const Ws<A> w = ws_of<A>(ws, rows * splits);
        const dim3 all((unsigned)std::min<int64_t>(kMaxGrid, rows * splits));
        hipLaunchKernelGGL((k_lp_parts<Ty, false>), all, dim3(kT), 0, st, zz, rows, width, ld, (A)scale, 0, splits, w, Out<Ty>{});
        hipLaunchKernelGGL((k_lp_slope<Ty>), all, dim3(kT), 0, st, zz, rows, width, ld, (A)scale, splits, w, out);
    }
    VQA_HIP(hipGetLastError());
    return VQA_OK;
}

}  // namespace

size_t log_probs_workspace_bytes(int dtype, int64_t rows, int64_t width, int top_k) {
    const Dealt d = dealt(rows, width);
    const size_t parts = (size_t)std::max<int64_t>(rows, 0) * std::max(d.score, d.loss);
    const bool wide = dtype == VQA_DTYPE_F64;
    return (parts * (wide ? sizeof(Part<double>) : sizeof(Part<float>)) + 15) / 16 * 16 +
           (size_t)std::max<int64_t>(rows, 0) * d.score * top_k * (wide ? sizeof(Best<double>) : sizeof(Best<float>));
}

int log_probs_launch(hipStream_t st, int dtype, const void* z, int64_t rows, int64_t width, int64_t ld, double scale,
                     const int32_t* target, int top_k, void* ws, void* lp, void* ent, void* top_lp, int32_t* top_ix) {
    switch (dtype) {
        case VQA_DTYPE_F64: return score<F64>(st, z, rows, width, ld, scale, target, top_k, ws, lp, ent, top_lp, top_ix);
        case VQA_DTYPE_F32: return score<F32>(st, z, rows, width, ld, scale, target, top_k, ws, lp, ent, top_lp, top_ix);
        case VQA_DTYPE_BF16: return score<BF16>(st, z, rows, width, ld, scale, target, top_k, ws, lp, ent, top_lp, top_ix);
        default: return score<F16>(st, z, rows, width, ld, scale, target, top_k, ws, lp, ent, top_lp, top_ix);
    }
}

int log_probs_grad_launch(hipStream_t st, int dtype, const void* z, int64_t rows, int64_t width, int64_t ld, double scale,
                          const int32_t* target, const void* dg, const void* dh, void* ws, void* lp, void* ent, void* dz,
                          int64_t ld_dz) {
    switch (dtype) {
        case VQA_DTYPE_F64: return loss<F64>(st, z, rows, width, ld, scale, target, dg, dh, ws, lp, ent, dz, ld_dz);
        case VQA_DTYPE_F32: return loss<F32>(st, z, rows, width, ld, scale, target, dg, dh, ws, lp, ent, dz, ld_dz);
        case VQA_DTYPE_BF16: return loss<BF16>(st, z, rows, width, ld, scale, target, dg, dh, ws, lp, ent, dz, ld_dz);
        default: return loss<F16>(st, z, rows, width, ld, scale, target, dg, dh, ws, lp, ent, dz, ld_dz);
    }
}

size_t psr_chain_workspace_bytes(int64_t B, int P) { return (size_t)((B + kChainRows - 1) / kChainRows) * P * 8; }

int psr_chain_launch(hipStream_t st, const double* e, int64_t B, int P, int n_obs, double factor, const double* d, double* ws,
                     double* out) {
    const int64_t chunks = (B + kChainRows - 1) / kChainRows;
    if (chunks > 0)
        hipLaunchKernelGGL(k_psr_chain, dim3((unsigned)chunks, (unsigned)((P + 63) / 64)), dim3(kT), 0, st, e, B, P, n_obs, d, ws);
    hipLaunchKernelGGL(k_psr_chain_sum, dim3((unsigned)((P + kSumRows - 1) / kSumRows)), dim3(kSumRows * kSumParts), 0, st, ws, chunks, P, factor, out);
    VQA_HIP(hipGetLastError());
    return VQA_OK;
}

}  // namespace vqa
