// Shared device code of the losses over a K x N matrix of logits (one token per
// column): log-probabilities, policy, preference and distillation losses.
//
// For a column x with maximum m:  t_i = x_i - m,  e_i = exp(t_i/T),  s = sum e_i,
// p_i = e_i/s.  The shift makes every exponent <= 0, so s is in [1, K] and nothing
// overflows.  Each kernel hands a column to a team of threads; a `Head` turns (m, s, ...)
// into the coefficients of the gradient,
//     d_i = e_i * (a + b*t_i)  (+ corrections at the label or the teacher's entries).
// What a team keeps in registers between the reductions is read once: a column of up to 4096
// logits, and up to 65536 where there are at most two columns per CU.  With more columns a team
// keeps 4096 (K up to 8192), 8192 (to 16384), 16384 (to 28672), all (to 32768) or 32768 logits
// (to 65536), beyond that, and for any number of columns, 65536; the rest is read a second time
// for the gradient, its last part first, as much of it out of the caches as fits there.  Columns
// cut into chunks are read twice in full.  What bounds all of them is memory: 8 bytes per logit,
// up to 12 with the second read, against about a dozen vector instructions.
//
// Accuracy: a thread adds sixteen exponentials in fp32 and everything further in 64 bits.  Those
// that are 1 are counted apart: where one logit stands out, what the others add to its 1 is what
// log s is made of, and fp32 would round it at 2^-24, a few 1e-8 per token that show in the
// log-probability of a likely token and in sums of small differences of them (reading alone of
// 512 MB less a quarter 61 -> 63 us, 5000 logits a column 52 -> 54.5; beside a gradient under 1 %).
// What happens once per column (log s, ratios, divergences) is done in 64 bits too.
#pragma once

#include "common.hpp"

#include <cmath>
#include <mutex>
#include <type_traits>

namespace jz {

// log2(e)/T as a sum of two floats, the second one positive
struct ExpScale {
    float hi, lo;
};
inline ExpScale exp_scale(double temperature) {
    const double c = 1.44269504088896340736 / temperature;
    ExpScale r;
    r.hi = static_cast<float>(c);
    if (static_cast<double>(r.hi) >= c) r.hi = std::nextafterf(r.hi, 0.0f);
    r.lo = static_cast<float>(c - static_cast<double>(r.hi));
    return r;
}

// exp(d/T) for d <= 0: the hardware's 2^u (0.7 ulp, mean error kExpShort; an exact 0 below
// 2^-126) of u = d*log2(e)/T rounded once.  The low part of the constant is what keeps
// the result without bias (-1.3e-8 * u otherwise); it is positive, so that d = -inf
// gives -inf - inf and 0.  A NaN stays one.
// What the hardware's 2^u falls short of on average (over u in [-1, 0], [-8, 0] and [-40, 0] alike,
// but for the exact 1 at 0): sums put it back.
constexpr double kExpShort = 3.4e-9;
__device__ __forceinline__ float exp_shifted(float d, const ExpScale& c) {
    return __builtin_amdgcn_exp2f(fmaf(d, c.hi, d * c.lo));
}

// ── scalars of a column, 64 bits ─────────────────────────────────────────
// Every wave that owns a column evaluates these once, and beside 16 to 64 exponentials per
// lane their length counts: the general library functions took longer than a column of
// 1024 logits.  Errors stay below 1e-10 relative, a thousandth of what the sums carry.

// log(v), v >= 0: v = f * 2^k with f in [1/sqrt 2, sqrt 2), log f = 2 atanh z,
// z = (f-1)/(f+1), |z| < 0.172; the series in z^2 is cut after z^13/13.
__device__ __forceinline__ double log64(double v) {
    double f = __builtin_amdgcn_frexp_mant(v);   // in [1/2, 1)
    int k = __builtin_amdgcn_frexp_exp(v);
    const bool low = f < 0.70710678118654752;
    f = low ? 2.0 * f : f;
    k = low ? k - 1 : k;
    const double z = (f - 1.0) / (f + 1.0), w = z * z;
    double p = 1.0 / 13.0;
    p = fma(p, w, 1.0 / 11.0);
    p = fma(p, w, 1.0 / 9.0);
    p = fma(p, w, 1.0 / 7.0);
    p = fma(p, w, 1.0 / 5.0);
    p = fma(p, w, 1.0 / 3.0);
    p = fma(p, w, 1.0);
    const double r = fma(static_cast<double>(k), 0.69314718055994531, 2.0 * z * p);
    return v == 0.0 ? -INFINITY : v == INFINITY ? v : r;
}
// exp(v): n = rint(v/ln 2), the Taylor series of exp(v - n ln 2) up to the tenth power
// (|r| <= 0.347: 0.347^11/11! = 2e-13).  The reduction is Cody and Waite's: ln 2 as its first
// 32 bits, whose product with n is exact, and what they leave.
__device__ __forceinline__ double exp64(double v) {
    const double n = rint(v * 1.44269504088896340736);
    const double r = fma(n, -1.90821492927058770e-10, fma(n, -0.693147180369123816490, v));
    double p = 1.0 / 3628800.0;
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    p = __builtin_amdgcn_ldexp(p, static_cast<int>(n));
    return v < -700.0 ? 0.0 : v > 709.0 ? INFINITY : p;
}
// exp(v) - 1 and exp(v) - 1 - v; near 0, where the differences would cancel, from the series
// (|v| < 0.06, cut after v^8/8!: 0.06^7 / 9! * 2 = 1e-14).
struct ExpTail {
    double minus1, tail;
};
__device__ __forceinline__ ExpTail exp_tail64(double v) {
    double p = 1.0 / 40320.0;
    p = fma(p, v, 1.0 / 5040.0);
    p = fma(p, v, 1.0 / 720.0);
    p = fma(p, v, 1.0 / 120.0);
    p = fma(p, v, 1.0 / 24.0);
    p = fma(p, v, 1.0 / 6.0);
    p = fma(p, v, 0.5) * v * v;
    const double e = exp64(v) - 1.0;
    if (fabs(v) < 0.06) return ExpTail{p + v, p};
    return ExpTail{e, v > 709.0 ? INFINITY : e - v};
}

struct AddOp {
    template <class T>
    __device__ __forceinline__ T operator()(T a, T b) const { return a + b; }
};
struct LargerOp {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};

template <int CTRL>
__device__ __forceinline__ double dpp_mov(double v) {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
    const unsigned lo = static_cast<unsigned>(b), hi = static_cast<unsigned>(b >> 32);
    const unsigned l = static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(lo), CTRL, 0xF, 0xF, true));
    const unsigned h = static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(hi), CTRL, 0xF, 0xF, true));
    return __builtin_bit_cast(double, (static_cast<unsigned long long>(h) << 32) | l);
}

// The threads that share one column: G lanes of a wave (G = 4 ... 64) or a whole
// workgroup of G threads.  Reductions run in one fixed order and leave the result in
// every thread.
template <int G>
struct Team {
    static constexpr int kSize = G;
    static constexpr int kWaves = G > kWave ? G / kWave : 1;
    static constexpr bool kWorkgroup = kWaves > 1;
    static constexpr int kLanes = G < kWave ? G : kWave;   // of one wave
    int rank;

    // over the team's lanes of one wave
    template <class T, class Op>
    __device__ __forceinline__ T lanes(T v, Op op) const {
        v = op(v, dpp_mov<0xB1>(v));                               // quad_perm [1,0,3,2]
        v = op(v, dpp_mov<0x4E>(v));                               // quad_perm [2,3,0,1]
        if constexpr (kLanes >= 8) v = op(v, dpp_mov<0x141>(v));   // row_half_mirror
        if constexpr (kLanes >= 16) v = op(v, dpp_mov<0x140>(v));  // row_mirror
        if constexpr (kLanes >= 32) v = op(v, __shfl_xor(v, 16, kWave));
        if constexpr (kLanes >= 64) v = op(v, __shfl_xor(v, 32, kWave));
        return v;
    }
    // over the team; `slots`: kWaves values in LDS that nothing else uses before the next barrier
    template <class T, class Op>
    __device__ __forceinline__ T reduce(T v, Op op, T* slots) const {
        v = lanes(v, op);
        if constexpr (kWorkgroup) {
            if ((rank & (kWave - 1)) == 0) slots[rank / kWave] = v;
            __syncthreads();
            v = slots[0];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) v = op(v, slots[w]);
        }
        return v;
    }
    // LDS and global writes of the team before it are seen after it.  Lanes of one wave run
    // in step: there it only keeps the compiler from moving memory operations across.
    __device__ __forceinline__ void sync() const {
        if constexpr (kWorkgroup) {
            __syncthreads();
        } else {
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
    }
    // What is done once per column is done by the first wave of a workgroup; by every lane of
    // a smaller team, whose wave issues it anyway.
    __device__ __forceinline__ bool leads() const { return !kWorkgroup || rank < kWave; }
    __device__ __forceinline__ Team<kLanes> lead() const { return Team<kLanes>{rank}; }
};

// What one sweep over a column leaves: its maximum, the sum of e_i and of e_i*t_i (heads
// that ask for the entropy).  Heads that ask for the rest (kRest) sweep over the logits that are
// none of the teacher's entries, with a maximum of their own, and add the entries themselves.
struct ColumnSums {
    float m;
    double s, et;
};
// Something is left but masked logits: a number, or a NaN.
__device__ __forceinline__ bool unmasked(float m, double s) { return !(m == -INFINITY && s == s); }
// d_i = e_i * (a + b*t_i); g is added at the label, whose logit is x.  (A head without the entropy
// has b for itself.)
struct Grad {
    float a, b, g, x;
};

__device__ __forceinline__ bool label_scored(int label, int K) { return label >= 0 && label < K; }

// log softmax of the value `x` of a column
__device__ __forceinline__ double log_prob(float x, const ColumnSums& c) {
    return (static_cast<double>(x) - static_cast<double>(c.m)) - log64(c.s);
}
__device__ __forceinline__ double entropy_of(const ColumnSums& c) { return log64(c.s) - c.et / c.s; }

template <bool LINEAR>
__device__ __forceinline__ float grad_value(float t, float e, float a, float b) {
    // (a shift of -inf goes with an exponential of 0)
    if constexpr (LINEAR) return e * (a + b * fmaxf(t, -200.f));
    else return e * a;
}

// Four consecutive logits.  Columns start at any multiple of ld, so an address is only known
// to be a multiple of 4 bytes; the hardware takes a 16-byte access at any of them.
typedef float Quad __attribute__((ext_vector_type(4), aligned(4)));

// A run of logits as `quads` quads from element `skew` on, 16-byte aligned at the address they are
// laid out for, and `odd` single ones in front and behind (six at most).
struct Span {
    int skew, quads, odd;
    __device__ __forceinline__ int single(int r) const { return r < skew ? r : 4 * quads + r; }
};
// ALIGN: an odd leading dimension costs a wave's 1 KB access a ninth cache line otherwise.
template <bool ALIGN>
__device__ __forceinline__ Span span_of(const float* p, int len) {
    int skew = ALIGN ? static_cast<int>((4 - (reinterpret_cast<uintptr_t>(p) >> 2)) & 3) : 0;
    skew = skew < len ? skew : len;
    const int quads = (len - skew) / 4;
    return Span{skew, quads, len - 4 * quads};
}

// Which logits of a column belong to the teacher's entries: one bit each (one word more than
// the last logit's is there).
__device__ __forceinline__ unsigned known_quad(const unsigned* bits, int i) {
    return __builtin_amdgcn_alignbit(bits[(i >> 5) + 1], bits[i >> 5], i & 31) & 15u;
}
__device__ __forceinline__ bool known_one(const unsigned* bits, int i) { return (bits[i >> 5] >> (i & 31)) & 1u; }

template <bool NT>
__device__ __forceinline__ Quad load_quad(const float* p) {
    if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const Quad*>(p));
    else return *reinterpret_cast<const Quad*>(p);
}
template <bool NT>
__device__ __forceinline__ void store_quad(float* p, const Quad& v) {
    if constexpr (NT) __builtin_nontemporal_store(v, reinterpret_cast<Quad*>(p));
    else *reinterpret_cast<Quad*>(p) = v;
}
// The largest number of three.  (fmaxf first quiets each operand that comes from memory, an instruction per
// logit: reading alone at 8000 logits a column 65 us with it, 63.5 without.)
__device__ __forceinline__ float max_of(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ float max_of(const Quad& a, const Quad& b, const Quad& c, const Quad& d) {
    const float l = max_of(max_of(a.x, a.y, a.z), max_of(a.w, b.x, b.y), max_of(b.z, b.w, c.x));
    const float r = max_of(max_of(c.y, c.z, c.w), max_of(d.x, d.y, d.z), d.w);
    return max_of(l, r, r);
}

// Sums of a group of quads relative to the group's own maximum.  A thread forms them while
// the quads behind are still on their way: exponentials need no maximum of the whole column,
// only a factor exp(m_group - m) once that is known.
constexpr int kGroupQuads = 4;
struct Group {
    float m, s, ones, et;   // s: of the exponentials below 1; ones: how many are 1
};
// x: the group's logits; without the entropy they become e_i relative to the group.  known(k): the
// teacher's entries among quad k, which do not count.
template <class Head, class Known>
__device__ __forceinline__ Group take_group(Quad (&x)[kGroupQuads], const ExpScale& scale, Known known) {
    Group g{-INFINITY, 0.f, 0.f, 0.f};
    if constexpr (Head::kRest) {
#pragma unroll
        for (int k = 0; k < kGroupQuads; ++k) {
            const unsigned b = known(k);
            x[k] = Quad{b & 1u ? -INFINITY : x[k].x, b & 2u ? -INFINITY : x[k].y, b & 4u ? -INFINITY : x[k].z,
                        b & 8u ? -INFINITY : x[k].w};
        }
    }
    static_assert(kGroupQuads == 4, "max_of");
    g.m = max_of(x[0], x[1], x[2], x[3]);
    const float shift = g.m == -INFINITY ? 0.f : g.m;   // nothing but -inf: sums of 0; a NaN still shows
    float s[kGroupQuads], all[kGroupQuads], et[kGroupQuads];
#pragma unroll
    for (int k = 0; k < kGroupQuads; ++k) {
        const float t0 = x[k].x - shift, t1 = x[k].y - shift, t2 = x[k].z - shift, t3 = x[k].w - shift;
        const float e0 = exp_shifted(t0, scale), e1 = exp_shifted(t1, scale);
        const float e2 = exp_shifted(t2, scale), e3 = exp_shifted(t3, scale);
        all[k] = (e0 + e1) + (e2 + e3);
        s[k] = (__builtin_amdgcn_fractf(e0) + __builtin_amdgcn_fractf(e1)) +   // (below 1: its own fraction)
               (__builtin_amdgcn_fractf(e2) + __builtin_amdgcn_fractf(e3));
        if constexpr (Head::kEntropy)
            et[k] = fmaf(e3, fmaxf(t3, -200.f), fmaf(e2, fmaxf(t2, -200.f), fmaf(e1, fmaxf(t1, -200.f), e0 * fmaxf(t0, -200.f))));
        else
            x[k] = Quad{e0, e1, e2, e3};
    }
    g.s = (s[0] + s[1]) + (s[2] + s[3]);
    g.ones = rintf(((all[0] + all[1]) + (all[2] + all[3])) - g.s);
    if constexpr (Head::kEntropy) g.et = (et[0] + et[1]) + (et[2] + et[3]);
    return g;
}
// Joins sums relative to two maxima (the shift of sums of nothing but -inf is 0: they are 0, or
// NaN, and stay so).
template <class Head>
__device__ __forceinline__ void scale_sums(ColumnSums& c, float m, const ExpScale& scale) {
    if (m == -INFINITY) return;
    const float t = c.m - m;
    const double f = t == 0.f ? 1.0 : static_cast<double>(exp_shifted(t, scale)) * (1.0 + kExpShort);
    if constexpr (Head::kEntropy) c.et = (c.et + c.s * static_cast<double>(fmaxf(t, -200.f))) * f;
    c.s *= f;
    c.m = m;
}
__device__ __forceinline__ ColumnSums sums_of(const Group& g) {
    return ColumnSums{g.m, static_cast<double>(g.ones) + static_cast<double>(g.s) * (1.0 + kExpShort), static_cast<double>(g.et)};
}
template <class Head>
__device__ __forceinline__ void add_group(ColumnSums& c, const Group& g, const ExpScale& scale) {
    ColumnSums more = sums_of(g);
    const float m = fmaxf(c.m, g.m);
    scale_sums<Head>(c, m, scale);
    scale_sums<Head>(more, m, scale);
    c.s += more.s;
    if constexpr (Head::kEntropy) c.et += more.et;
}
// of a single logit
__device__ __forceinline__ Group take_one(float x) {
    const float e = x == -INFINITY ? 0.f : x - x + 1.f;   // exp of its shift from itself; a NaN or +inf shows
    return Group{x, 0.f, e, 0.f};
}

// The compiler would interleave the independent work of an unrolled loop and spill what it
// thereby has live; where a thread holds many quads it is kept in order.
template <int NV>
__device__ __forceinline__ void in_order() {
    if constexpr (NV > kGroupQuads) __builtin_amdgcn_sched_barrier(0);
}

// The label's element, behind the sweep that wrote it as any other: after a team.sync(), by one thread.
template <bool LINEAR>
__device__ __forceinline__ void correct_label(int label, float m, const Grad& f, const ExpScale& scale, float* out) {
    const float t = f.x - m;
    out[label] = grad_value<LINEAR>(t, exp_shifted(t, scale), f.a, f.b) + f.g;
}

// Where the quads of a tile lie: up to NV per thread from quad `base` on.  STRETCH: those of a
// wave are one stretch of memory, which suits the writing sweep (one read and one write of
// 512 MB each: 182 us, 193 with a wave that strides by the workgroup's width) and not reading
// alone (512 MB less a quarter: 69 us against 66).
template <int G, int NV, bool STRETCH>
struct Tile {
    int first, count;
    static constexpr int kLanes = Team<G>::kLanes;
    __device__ __forceinline__ Tile(int rank, int base, int quads) {
        const int n = (quads - base + G - 1) / G;
        count = n < NV ? n : NV;
        first = base + (STRETCH ? rank / kLanes * kLanes * count + rank % kLanes : rank);
    }
    __device__ __forceinline__ int at(int k) const { return first + k * (STRETCH ? kLanes : G); }
    __device__ __forceinline__ bool has(int k, int quads) const { return k < count && at(k) < quads; }
};

template <int G>
struct ColumnShared {
    float max[Team<G>::kWaves];
    double s[Team<G>::kWaves], other[Team<G>::kWaves];
    Grad grad;
    int live;   // 2: also if nothing but the teacher's entries is left
};

// One column by one team: NV quads per thread in registers, what is beyond them (STREAM) in tiles
// of the same size that are read again for the gradient, the last one first: they come out of the
// caches as long as the columns under way fit there.
//   own: head.team_bytes(K) of LDS
template <class Head, int G, int NV, bool NT, bool STREAM>
__device__ __forceinline__ void token_column(const Head& head, const Team<G>& team, ColumnShared<G>& sh, char* own,
                                             size_t col, float* out, const float* p, int K) {
    static_assert(NV % kGroupQuads == 0, "whole groups");
    constexpr int kGroups = NV / kGroupQuads, kTile = NV * G;
    constexpr bool kKeepMax = Head::kWrites && !Head::kEntropy;   // the kept exponentials are relative to it
    const Span span = span_of<(G > 4)>(p, K);   // (by the logits: values are the same bits with and without a gradient)
    const float* const body = p + span.skew;
    using ColumnTile = Tile<G, NV, Head::kWrites>;
    const ColumnTile mine(team.rank, 0, span.quads);
    bool live = head.live(col, K);
    Quad v[kGroups][kGroupQuads];
    float group_max[kGroups];
    float last = -INFINITY;
    ColumnSums c{-INFINITY, 0.0, 0.0};
    typename Head::Early early{};
    if (live) {
        const unsigned* bits = nullptr;
        auto take = [&](Quad (&x)[kGroupQuads], const ColumnTile& tile, int first, bool only) {
            const Group g = take_group<Head>(x, head.scale, [&](int k) {
                const int q = tile.at(first + k);
                return known_quad(bits, span.skew + 4 * (q < span.quads ? q : 0));   // (nothing counts behind the column)
            });
            if (only) {   // the first one
                c = sums_of(g);
                c.m = fmaxf(g.m, -INFINITY);   // (of nothing but NaN: none)
            } else {
                add_group<Head>(c, g, head.scale);
            }
            return g.m;
        };
        // The teacher's part is the first wave's and runs while the loads of the others are under
        // way; where few registers hold the column, behind the team's own.
        constexpr bool kTeacherFirst = Team<G>::kWorkgroup || NV > 2 * kGroupQuads;
        auto teach = [&] {
            if constexpr (Head::kTeacher) {
                unsigned* marks = head.bits(own);
                for (int i = team.rank; i < (K + 31) / 32; i += G) marks[i] = 0u;
                team.sync();
                if (!team.leads()) return;
                const bool some = head.prologue(team.lead(), own, marks, col, K, p, early);
                if constexpr (Team<G>::kWorkgroup) {
                    if (team.rank == 0) sh.live = some ? 1 + unmasked(early.m, early.s) : 0;
                } else {
                    live = some;
                }
            }
        };
        early = head.early(col, p);
        if constexpr (Head::kTeacher && kTeacherFirst) teach();
        // the entries are marked: waited for behind the first loads
        auto marked = [&] {
            if constexpr (Head::kRest) {
                if (!bits) team.sync();
                bits = head.bits(own);
            }
        };
        auto load = [&](const ColumnTile& tile, auto cached) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                Quad& x = v[k / kGroupQuads][k % kGroupQuads];
                x = Quad(-INFINITY);
                if (tile.has(k, span.quads)) x = load_quad<NT && !decltype(cached)::value>(body + 4 * static_cast<size_t>(tile.at(k)));
            }
        };
        if constexpr (STREAM) {
            for (int base = kTile; base < span.quads; base += kTile) {
                const ColumnTile tile(team.rank, base, span.quads);
                load(tile, std::bool_constant<Head::kWrites>{});   // read again later
                marked();
#pragma unroll
                for (int i = 0; i < kGroups; ++i) {
                    take(v[i], tile, i * kGroupQuads, false);
                    in_order<NV>();
                }
            }
        }
        load(mine, std::false_type{});
        if (team.rank < span.odd) last = p[span.single(team.rank)];
        if constexpr (Head::kTeacher && !kTeacherFirst) teach();
        marked();
#pragma unroll
        for (int i = 0; i < kGroups; ++i) {
            const float m = take(v[i], mine, i * kGroupQuads, !STREAM && i == 0);
            if constexpr (kKeepMax) group_max[i] = m;
            in_order<NV>();
        }
        if (team.rank < span.odd) {
            if constexpr (Head::kRest)
                if (known_one(bits, span.single(team.rank))) last = -INFINITY;
            add_group<Head>(c, take_one(last), head.scale);
        }
        scale_sums<Head>(c, team.reduce(c.m, LargerOp{}, sh.max), head.scale);
        bool filled = false;   // an entry that is not masked
        if constexpr (Head::kTeacher) {
            filled = unmasked(early.m, early.s);
            if constexpr (Team<G>::kWorkgroup) {   // behind that barrier
                live = sh.live != 0;
                filled = sh.live == 2;
            }
        }
        if constexpr (Head::kEntropy) {
            c.et = team.lanes(c.et, AddOp{});
            if constexpr (Team<G>::kWorkgroup)
                if ((team.rank & (kWave - 1)) == 0) sh.other[team.rank / kWave] = c.et;
            c.s = team.reduce(c.s, AddOp{}, sh.s);
            if constexpr (Team<G>::kWorkgroup) {
                c.et = sh.other[0];
#pragma unroll
                for (int k = 1; k < Team<G>::kWaves; ++k) c.et += sh.other[k];
            }
        } else {
            c.s = team.reduce(c.s, AddOp{}, sh.s);
        }
        live = live && (filled || unmasked(c.m, c.s));
    }
    if (!live) {
        if (team.rank == 0) head.idle(col);
        if (Head::kWrites && out) {
            for (int q = team.rank; q < span.quads; q += G) store_quad<NT>(out + span.skew + 4 * static_cast<size_t>(q), Quad(0.f));
            if (team.rank < span.odd) out[span.single(team.rank)] = 0.f;
        }
        return;
    }
    Grad f{};
    if (team.leads()) f = head.finish(team.lead(), own, early, col, c);
    if (!Head::kWrites || !out) return;
    if constexpr (Team<G>::kWorkgroup) {
        if (team.rank == 0) sh.grad = f;
        __syncthreads();
        f = sh.grad;
    }
    float* const to = out + span.skew;
    // No maximum: in the rest alone, whose exponentials are 0 then; else the column holds a NaN, and f.a is one.
    const float shift = Head::kRest && c.m == -INFINITY ? 0.f : c.m;
    auto value = [&](float x) {   // (at an entry of the rest anything: its own gradient comes behind)
        const float t = x - shift;
        return grad_value<Head::kEntropy>(t, exp_shifted(t, head.scale), f.a, f.b);
    };
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
        float scale = 0.f;
        if constexpr (kKeepMax) scale = exp_shifted(group_max[i] - shift, head.scale) * f.a;
#pragma unroll
        for (int k = 0; k < kGroupQuads; ++k) {
            const Quad x = v[i][k];
            if (!mine.has(i * kGroupQuads + k, span.quads)) continue;
            Quad r;
            if constexpr (Head::kEntropy) r = Quad{value(x.x), value(x.y), value(x.z), value(x.w)};   // x: logits
            else r = Quad{x.x * scale, x.y * scale, x.z * scale, x.w * scale};
            store_quad<NT>(to + 4 * static_cast<size_t>(mine.at(i * kGroupQuads + k)), r);
        }
        in_order<NV>();
    }
    if (team.rank < span.odd) out[span.single(team.rank)] = value(last);
    if constexpr (STREAM) {
        constexpr int kQuads = NV % 8 == 0 ? 8 : 4, kStep = kQuads * G;   // whole steps to a tile
        for (int base = (span.quads - 1) / kStep * kStep; base >= kTile; base -= kStep) {
            const Tile<G, kQuads, true> tile(team.rank, base, span.quads);
            Quad x[kQuads];
#pragma unroll
            for (int k = 0; k < kQuads; ++k) {
                x[k] = Quad(0.f);
                if (tile.has(k, span.quads)) x[k] = load_quad<NT>(body + 4 * static_cast<size_t>(tile.at(k)));
            }
#pragma unroll
            for (int k = 0; k < kQuads; ++k) {
                const Quad r{value(x[k].x), value(x[k].y), value(x[k].z), value(x[k].w)};
                if (tile.has(k, span.quads)) store_quad<NT>(to + 4 * static_cast<size_t>(tile.at(k)), r);
            }
        }
    }
    team.sync();   // behind the sweep that wrote these elements as any other
    if (team.leads()) head.correct(team.lead(), own, col, shift, f, out);
}

// *out = scale * sum of p[0 ... n) by a wave or a workgroup of BLOCK threads, in 64 bits in a fixed order.
template <int BLOCK>
__device__ __forceinline__ void fold_parts(float* out, const double* p, int n, double scale, double* slots) {
    const Team<BLOCK> team{static_cast<int>(threadIdx.x % BLOCK)};
    double a0 = 0.0, a1 = 0.0, a2 = 0.0, a3 = 0.0;
    int i = team.rank;
    for (; i + 3 * BLOCK < n; i += 4 * BLOCK) {
        const double x0 = p[i], x1 = p[i + BLOCK], x2 = p[i + 2 * BLOCK], x3 = p[i + 3 * BLOCK];
        a0 += x0; a1 += x1;
        a2 += x2; a3 += x3;
    }
    for (; i < n; i += BLOCK) a0 += p[i];
    a0 = team.reduce((a0 + a1) + (a2 + a3), AddOp{}, slots);
    if (team.rank == 0) *out = static_cast<float>(scale * a0);
}
constexpr int kFoldBlock = 1024;
template <int BLOCK>
__global__ __launch_bounds__(BLOCK) void token_fold_kernel(float* out, const double* part, int n, size_t stride, double scale) {
    __shared__ double slots[BLOCK / kWave];
    fold_parts<BLOCK>(out + blockIdx.x, part + blockIdx.x * stride, n, scale, slots);
}

// The sums over tokens of an entry point: out[k] = sum of part[k*N ...], k < count.  Parts have 64 bits: with
// centred advantages or weights of both signs a loss is a small difference of them.
struct TokenSums {
    float* out;
    double* part;
    int count;
};
// Where a head leaves its columns' parts: sum k of column n at part[k*stride + n - first].
struct TokenParts {
    double* part;
    size_t stride, first = 0;
    __device__ __forceinline__ double& at(size_t col, int k) const { return part[static_cast<size_t>(k) * stride + (col - first)]; }
};

//   dynamic LDS: head.team_bytes(K) per team
//   FOLD: a single workgroup holds all columns, and its sums are the call's
// Where a workgroup has several columns it leaves one part per sum (policy loss of 16384 columns of 256: 11.2 us, with
// a part per column 12.3, as 64-bit parts are 128 KB a sum to one workgroup; of 1000 24.1 and 26.3).
template <class Head, int G, int NV, int BLOCK, bool NT, bool STREAM, bool FOLD>
__global__ __launch_bounds__(BLOCK, 4) void token_column_kernel(Head head, TokenSums sums, float* d, const float* x,
                                                                int K, int N, size_t ld, size_t ldd) {
    constexpr int kTeams = BLOCK / G;
    constexpr bool kJoin = kTeams > 1 && Head::kSums > 0;
    static_assert(!kJoin || Head::kSums <= BLOCK / kWave, "a wave per sum");
    __shared__ ColumnShared<G> shared;
    __shared__ double parts[kJoin ? Head::kSums * kTeams : 1];
    extern __shared__ __align__(16) char dynamic[];
    const Team<G> team{static_cast<int>(kTeams > 1 ? threadIdx.x % G : threadIdx.x)};
    int slot = kTeams > 1 ? threadIdx.x / G : 0;
    // A wave's column: scalar addresses, where registers are short (policy loss of 8192 columns of 4000 43.4 -> 40.0 us,
    // distillation of 2000 27.6 -> 25.9; of 1000, where scalar loads wait for each other, 31.5 -> 32.7).
    if constexpr (kTeams > 1 && G == kWave && NV > kGroupQuads) slot = __builtin_amdgcn_readfirstlane(slot);
    const size_t first = static_cast<size_t>(blockIdx.x) * kTeams, col = first + slot;
    if constexpr (kJoin) {
        head.to = TokenParts{parts, kTeams, first};
        if (team.rank < Head::kSums && col >= static_cast<size_t>(N)) parts[team.rank * kTeams + slot] = 0.0;
    } else if constexpr (Head::kSums > 0) {
        head.to.first = 0;   // known to the compiler
    }
    if (kTeams == 1 || col < static_cast<size_t>(N)) {   // whole teams
        token_column<Head, G, NV, NT, STREAM>(head, team, shared, dynamic + static_cast<size_t>(slot) * head.team_bytes(K),
                                              col, d ? d + col * ldd : nullptr, x + col * ld, K);
    }
    if constexpr (kJoin) {
        __syncthreads();
        const int k = threadIdx.x / kWave, lane = threadIdx.x % kWave;
        if (k < Head::kSums) {
            double v = 0.0;
            for (int i = lane; i < kTeams; i += kWave) v += parts[k * kTeams + i];
            v = Team<kWave>{lane}.lanes(v, AddOp{});
            if (lane == 0) {
                if constexpr (FOLD) sums.out[k] = static_cast<float>(v);
                else sums.part[static_cast<size_t>(k) * gridDim.x + blockIdx.x] = v;
            }
        }
    }
}

// ── columns cut into chunks ──────────────────────────────────────────────
// For columns that no workgroup holds: one workgroup per chunk leaves its
// maximum and sums (chunk kernel), one per column joins them and makes the coefficients
// (join), one per chunk writes the gradient (apply).
constexpr int kChunkBlock = 256;
constexpr int kChunk = 4 * kChunkBlock * kGroupQuads;
struct ChunkSums {
    double s, et;
    float m, pad[3];
};
struct ColumnCoef {
    Grad f;
    float m;
    int live, label, pad;
};
// the fixed 2^20 floats of the scratch: chunk sums in the first half, columns' coefficients behind
constexpr int kMaxChunks = (1 << 19) * 4 / static_cast<int>(sizeof(ChunkSums));
constexpr int kMaxColumns = (1 << 19) * 4 / static_cast<int>(sizeof(ColumnCoef));
constexpr size_t kScratchFixed = size_t(1) << 20;
constexpr int kMaxK = kChunk * kMaxChunks;
constexpr int kMaxTokens = 1 << 25;
constexpr unsigned long long kMaxLogits = 1ull << 36, kMaxThreads = (1ull << 32) - 1;   // of a launch
static_assert(sizeof(ChunkSums) == 32 && sizeof(ColumnCoef) == 32, "scratch layout");

template <class Head>
__global__ __launch_bounds__(kChunkBlock) void token_chunk_kernel(Head head, ChunkSums* sums, const float* x, int K,
                                                                  int chunks, size_t col0, size_t ld) {
    constexpr int G = kChunkBlock;
    __shared__ ColumnShared<G> sh;
    __shared__ unsigned bits[Head::kRest ? kChunk / 32 + 1 : 1];
    const Team<G> team{static_cast<int>(threadIdx.x)};
    const int part = blockIdx.x % chunks;
    const size_t col = col0 + blockIdx.x / chunks;
    if (!head.live(col, K)) return;
    const int begin = part * kChunk, len = K - begin < kChunk ? K - begin : kChunk;
    const float* p = x + col * ld + begin;
    const Span span = span_of<true>(p, len);
    Quad v[kGroupQuads];
#pragma unroll
    for (int k = 0; k < kGroupQuads; ++k) {
        const int q = team.rank + k * G;
        v[k] = Quad(-INFINITY);
        if (q < span.quads) v[k] = load_quad<false>(p + span.skew + 4 * q);
    }
    float last = team.rank < span.odd ? p[span.single(team.rank)] : -INFINITY;
    if constexpr (Head::kRest) {
        for (int i = team.rank; i < kChunk / 32; i += G) bits[i] = 0u;
        __syncthreads();
        head.mark(team, bits, col, begin, len);
        __syncthreads();
    }
    const Group g = take_group<Head>(v, head.scale, [&](int k) {
        const int q = team.rank + k * G;
        return known_quad(bits, span.skew + 4 * (q < span.quads ? q : 0));
    });
    ColumnSums c{-INFINITY, 0.0, 0.0};
    add_group<Head>(c, g, head.scale);
    if (team.rank < span.odd) {
        if constexpr (Head::kRest)
            if (known_one(bits, span.single(team.rank))) last = -INFINITY;
        add_group<Head>(c, take_one(last), head.scale);
    }
    scale_sums<Head>(c, team.reduce(c.m, LargerOp{}, sh.max), head.scale);
    if constexpr (Head::kEntropy) c.et = team.reduce(c.et, AddOp{}, sh.other);
    c.s = team.reduce(c.s, AddOp{}, sh.s);
    if (team.rank == 0) sums[blockIdx.x] = ChunkSums{c.s, c.et, c.m, {}};
}

template <class Head>
__global__ __launch_bounds__(kChunkBlock) void token_join_kernel(Head head, ColumnCoef* coef, const ChunkSums* sums,
                                                                 const float* x, int K, int chunks, size_t col0,
                                                                 size_t ld) {
    constexpr int G = kChunkBlock;
    __shared__ ColumnShared<G> sh;
    extern __shared__ __align__(16) char dynamic[];
    const Team<G> team{static_cast<int>(threadIdx.x)};
    const size_t col = col0 + blockIdx.x;
    const float* p = x + col * ld;
    ColumnCoef r{};
    bool live = head.live(col, K);
    if (live) {   // for the whole workgroup
        typename Head::Early early = head.early(col, p);
        ColumnSums c{-INFINITY, 0.0, 0.0};
        const ChunkSums* q = sums + static_cast<size_t>(blockIdx.x) * chunks;
        for (int i = team.rank; i < chunks; i += G) c.m = fmaxf(c.m, q[i].m);
        c.m = team.reduce(c.m, LargerOp{}, sh.max);
        const double inv = static_cast<double>(head.scale.hi) + static_cast<double>(head.scale.lo);
        for (int i = team.rank; i < chunks; i += G) {
            const ChunkSums w = q[i];
            // a chunk of -inf adds its sums as they are: 0, or NaN
            const double t = w.m == -INFINITY ? 0.0 : static_cast<double>(w.m) - static_cast<double>(c.m);
            const double f = exp64(t * inv * 0.69314718055994531);
            c.s += w.s * f;
            c.et += (w.et + w.s * (t < -1e4 ? -1e4 : t)) * f;
        }
        c.s = team.reduce(c.s, AddOp{}, sh.s);
        if constexpr (Head::kEntropy) c.et = team.reduce(c.et, AddOp{}, sh.other);
        if (!team.leads()) return;
        bool filled = false;
        if constexpr (Head::kTeacher) {
            live = head.prologue(team.lead(), dynamic, nullptr, col, K, p, early);
            filled = unmasked(early.m, early.s);
        }
        live = live && (filled || unmasked(c.m, c.s));
        if (live) {
            r.f = head.finish(team.lead(), dynamic, early, col, c);
            r.m = c.m == -INFINITY ? 0.f : c.m;   // as in token_column
            r.live = 1;
            r.label = head.label(col);
        }
    }
    if (team.rank == 0) {
        if (!live) head.idle(col);
        coef[blockIdx.x] = r;
    }
}

template <class Head>
__global__ __launch_bounds__(kChunkBlock) void token_apply_kernel(Head head, TokenSums sums, float* d,
                                                                  const ColumnCoef* coef, const float* x, int K, int N,
                                                                  int chunks, size_t col0, size_t ld, size_t ldd) {
    __shared__ double slots[kChunkBlock / kWave];
    extern __shared__ __align__(16) char dynamic[];
    const int rank = threadIdx.x, part = blockIdx.x % chunks;
    if (blockIdx.x == 0)   // every column is joined: the last group's first workgroup adds up their parts
        for (int k = 0; k < sums.count; ++k) {
            fold_parts<kChunkBlock>(sums.out + k, sums.part + static_cast<size_t>(k) * N, N, 1.0, slots);
            __syncthreads();
        }
    const size_t col = col0 + blockIdx.x / chunks;
    const ColumnCoef r = coef[blockIdx.x / chunks];
    const int begin = part * kChunk, len = K - begin < kChunk ? K - begin : kChunk;
    const float* p = x + col * ld + begin;
    float* out = d + col * ldd + begin;
    const Span span = span_of<true>(out, len);
    p += span.skew;
    float* const to = out + span.skew;
    if (!r.live) {
        for (int q = rank; q < span.quads; q += kChunkBlock) store_quad<false>(to + 4 * q, Quad(0.f));
        if (rank < span.odd) out[span.single(rank)] = 0.f;
        return;
    }
    auto value = [&](float y) {
        const float t = y - r.m;
        return grad_value<Head::kEntropy>(t, exp_shifted(t, head.scale), r.f.a, r.f.b);
    };
    Quad v[kGroupQuads];
#pragma unroll
    for (int k = 0; k < kGroupQuads; ++k) {
        const int q = rank + k * kChunkBlock;
        if (q < span.quads) v[k] = load_quad<false>(p + 4 * q);
    }
    const float last = rank < span.odd ? p[span.single(rank) - span.skew] : 0.f;
#pragma unroll
    for (int k = 0; k < kGroupQuads; ++k) {
        const int q = rank + k * kChunkBlock;
        if (q < span.quads)
            store_quad<false>(to + 4 * q, Quad{value(v[k].x), value(v[k].y), value(v[k].z), value(v[k].w)});
    }
    if (rank < span.odd) out[span.single(rank)] = value(last);
    const int label = r.label - begin;
    __syncthreads();   // behind the sweep that wrote these elements as any other
    if (rank == 0 && label >= 0 && label < len) correct_label<Head::kEntropy>(label, r.m, r.f, head.scale, out);
    if constexpr (Head::kTeacher) {
        head.correct_chunk(Team<kChunkBlock>{rank}, dynamic, col, begin, len, out);
    }
}

// Logits of a group of columns that several launches read twice: they and their gradient fit the
// 256 MB memory-side cache.
constexpr size_t kReadTwiceBytes = size_t(96) << 20;

// n parts to a sum
template <int BLOCK>
int launch_token_fold(const TokenSums& sums, int n) {
    if (sums.count == 0) return 0;
    token_fold_kernel<BLOCK><<<sums.count, BLOCK, 0, stream()>>>(sums.out, sums.part, n, static_cast<size_t>(n), 1.0);
    return launch_rc();
}

template <class Head>
int launch_token_chunks(Head head, const TokenSums& sums, float* scratch, float* d, const float* x, int K, int N,
                        size_t ld, size_t ldd) {
    const int chunks = (K + kChunk - 1) / kChunk;
    size_t group = Head::kWrites ? kReadTwiceBytes / (static_cast<size_t>(K) * sizeof(float)) : static_cast<size_t>(N);
    if (group > static_cast<size_t>(kMaxChunks / chunks)) group = kMaxChunks / chunks;
    if (group > static_cast<size_t>(kMaxColumns)) group = kMaxColumns;
    if (group < 1) group = 1;
    ChunkSums* part = reinterpret_cast<ChunkSums*>(scratch);
    ColumnCoef* coef = reinterpret_cast<ColumnCoef*>(scratch + kScratchFixed / 2);
    const size_t lds = head.team_bytes(0);
    if constexpr (Head::kTeacher) head.chunked = true;
    hipStream_t st = stream();
    for (size_t at = 0; at < static_cast<size_t>(N); at += group) {
        const bool last = static_cast<size_t>(N) - at <= group;
        const unsigned n = static_cast<unsigned>(last ? static_cast<size_t>(N) - at : group);
        token_chunk_kernel<<<n * chunks, kChunkBlock, 0, st>>>(head, part, x, K, chunks, at, ld);
        token_join_kernel<<<n, kChunkBlock, lds, st>>>(head, coef, part, x, K, chunks, at, ld);
        if constexpr (Head::kWrites) {
            if (d)
                token_apply_kernel<<<n * chunks, kChunkBlock, lds, st>>>(head, last ? sums : TokenSums{}, d, coef, x, K, N,
                                                                         chunks, at, ld, ldd);
        }
        const int rc = launch_rc();
        if (rc) return rc;
    }
    return d ? 0 : launch_token_fold<kChunkBlock>(sums, N);   // in the order of the apply kernel's
}

constexpr size_t kMaxLds = size_t(150) << 10;   // of 160 KB, beside what the kernels declare themselves

template <class Head, int G, int NV, int BLOCK, bool NT, bool STREAM, bool FOLD>
int launch_token_columns_as(const Head& head, const TokenSums& sums, float* d, const float* x, int K, int N, size_t ld,
                            size_t ldd) {
    constexpr int kTeams = BLOCK / G;
    const size_t lds = static_cast<size_t>(kTeams) * head.team_bytes(K);
    auto kernel = token_column_kernel<Head, G, NV, BLOCK, NT, STREAM, FOLD>;
    if (lds > (size_t(64) << 10)) {   // beyond the default limit
        static std::once_flag once;   // per instantiation
        static int configure_rc = 0;
        std::call_once(once, [&] {
            configure_rc = rc_of(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMaxLds)));
        });
        if (configure_rc) return configure_rc;
    }
    const unsigned blocks = (static_cast<unsigned>(N) + kTeams - 1) / kTeams;
    kernel<<<blocks, BLOCK, lds, stream()>>>(head, sums, d, x, K, N, ld, ldd);
    const int rc = launch_rc();
    return rc || FOLD ? rc : launch_token_fold<kFoldBlock>(sums, static_cast<int>(blocks));
}
template <class Head, int G, int NV, int BLOCK, bool STREAM>
int launch_token_columns(const Head& head, const TokenSums& sums, float* d, const float* x, int K, int N, size_t ld,
                         size_t ldd) {
    if (streams_past_cache(static_cast<size_t>(K) * N * sizeof(float) * (d ? 2 : 1)))
        return launch_token_columns_as<Head, G, NV, BLOCK, true, STREAM, false>(head, sums, d, x, K, N, ld, ldd);
    return launch_token_columns_as<Head, G, NV, BLOCK, false, STREAM, false>(head, sums, d, x, K, N, ld, ldd);
}
// teams of one wave or less: where one workgroup holds all columns, its sums are the call's
// (policy loss of 64 x 256: 9.0 us in two launches, 5.6 in one)
template <class Head, int G, int NV>
int launch_token_teams(const Head& head, const TokenSums& sums, float* d, const float* x, int K, int N, size_t ld,
                       size_t ldd) {
    if constexpr (Head::kWrites && NV == kGroupQuads) {
        if (N <= 1024 / G && (1024 / G) * head.team_bytes(K) <= (size_t(64) << 10))
            return launch_token_columns_as<Head, G, NV, 1024, false, false, true>(head, sums, d, x, K, N, ld, ldd);
    }
    return launch_token_columns<Head, G, NV, 256, false>(head, sums, d, x, K, N, ld, ldd);
}

// Which way a call goes.  us on MI355X, 512 MB of logits (a quarter of the tokens unscored) unless said
// otherwise; "values": logprobs, "gradient": the policy loss.
constexpr int kMaxTeam = 4096, kMaxResident = 32768;
inline bool token_in_chunks(int K, int N, bool gradient) {
    // A few long columns occupy as many CUs: 1 x 262144 values 25 -> 7, gradient 41 -> 14; 64 x 131072
    // 15 -> 8.5 and 25 -> 19.  With more columns the second read of the gradient decides: 128 x 262144 gradient
    // 56 in one piece, 63 in chunks; values 28 and 21, 256 x 262144 36 and 34.  Below K = 45056 one workgroup is
    // through before the further launches are (1 x 32000 values 6.2, 7.9 in chunks, gradient 8.7, 11.5; 1 x 50000
    // 8.5, 7.7 and 11.4, 11.4, with the teacher's rest 14.9, 12.7).
    return K > 11 * kChunk && static_cast<long long>(N) * (gradient ? 4 : 2) <= num_cus();
}
template <class Head>
int launch_token_kernel(const Head& head, const TokenSums& sums, float* scratch, float* d, const float* x, int K, int N,
                        size_t ld, size_t ldd) {
    if (K <= 64) return launch_token_teams<Head, 4, 4>(head, sums, d, x, K, N, ld, ldd);
    if (K <= 128) return launch_token_teams<Head, 8, 4>(head, sums, d, x, K, N, ld, ldd);
    if (K <= 256) return launch_token_teams<Head, 16, 4>(head, sums, d, x, K, N, ld, ldd);
    if (K <= 512) return launch_token_teams<Head, 32, 4>(head, sums, d, x, K, N, ld, ldd);
    if (K <= 1024) return launch_token_teams<Head, 64, 4>(head, sums, d, x, K, N, ld, ldd);
    if (K <= 2048) return launch_token_teams<Head, 64, 8>(head, sums, d, x, K, N, ld, ldd);
    if (K <= kMaxTeam) return launch_token_teams<Head, 64, 16>(head, sums, d, x, K, N, ld, ldd);
    if (token_in_chunks(K, N, Head::kWrites) || head.team_bytes(K) > kMaxLds)
        return launch_token_chunks(head, sums, scratch, d, x, K, N, ld, ldd);
    if constexpr (!Head::kWrites) {
        // Values alone need no column kept; small tiles waste least of their last round: K = 24000 61 (512 x 16
        // quads in one tile: 68), 131072 65 (1024 x 24 quads: 90).
        if (K <= 8192) return launch_token_columns<Head, 256, 8, 256, false>(head, sums, d, x, K, N, ld, ldd);
        if (K <= 16384) return launch_token_columns<Head, 256, 4, 256, true>(head, sums, d, x, K, N, ld, ldd);
        return launch_token_columns<Head, 512, 4, 512, true>(head, sums, d, x, K, N, ld, ldd);
    } else if (N > 2 * num_cus()) {
        // Half of the column kept, so that several workgroups on a CU overlap their loads and stores (policy /
        // distillation; in brackets: all of it kept by 256 x 8, 256 x 16, 512 x 16, 1024 x 16 quads): K = 5000
        // 109 / 123 (118 / 134), 12000 150 / 172 (165 / 188), 16000 153 / 176 (162 / 187), 24000 154 / 174
        // (165 / 187), 48000 157 / 181 (177 / 203), 64000 169 / 192 (169 / 194), the rest of the teacher's mass
        // at 48000 188 (237); 32000 161 / 183 either way.
        if (K <= 8192) return launch_token_columns<Head, 256, 4, 256, true>(head, sums, d, x, K, N, ld, ldd);
        if (K <= 16384) return launch_token_columns<Head, 512, 4, 512, true>(head, sums, d, x, K, N, ld, ldd);
        if (K <= 28672) return launch_token_columns<Head, 512, 8, 512, true>(head, sums, d, x, K, N, ld, ldd);
        if (K <= kMaxResident) return launch_token_columns<Head, 512, 16, 512, false>(head, sums, d, x, K, N, ld, ldd);
        if (K <= 2 * kMaxResident) return launch_token_columns<Head, 512, 16, 512, true>(head, sums, d, x, K, N, ld, ldd);
    } else {
        // No second workgroup to overlap with: one read (256 x 64000 23, half of it read again 25).
        if (K <= 8192) return launch_token_columns<Head, 256, 8, 256, false>(head, sums, d, x, K, N, ld, ldd);
        if (K <= 16384) return launch_token_columns<Head, 256, 16, 256, false>(head, sums, d, x, K, N, ld, ldd);
        if (K <= kMaxResident) return launch_token_columns<Head, 512, 16, 512, false>(head, sums, d, x, K, N, ld, ldd);
        if (K <= 2 * kMaxResident) return launch_token_columns<Head, 1024, 16, 1024, false>(head, sums, d, x, K, N, ld, ldd);
    }
    // K = 98000 174 (512 threads: 197; 24 quads: 183), 262144 195 (215; 191), rest 230 (239; 248); chunks read
    // twice over several launches 280.
    if constexpr (Head::kWrites) return launch_token_columns<Head, 1024, 16, 1024, true>(head, sums, d, x, K, N, ld, ldd);
}

// The arguments every entry point of this family checks alike.  With at most 64 threads to a column of up
// to 4096 logits, 256 to 8192, 512 to 65536 and 1024 beyond, kMaxTokens columns and kMaxLogits logits keep every
// launch below kMaxThreads.
inline bool token_args_ok(const float* x, const float* d, const float* scratch, int K, int N, int ld, int ldd) {
    if (K <= 0 || K > kMaxK || N <= 0 || ld < K || !x || !aligned16(scratch)) return false;
    if (N > kMaxTokens || static_cast<unsigned long long>(K) * N > kMaxLogits) return false;
    if (d && (ldd < K || (d == x && ldd != ld))) return false;
    return true;
}

}  // namespace jz
