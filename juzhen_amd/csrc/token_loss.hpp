// Shared device code of the losses over a K x N matrix of logits (one token per
// column): log-probabilities, policy, preference and distillation losses.
//
// For a column x with maximum m:  t_i = (x_i - m)/T,  e_i = exp(t_i),  s = sum e_i,
// p_i = e_i/s.  The shift makes every exponent <= 0, so s is in [1, K] and nothing
// overflows.  Each kernel hands a column to a team of threads; a `Head` turns
// (m, s, ...) into the coefficients of that column's gradient
//     d_i = e_i * (a + b*t_i)  (+ corrections at the label or the teacher's entries).
// Everything that happens once per column (log s, ratios, divergences) is done in
// 64 bits: it costs nothing beside K exponentials, and a ratio that lies near a
// clipping border falls on the side the exact value does.
#pragma once

#include "common.hpp"

namespace jz {

// log2(e)/T as a sum of two floats
struct ExpScale {
    float hi, lo;
};
inline ExpScale exp_scale(double temperature) {
    const double c = 1.44269504088896340736 / temperature;
    ExpScale r;
    r.hi = static_cast<float>(c);
    r.lo = static_cast<float>(c - static_cast<double>(r.hi));
    return r;
}

// exp(d/T) for d <= 0 through the hardware exp2, the rounding error of the product
// folded back in (about 2 ulp).  Below 2^-126 the result is an exact 0, for -inf
// too; a NaN stays one.
__device__ __forceinline__ float exp_shifted(float d, const ExpScale& c) {
    const float u = d * c.hi;
    const float err = fmaf(d, c.hi, -u) + d * c.lo;
    const float r = __builtin_amdgcn_exp2f(u) * (1.0f + 0.693147180559945309f * err);
    return u < -126.0f ? 0.0f : r;
}

struct AddOp {
    template <class T>
    __device__ __forceinline__ T operator()(T a, T b) const { return a + b; }
};
struct LargerOp {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};

// The threads that share one column: G lanes of a wave (G <= 64) or a whole workgroup
// of G threads.  Reductions run in one fixed order and leave the result in every thread.
template <int G>
struct Team {
    static constexpr int kSize = G;
    static constexpr int kWaves = G > kWave ? G / kWave : 1;
    int rank;
    double* red;   // kWaves values, workgroup teams only

    template <class T, class Op>
    __device__ __forceinline__ T reduce(T v, Op op) const {
        constexpr int W = G < kWave ? G : kWave;
#pragma unroll
        for (int o = 1; o < W; o *= 2) v = op(v, __shfl_xor(v, o, kWave));
        if constexpr (kWaves > 1) {
            T* slot = reinterpret_cast<T*>(red);
            __syncthreads();
            if ((rank & (kWave - 1)) == 0) slot[rank / kWave] = v;
            __syncthreads();
            v = slot[0];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) v = op(v, slot[w]);
        }
        return v;
    }
    template <class T>
    __device__ __forceinline__ T sum(T v) const { return reduce(v, AddOp{}); }
    __device__ __forceinline__ float max(float v) const { return reduce(v, LargerOp{}); }
    __device__ __forceinline__ bool any(bool v) const { return reduce(v ? 1.f : 0.f, LargerOp{}) != 0.f; }
    __device__ __forceinline__ void sync() const {
        if constexpr (kWaves > 1) __syncthreads();
    }
};

// What one sweep over a column leaves: its maximum, the sum of e_i, of e_i*t_i (heads
// that ask for the entropy) and of the e_i that are none of the teacher's entries
// (heads that ask for the rest).
struct ColumnSums {
    float m, s, et, rest;
};
// d_i = e_i * (a + b*t_i)
struct Coef {
    float a, b;
};

__device__ __forceinline__ bool label_scored(int label, int K) { return label >= 0 && label < K; }

// log softmax of the value `x` of a column, in 64 bits
__device__ __forceinline__ double log_prob(float x, const ColumnSums& c) {
    return (static_cast<double>(x) - static_cast<double>(c.m)) - log(static_cast<double>(c.s));
}
__device__ __forceinline__ double entropy_of(const ColumnSums& c) {
    return log(static_cast<double>(c.s)) - static_cast<double>(c.et) / static_cast<double>(c.s);
}

// One workgroup per column, three sweeps (maximum, sums, gradient).
constexpr int kSweepBlock = 256;
template <class Head>
__global__ __launch_bounds__(kSweepBlock) void token_sweep_kernel(Head head, float* d, const float* x, int K,
                                                                  size_t ld, size_t ldd) {
    __shared__ double red[kSweepBlock / kWave];
    __shared__ typename Head::Shared shared;
    const Team<kSweepBlock> team{static_cast<int>(threadIdx.x), red};
    const size_t col = blockIdx.x;
    const float* p = x + col * ld;
    float* out = d ? d + col * ldd : nullptr;
    bool live = head.live(col, K) && head.prologue(team, shared, col, K);
    ColumnSums c{-INFINITY, 0.f, 0.f, 0.f};
    if (live) {
        for (int i = team.rank; i < K; i += kSweepBlock) c.m = fmaxf(c.m, p[i]);
        c.m = team.max(c.m);
        if (c.m == -INFINITY) {   // nothing but masked entries, or NaN
            bool nan = false;
            for (int i = team.rank; i < K; i += kSweepBlock) nan |= p[i] != p[i];
            live = team.any(nan);
        }
    }
    if (!live) {
        if (team.rank == 0) head.idle(col);
        if (out)
            for (int i = team.rank; i < K; i += kSweepBlock) out[i] = 0.f;
        return;
    }
    for (int i = team.rank; i < K; i += kSweepBlock) {
        const float t = p[i] - c.m;
        const float e = exp_shifted(t, head.scale);
        c.s += e;
        if constexpr (Head::kEntropy) c.et += e != 0.f ? e * t : 0.f;
        if constexpr (Head::kRest) c.rest += head.known(shared, i) ? 0.f : e;
    }
    c.s = team.sum(c.s);
    if constexpr (Head::kEntropy) c.et = team.sum(c.et);
    if constexpr (Head::kRest) c.rest = team.sum(c.rest);
    const Coef f = head.finish(team, shared, col, c, p);
    if (!out) return;
    team.sync();   // the gradient may replace the logits: the head has read what it needs
    for (int i = team.rank; i < K; i += kSweepBlock) {
        const float t = p[i] - c.m;
        const float e = exp_shifted(t, head.scale);
        float v = e * f.a;
        if constexpr (Head::kEntropy) v = e != 0.f ? e * (f.a + f.b * t) : 0.f;
        out[i] = v;
    }
    team.sync();   // its corrections are written over what the sweep wrote
    head.correct(team, shared, col, c, f, out);
}

// out[k] = scale * sum_i part[k*stride + i]: one workgroup per output, accumulated in
// 64 bits in a fixed order.
constexpr int kFoldBlock = 1024;
template <class T>
__global__ __launch_bounds__(kFoldBlock) void token_fold_kernel(float* out, const T* part, int n, size_t stride,
                                                                double scale) {
    __shared__ double red[kFoldBlock / kWave];
    const Team<kFoldBlock> team{static_cast<int>(threadIdx.x), red};
    const T* p = part + blockIdx.x * stride;
    double a = 0.0;
    for (int i = team.rank; i < n; i += kFoldBlock) a += static_cast<double>(p[i]);
    a = team.sum(a);
    if (team.rank == 0) out[blockIdx.x] = static_cast<float>(scale * a);
}

template <class Head>
int launch_token_kernel(const Head& head, float* d, const float* x, int K, int N, size_t ld, size_t ldd) {
    token_sweep_kernel<<<static_cast<unsigned>(N), kSweepBlock, 0, stream()>>>(head, d, x, K, ld, ldd);
    return launch_rc();
}

// The arguments every entry point of this family checks alike.
inline bool token_args_ok(const float* x, const float* d, const float* scratch, int K, int N, int ld, int ldd) {
    if (K <= 0 || N <= 0 || ld < K || !x || !aligned16(scratch)) return false;
    if (d && (ldd < K || (d == x && ldd != ld))) return false;
    return true;
}

}  // namespace jz
