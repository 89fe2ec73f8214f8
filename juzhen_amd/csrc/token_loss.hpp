// Shared device code of the losses over a K x N matrix of logits (one token per
// column): log-probabilities, policy, preference and distillation losses.
//
// For a column x with maximum m:  t_i = x_i - m,  e_i = exp(t_i/T),  s = sum e_i,
// p_i = e_i/s.  The shift makes every exponent <= 0, so s is in [1, K] and nothing
// overflows.  Each kernel hands a column to a team of threads that keeps it in
// registers between the reductions, so it is read once and its gradient written once;
// a `Head` turns (m, s, ...) into the coefficients of that gradient,
//     d_i = e_i * (a + b*t_i)  (+ corrections at the label or the teacher's entries).
// What bounds all of them is memory: 8 bytes per logit against about 20 vector
// instructions (a third of what a CU issues in the time its share of 6.4 TB/s takes).
//
// Accuracy: exponentials within 0.7 ulp and without bias; a thread adds eight of them in
// fp32 and everything further in 64 bits (two 64-bit instructions per eight elements).
// Losses over many tokens cancel (the reward of an answer is a sum of small differences
// of log-probabilities), so a bias of a few 1e-8 per token would show in them.  What
// happens once per column (log s, ratios, divergences) is done in 64 bits too.
#pragma once

#include "common.hpp"

#include <atomic>

namespace jz {

// log2(e)/T as a sum of two floats, and the shift below which exp(d/T) < 2^-126
struct ExpScale {
    float hi, lo, least;
};
inline ExpScale exp_scale(double temperature) {
    const double c = 1.44269504088896340736 / temperature;
    ExpScale r;
    r.hi = static_cast<float>(c);
    r.lo = static_cast<float>(c - static_cast<double>(r.hi));
    r.least = static_cast<float>(-126.0 / c);
    return r;
}

// exp(d/T) for d <= 0: 2^n * 2^f with n = rint(d*c), f = d*c - n in [-1/2, 1/2] formed by
// fused products, 2^f by a polynomial of degree 6 (its own minimax fit of 2^f with the
// constant term 1, relative error 2e-9, rounded coefficients: 0.67 ulp at most, mean
// 1e-9).  Below 2^-126 the result is an exact 0, for -inf too; a NaN stays one.
__device__ __forceinline__ float exp_shifted(float d, const ExpScale& c) {
    constexpr float kRound = 12582912.0f;   // 1.5 * 2^23: adding it rounds to an integer
    const float r = fmaf(d, c.hi, kRound);
    const float n = r - kRound;
    const float f = fmaf(d, c.lo, fmaf(d, c.hi, -n));
    float p = 0x1.41fbbcp-13f;
    p = fmaf(p, f, 0x1.5f3e54p-10f);
    p = fmaf(p, f, 0x1.3b2d4cp-7f);
    p = fmaf(p, f, 0x1.c6aee8p-5f);
    p = fmaf(p, f, 0x1.ebfbdcp-3f);
    p = fmaf(p, f, 0x1.62e430p-1f);
    p = fmaf(p, f, 1.0f);
    p = __builtin_amdgcn_ldexpf(p, __builtin_bit_cast(int, r) - __builtin_bit_cast(int, kRound));
    return d < c.least ? 0.0f : p;
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
    int rank;
    double* red;   // 2*kWaves values, workgroup teams only

    template <class T, class Op>
    __device__ __forceinline__ T reduce(T v, Op op) const {
        constexpr int W = G < kWave ? G : kWave;
        v = op(v, dpp_mov<0xB1>(v));                          // quad_perm [1,0,3,2]
        v = op(v, dpp_mov<0x4E>(v));                          // quad_perm [2,3,0,1]
        if constexpr (W >= 8) v = op(v, dpp_mov<0x141>(v));   // row_half_mirror
        if constexpr (W >= 16) v = op(v, dpp_mov<0x140>(v));  // row_mirror
        if constexpr (W >= 32) v = op(v, __shfl_xor(v, 16, kWave));
        if constexpr (W >= 64) v = op(v, __shfl_xor(v, 32, kWave));
        if constexpr (kWorkgroup) {
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
    // two sums behind one pair of barriers
    __device__ __forceinline__ void sum2(double& a, double& b) const {
        Team<(G < kWave ? G : kWave)> wave{rank, nullptr};
        a = wave.sum(a);
        b = wave.sum(b);
        if constexpr (kWorkgroup) {
            __syncthreads();
            if ((rank & (kWave - 1)) == 0) {
                red[rank / kWave] = a;
                red[kWaves + rank / kWave] = b;
            }
            __syncthreads();
            a = red[0];
            b = red[kWaves];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) {
                a += red[w];
                b += red[kWaves + w];
            }
        }
    }
    __device__ __forceinline__ float max(float v) const { return reduce(v, LargerOp{}); }
    __device__ __forceinline__ bool any(bool v) const { return reduce(v ? 1.f : 0.f, LargerOp{}) != 0.f; }
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
    // Work that is done once per column: by the first wave of a workgroup; by every lane of
    // a smaller team, whose wave issues it anyway.
    __device__ __forceinline__ bool leads() const { return !kWorkgroup || rank < kWave; }
};

// Keeps the 64-bit functions of a column's scalars apart: interleaved they would need the
// registers that hold the column.
__device__ __forceinline__ double one_at_a_time(double v) {
    asm volatile("" : "+v"(v));
    __builtin_amdgcn_sched_barrier(0);
    return v;
}

// What one sweep over a column leaves: its maximum, the sum of e_i, of e_i*t_i (heads
// that ask for the entropy) and of the e_i that are none of the teacher's entries
// (heads that ask for the rest).
struct ColumnSums {
    float m;
    double s, et, rest;
};
// d_i = e_i * (a + b*t_i); g is added at the label, whose logit is x.
struct Grad {
    float a, b, g, x;
};

__device__ __forceinline__ bool label_scored(int label, int K) { return label >= 0 && label < K; }

// log softmax of the value `x` of a column
__device__ __forceinline__ double log_prob(float x, const ColumnSums& c) {
    return (static_cast<double>(x) - static_cast<double>(c.m)) - log(c.s);
}
__device__ __forceinline__ double entropy_of(const ColumnSums& c) { return log(c.s) - c.et / c.s; }

template <bool LINEAR>
__device__ __forceinline__ float grad_value(float t, float e, float a, float b) {
    if constexpr (LINEAR) return e != 0.f ? e * (a + b * t) : 0.f;
    else return e * a;
}

// Four consecutive logits.  Columns start at any multiple of ld, so the address is only
// known to be a multiple of 4 bytes; the hardware takes a 16-byte access at any of them.
typedef float Quad __attribute__((ext_vector_type(4), aligned(4)));

// Which logits of a column of K belong to the teacher's entries: one bit each.
__device__ __forceinline__ unsigned known_quad(const unsigned* bits, int quad) {
    return (bits[quad >> 3] >> ((quad & 7) * 4)) & 15u;
}
__device__ __forceinline__ bool known_one(const unsigned* bits, int i) { return (bits[i >> 5] >> (i & 31)) & 1u; }

// Adds fp32 values: eight (two quads) in fp32, these in 64 bits.
struct Total {
    double all = 0.0;
    float open = 0.f;
    int have = 0;
    __device__ __forceinline__ void quad(float a, float b, float c, float d) {
        const float q = (a + b) + (c + d);
        if (have == 0) open = q;
        else all += static_cast<double>(open + q);
        have ^= 1;   // a constant in unrolled code
    }
    __device__ __forceinline__ double value(float last) const {
        return all + static_cast<double>((have ? open : 0.f) + last);
    }
};

// The compiler would interleave all the independent exponentials of an unrolled loop and
// spill what it thereby has live; where a thread holds many quads it is kept to two at a time.
template <int NV>
__device__ __forceinline__ void together(int k) {
    if constexpr (NV > 4)
        if (k % 2) __builtin_amdgcn_sched_barrier(0);
}
// Keeps a running sum from being formed only where it is used, its terms live until then.
template <int NV>
__device__ __forceinline__ void settle(Total& t, int k) {
    if constexpr (NV > 4)
        if (k % 2) asm volatile("" : "+v"(t.all));
}

// Columns held by teams of one wave or less (K <= 16*G, G lanes of up to four quads each) or
// by a workgroup (K <= 4*G*(NV + NL), NV quads per thread in registers, NL in LDS).
// A column's K % 4 last logits are one more value in the first threads of its team.
//   dynamic LDS: NL*G quads, then per team head.team_bytes() rounded up to 16
template <class Head, int G, int NV, int NL, int BLOCK>
__global__ __launch_bounds__(BLOCK, 4) void token_column_kernel(Head head, float* d, const float* x, int K, int N,
                                                             size_t ld, size_t ldd) {
    constexpr int kTeams = BLOCK / G;
    __shared__ double red[2 * Team<G>::kWaves];
    __shared__ Grad shared_grad;
    extern __shared__ __align__(16) char dynamic[];
    const Team<G> team{static_cast<int>(kTeams > 1 ? threadIdx.x % G : threadIdx.x), red};
    const int slot = kTeams > 1 ? threadIdx.x / G : 0;
    const size_t col = static_cast<size_t>(blockIdx.x) * kTeams + slot;
    if (kTeams > 1 && col >= static_cast<size_t>(N)) return;   // whole teams
    Quad* kept = reinterpret_cast<Quad*>(dynamic);
    char* own = dynamic + sizeof(Quad) * NL * G + static_cast<size_t>(slot) * head.team_bytes(K);
    const float* p = x + col * ld;
    float* out = d ? d + col * ldd : nullptr;
    const int quads = K / 4, odd = K % 4;

    bool live = head.live(col, K);
    Quad v[NV];
    float last = -INFINITY;
    ColumnSums c{-INFINITY, 0.0, 0.0, 0.0};
    if (live) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int q = team.rank + k * G;
            v[k] = Quad(-INFINITY);
            if (q < quads) v[k] = *reinterpret_cast<const Quad*>(p + 4 * static_cast<size_t>(q));
        }
        if (team.rank < odd) last = p[4 * static_cast<size_t>(quads) + team.rank];
#pragma unroll
        for (int k = 0; k < NL; ++k) {
            const int q = team.rank + (NV + k) * G;
            Quad w = Quad(-INFINITY);
            if (q < quads) w = *reinterpret_cast<const Quad*>(p + 4 * static_cast<size_t>(q));
            kept[k * G + team.rank] = w;
        }
        live = head.prologue(team, own, col, K);   // while the loads are under way
    }
    const unsigned* bits = nullptr;
    if constexpr (Head::kRest) {
        if (live) {
            unsigned* all = head.bits(own);
            for (int i = team.rank; i < (K + 31) / 32; i += G) all[i] = 0u;
            team.sync();
            head.mark(team, all, col, 0, K);
            team.sync();
            bits = all;
        }
    }
    if (live) {
        float m = last;
#pragma unroll
        for (int k = 0; k < NV; ++k) m = fmaxf(m, fmaxf(fmaxf(v[k].x, v[k].y), fmaxf(v[k].z, v[k].w)));
#pragma unroll
        for (int k = 0; k < NL; ++k) {
            const Quad w = kept[k * G + team.rank];
            m = fmaxf(m, fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w)));
        }
        c.m = team.max(m);
        if (c.m == -INFINITY) {   // nothing but masked entries, or NaN
            bool nan = last != last;
#pragma unroll
            for (int k = 0; k < NV; ++k)
                nan |= v[k].x != v[k].x || v[k].y != v[k].y || v[k].z != v[k].z || v[k].w != v[k].w;
#pragma unroll
            for (int k = 0; k < NL; ++k) {
                const Quad w = kept[k * G + team.rank];
                nan |= w.x != w.x || w.y != w.y || w.z != w.z || w.w != w.w;
            }
            live = team.any(nan);
        }
    }
    if (!live) {
        if (team.rank == 0) head.idle(col);
        if (out) {
            for (int q = team.rank; q < quads; q += G) *reinterpret_cast<Quad*>(out + 4 * static_cast<size_t>(q)) = Quad(0.f);
            if (team.rank < odd) out[4 * static_cast<size_t>(quads) + team.rank] = 0.f;
        }
        return;
    }

    Total s, et, rest;
    auto add = [&](Quad& w, int q) {
        const float t0 = w.x - c.m, t1 = w.y - c.m, t2 = w.z - c.m, t3 = w.w - c.m;
        const float e0 = exp_shifted(t0, head.scale), e1 = exp_shifted(t1, head.scale);
        const float e2 = exp_shifted(t2, head.scale), e3 = exp_shifted(t3, head.scale);
        s.quad(e0, e1, e2, e3);
        if constexpr (Head::kEntropy) {
            et.quad(e0 != 0.f ? e0 * t0 : 0.f, e1 != 0.f ? e1 * t1 : 0.f, e2 != 0.f ? e2 * t2 : 0.f,
                    e3 != 0.f ? e3 * t3 : 0.f);
            w = Quad{t0, t1, t2, t3};
        } else {
            w = Quad{e0, e1, e2, e3};
        }
        if constexpr (Head::kRest) {
            const unsigned k = q < quads ? known_quad(bits, q) : 15u;
            rest.quad(k & 1u ? 0.f : e0, k & 2u ? 0.f : e1, k & 4u ? 0.f : e2, k & 8u ? 0.f : e3);
        }
    };
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        add(v[k], team.rank + k * G);
        if constexpr (Head::kEntropy) settle<NV>(et, k);
        if constexpr (Head::kRest) settle<NV>(rest, k);
        together<NV>(k);
    }
#pragma unroll
    for (int k = 0; k < NL; ++k) {
        Quad w = kept[k * G + team.rank];
        add(w, team.rank + (NV + k) * G);
        kept[k * G + team.rank] = w;
        if constexpr (Head::kEntropy) settle<NV>(et, k);
        if constexpr (Head::kRest) settle<NV>(rest, k);
        together<NV>(k);
    }
    const float tl = last - c.m, el = exp_shifted(tl, head.scale);
    c.s = s.value(el);
    if constexpr (Head::kEntropy) {
        c.et = et.value(el != 0.f ? el * tl : 0.f);
        team.sum2(c.s, c.et);
    } else if constexpr (Head::kRest) {
        c.rest = rest.value(team.rank < odd && !known_one(bits, 4 * quads + team.rank) ? el : 0.f);
        team.sum2(c.s, c.rest);
    } else {
        c.s = team.sum(c.s);
    }
    Grad f = head.finish(team, own, col, c, p);
    if constexpr (Team<G>::kWorkgroup && !Head::kTeamwork) {
        if (team.rank == 0) shared_grad = f;
        __syncthreads();
        f = shared_grad;
    } else {
        team.sync();   // the gradient may replace the logits: the head has read what it needs
    }
    if (!Head::kWrites || !out) return;
    auto write = [&](Quad w, int q) {
        if (q >= quads) return;
        Quad r;
        if constexpr (Head::kEntropy) {
            // the shifts are kept, not the exponentials too: those are formed again
            asm volatile("" : "+v"(w.x), "+v"(w.y), "+v"(w.z), "+v"(w.w));
            r.x = grad_value<true>(w.x, exp_shifted(w.x, head.scale), f.a, f.b);
            r.y = grad_value<true>(w.y, exp_shifted(w.y, head.scale), f.a, f.b);
            r.z = grad_value<true>(w.z, exp_shifted(w.z, head.scale), f.a, f.b);
            r.w = grad_value<true>(w.w, exp_shifted(w.w, head.scale), f.a, f.b);
        } else {
            r = Quad{w.x * f.a, w.y * f.a, w.z * f.a, w.w * f.a};
        }
        *reinterpret_cast<Quad*>(out + 4 * static_cast<size_t>(q)) = r;
    };
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        write(v[k], team.rank + k * G);
        together<NV>(k);
    }
#pragma unroll
    for (int k = 0; k < NL; ++k) {
        write(kept[k * G + team.rank], team.rank + (NV + k) * G);
        together<NV>(k);
    }
    if (team.rank < odd)
        out[4 * static_cast<size_t>(quads) + team.rank] = grad_value<Head::kEntropy>(tl, el, f.a, f.b);
    head.correct(team, own, col, c.m, f, out, quads);
}

// The label's element: the thread that wrote its quad writes it again.
template <bool LINEAR, class T>
__device__ __forceinline__ void correct_label(const T& team, int label, int quads, float m, const Grad& f,
                                              const ExpScale& scale, float* out) {
    const int quad = label / 4;
    if (team.rank == (quad < quads ? quad % T::kSize : label - 4 * quads)) {
        const float t = f.x - m;
        out[label] = grad_value<LINEAR>(t, exp_shifted(t, scale), f.a, f.b) + f.g;
    }
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
    double a0 = 0.0, a1 = 0.0, a2 = 0.0, a3 = 0.0;
    int i = team.rank;
    for (; i + 3 * kFoldBlock < n; i += 4 * kFoldBlock) {
        const T x0 = p[i], x1 = p[i + kFoldBlock], x2 = p[i + 2 * kFoldBlock], x3 = p[i + 3 * kFoldBlock];
        a0 += static_cast<double>(x0); a1 += static_cast<double>(x1);
        a2 += static_cast<double>(x2); a3 += static_cast<double>(x3);
    }
    for (; i < n; i += kFoldBlock) a0 += static_cast<double>(p[i]);
    a0 = team.sum((a0 + a1) + (a2 + a3));
    if (team.rank == 0) out[blockIdx.x] = static_cast<float>(scale * a0);
}

// ── columns cut into chunks ──────────────────────────────────────────────
// For columns that no workgroup holds: one workgroup per chunk leaves its
// maximum and sums (chunk kernel), one per column joins them and makes the coefficients
// (join), one per chunk writes the gradient (apply), where the head needs it one
// per column its corrections.
constexpr int kChunkBlock = 256, kChunkQuads = 4;
constexpr int kChunk = 4 * kChunkBlock * kChunkQuads;
struct ChunkSums {
    double s, et, rest;
    float m, pad;
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
static_assert(sizeof(ChunkSums) == 32 && sizeof(ColumnCoef) == 32, "scratch layout");

template <class Head>
__global__ __launch_bounds__(kChunkBlock) void token_chunk_kernel(Head head, ChunkSums* sums, const float* x, int K,
                                                                  int chunks, size_t col0, size_t ld) {
    __shared__ double red[2 * kChunkBlock / kWave];
    __shared__ unsigned bits[Head::kRest ? kChunk / 32 : 1];
    const Team<kChunkBlock> team{static_cast<int>(threadIdx.x), red};
    const int part = blockIdx.x % chunks;
    const size_t col = col0 + blockIdx.x / chunks;
    if (!head.live(col, K)) return;
    const int begin = part * kChunk, len = K - begin < kChunk ? K - begin : kChunk;
    const float* p = x + col * ld + begin;
    const int quads = len / 4, odd = len % 4;
    Quad v[kChunkQuads];
#pragma unroll
    for (int k = 0; k < kChunkQuads; ++k) {
        const int q = team.rank + k * kChunkBlock;
        v[k] = Quad(-INFINITY);
        if (q < quads) v[k] = *reinterpret_cast<const Quad*>(p + 4 * q);
    }
    float last = team.rank < odd ? p[4 * quads + team.rank] : -INFINITY;
    if constexpr (Head::kRest) {
        for (int i = team.rank; i < kChunk / 32; i += kChunkBlock) bits[i] = 0u;
        __syncthreads();
        head.mark(team, bits, col, begin, len);
        __syncthreads();
    }
    float m = last;
#pragma unroll
    for (int k = 0; k < kChunkQuads; ++k) m = fmaxf(m, fmaxf(fmaxf(v[k].x, v[k].y), fmaxf(v[k].z, v[k].w)));
    m = team.max(m);
    // a chunk of -inf only: shifts of 0 - inf, sums of 0; a NaN still shows
    const float shift = m == -INFINITY ? 0.f : m;
    Total s, et, rest;
    auto add = [&](float t0, float t1, float t2, float t3, unsigned known) {
        const float e0 = exp_shifted(t0, head.scale), e1 = exp_shifted(t1, head.scale);
        const float e2 = exp_shifted(t2, head.scale), e3 = exp_shifted(t3, head.scale);
        s.quad(e0, e1, e2, e3);
        if constexpr (Head::kEntropy)
            et.quad(e0 != 0.f ? e0 * t0 : 0.f, e1 != 0.f ? e1 * t1 : 0.f, e2 != 0.f ? e2 * t2 : 0.f,
                    e3 != 0.f ? e3 * t3 : 0.f);
        if constexpr (Head::kRest)
            rest.quad(known & 1u ? 0.f : e0, known & 2u ? 0.f : e1, known & 4u ? 0.f : e2, known & 8u ? 0.f : e3);
    };
#pragma unroll
    for (int k = 0; k < kChunkQuads; ++k) {
        const int q = team.rank + k * kChunkBlock;
        add(v[k].x - shift, v[k].y - shift, v[k].z - shift, v[k].w - shift,
            Head::kRest && q < quads ? known_quad(bits, q) : 0u);
    }
    const float tl = last - shift, el = exp_shifted(tl, head.scale);
    ChunkSums r{0.0, 0.0, 0.0, m, 0.f};
    r.s = s.value(el);
    if constexpr (Head::kEntropy) {
        r.et = et.value(el != 0.f ? el * tl : 0.f);
        team.sum2(r.s, r.et);
    } else if constexpr (Head::kRest) {
        r.rest = rest.value(team.rank < odd && !known_one(bits, 4 * quads + team.rank) ? el : 0.f);
        team.sum2(r.s, r.rest);
    } else {
        r.s = team.sum(r.s);
    }
    if (team.rank == 0) sums[blockIdx.x] = r;
}

template <class Head>
__global__ __launch_bounds__(kChunkBlock) void token_join_kernel(Head head, ColumnCoef* coef, const ChunkSums* sums,
                                                                 const float* x, int K, int chunks, size_t col0,
                                                                 size_t ld) {
    __shared__ double red[2 * kChunkBlock / kWave];
    extern __shared__ __align__(16) char dynamic[];
    const Team<kChunkBlock> team{static_cast<int>(threadIdx.x), red};
    const size_t col = col0 + blockIdx.x;
    ColumnCoef r{};
    bool live = head.live(col, K) && head.prologue(team, dynamic, col, K);
    ColumnSums c{-INFINITY, 0.0, 0.0, 0.0};
    if (live) {
        const ChunkSums* q = sums + static_cast<size_t>(blockIdx.x) * chunks;
        for (int i = team.rank; i < chunks; i += kChunkBlock) c.m = fmaxf(c.m, q[i].m);
        c.m = team.max(c.m);
        bool nan = false;
        const double inv = static_cast<double>(head.scale.hi) + static_cast<double>(head.scale.lo);
        for (int i = team.rank; i < chunks; i += kChunkBlock) {
            const ChunkSums w = q[i];
            nan |= w.s != w.s;
            if (w.m == -INFINITY) {
                if (w.s != w.s) c.s += w.s;
                continue;
            }
            const double t = static_cast<double>(w.m) - static_cast<double>(c.m);
            const double scale = exp2(t * inv);
            c.s += w.s * scale;
            if (scale != 0.0) c.et += (w.et + w.s * t) * scale;
            c.rest += w.rest * scale;
        }
        c.s = team.sum(c.s);
        if constexpr (Head::kEntropy) c.et = team.sum(c.et);
        if constexpr (Head::kRest) c.rest = team.sum(c.rest);
        nan = team.any(nan);
        if (c.m == -INFINITY) live = nan;
    }
    if (live) {
        r.f = head.finish(team, dynamic, col, c, x + col * ld);
        r.m = c.m;
        r.live = 1;
        r.label = head.label(col);
    } else if (team.rank == 0) {
        head.idle(col);
    }
    if (team.rank == 0) coef[blockIdx.x] = r;
}

template <class Head>
__global__ __launch_bounds__(kChunkBlock) void token_apply_kernel(Head head, float* d, const ColumnCoef* coef,
                                                                  const float* x, int K, int chunks, size_t col0,
                                                                  size_t ld, size_t ldd) {
    const int rank = threadIdx.x, part = blockIdx.x % chunks;
    const size_t col = col0 + blockIdx.x / chunks;
    const ColumnCoef r = coef[blockIdx.x / chunks];
    const int begin = part * kChunk, len = K - begin < kChunk ? K - begin : kChunk;
    const float* p = x + col * ld + begin;
    float* out = d + col * ldd + begin;
    const int quads = len / 4, odd = len % 4;
    if (!r.live) {
        for (int q = rank; q < quads; q += kChunkBlock) *reinterpret_cast<Quad*>(out + 4 * q) = Quad(0.f);
        if (rank < odd) out[4 * quads + rank] = 0.f;
        return;
    }
    auto value = [&](float y) {
        const float t = y - r.m;
        return grad_value<Head::kEntropy>(t, exp_shifted(t, head.scale), r.f.a, r.f.b);
    };
    Quad v[kChunkQuads];
#pragma unroll
    for (int k = 0; k < kChunkQuads; ++k) {
        const int q = rank + k * kChunkBlock;
        if (q < quads) v[k] = *reinterpret_cast<const Quad*>(p + 4 * q);
    }
    const float last = rank < odd ? p[4 * quads + rank] : 0.f;
#pragma unroll
    for (int k = 0; k < kChunkQuads; ++k) {
        const int q = rank + k * kChunkBlock;
        if (q < quads) *reinterpret_cast<Quad*>(out + 4 * q) = Quad{value(v[k].x), value(v[k].y), value(v[k].z), value(v[k].w)};
    }
    if (rank < odd) out[4 * quads + rank] = value(last);
    const int label = r.label - begin;
    if (label >= 0 && label < len) {
        const Team<kChunkBlock> team{rank, nullptr};
        correct_label<Head::kEntropy>(team, label, quads, r.m, r.f, head.scale, out);
    }
}

template <class Head>
__global__ __launch_bounds__(kChunkBlock) void token_correct_kernel(Head head, float* d, const ColumnCoef* coef, int K,
                                                                    size_t col0, size_t ldd) {
    __shared__ double red[2 * kChunkBlock / kWave];
    extern __shared__ __align__(16) char dynamic[];
    const Team<kChunkBlock> team{static_cast<int>(threadIdx.x), red};
    const size_t col = col0 + blockIdx.x;
    const ColumnCoef r = coef[blockIdx.x];
    if (!r.live || !head.prologue(team, dynamic, col, K)) return;
    head.restore(team, dynamic, col, r.f);
    head.correct(team, dynamic, col, r.m, r.f, d + col * ldd, 0);
}

// Logits of a group of columns that are read twice: the second read comes out of the
// 256 MB memory-side cache when they and their gradient fit it.
constexpr size_t kGroupBytes = size_t(96) << 20;

template <class Head>
int launch_token_chunks(const Head& head, float* scratch, float* d, const float* x, int K, int N, size_t ld,
                        size_t ldd) {
    const int chunks = (K + kChunk - 1) / kChunk;
    size_t group = kGroupBytes / (static_cast<size_t>(K) * sizeof(float));
    if (group > static_cast<size_t>(kMaxChunks / chunks)) group = kMaxChunks / chunks;
    if (group > static_cast<size_t>(kMaxColumns)) group = kMaxColumns;
    if (group < 1) group = 1;
    ChunkSums* sums = reinterpret_cast<ChunkSums*>(scratch);
    ColumnCoef* coef = reinterpret_cast<ColumnCoef*>(scratch + kScratchFixed / 2);
    const size_t lds = head.team_bytes(0);
    hipStream_t st = stream();
    for (size_t at = 0; at < static_cast<size_t>(N); at += group) {
        const unsigned n = static_cast<unsigned>(static_cast<size_t>(N) - at < group ? static_cast<size_t>(N) - at : group);
        token_chunk_kernel<<<n * chunks, kChunkBlock, 0, st>>>(head, sums, x, K, chunks, at, ld);
        token_join_kernel<<<n, kChunkBlock, lds, st>>>(head, coef, sums, x, K, chunks, at, ld);
        if (d) {
            token_apply_kernel<<<n * chunks, kChunkBlock, 0, st>>>(head, d, coef, x, K, chunks, at, ld, ldd);
            if constexpr (Head::kTeamwork)
                token_correct_kernel<<<n, kChunkBlock, lds, st>>>(head, d, coef, K, at, ldd);
        }
        const int rc = launch_rc();
        if (rc) return rc;
    }
    return 0;
}

template <class Head, int G, int NV, int NL, int BLOCK>
int launch_token_columns(const Head& head, float* d, const float* x, int K, int N, size_t ld, size_t ldd) {
    constexpr int kTeams = BLOCK / G;
    const size_t lds = sizeof(Quad) * NL * G + static_cast<size_t>(kTeams) * head.team_bytes(K);
    auto kernel = token_column_kernel<Head, G, NV, NL, BLOCK>;
    if (lds > (size_t(64) << 10)) {   // beyond the default limit
        static std::atomic<size_t> allowed{0};
        if (allowed.load(std::memory_order_relaxed) < lds) {
            const int rc = rc_of(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
            if (rc) return rc;
            allowed.store(lds, std::memory_order_relaxed);
        }
    }
    kernel<<<(static_cast<unsigned>(N) + kTeams - 1) / kTeams, BLOCK, lds, stream()>>>(head, d, x, K, N, ld, ldd);
    return launch_rc();
}

template <class Head>
int launch_token_kernel(const Head& head, float* scratch, float* d, const float* x, int K, int N, size_t ld,
                        size_t ldd) {
    if (K <= 64) return launch_token_columns<Head, 4, 4, 0, 256>(head, d, x, K, N, ld, ldd);
    if (K <= 128) return launch_token_columns<Head, 8, 4, 0, 256>(head, d, x, K, N, ld, ldd);
    if (K <= 256) return launch_token_columns<Head, 16, 4, 0, 256>(head, d, x, K, N, ld, ldd);
    if (K <= 512) return launch_token_columns<Head, 32, 4, 0, 256>(head, d, x, K, N, ld, ldd);
    if (K <= 1024) return launch_token_columns<Head, 64, 4, 0, 256>(head, d, x, K, N, ld, ldd);
    if (K <= 4096) return launch_token_columns<Head, 256, 4, 0, 256>(head, d, x, K, N, ld, ldd);
    if (K <= 8192) return launch_token_columns<Head, 256, 8, 0, 256>(head, d, x, K, N, ld, ldd);
    if (K <= 16384) return launch_token_columns<Head, 512, 8, 0, 512>(head, d, x, K, N, ld, ldd);
    if (K <= 32768) return launch_token_columns<Head, 512, 16, 0, 512>(head, d, x, K, N, ld, ldd);
    if (K <= 65536) return launch_token_columns<Head, 1024, 16, 0, 1024>(head, d, x, K, N, ld, ldd);
    if (K <= 98304) return launch_token_columns<Head, 1024, 24, 0, 1024>(head, d, x, K, N, ld, ldd);
    if (K <= 131072) return launch_token_columns<Head, 1024, 24, 8, 1024>(head, d, x, K, N, ld, ldd);
    return launch_token_chunks(head, scratch, d, x, K, N, ld, ldd);
}

// The arguments every entry point of this family checks alike.
inline bool token_args_ok(const float* x, const float* d, const float* scratch, int K, int N, int ld, int ldd) {
    if (K <= 0 || K > kMaxK || N <= 0 || ld < K || !x || !aligned16(scratch)) return false;
    if (d && (ldd < K || (d == x && ldd != ld))) return false;
    return true;
}

}  // namespace jz
