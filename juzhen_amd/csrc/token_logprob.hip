// Log-probabilities of one label per token, their gradient, and the paired
// log-ratio (preference) loss built on the two.
#include "token_loss.hpp"

namespace jz {
namespace {

template <bool ENTROPY>
struct LogprobHead {
    static constexpr bool kEntropy = ENTROPY, kRest = false, kTeacher = false, kWrites = false;
    struct Early {
        float x;   // the label's logit
    };
    ExpScale scale;
    const int32_t* labels;
    float *logp, *entropy, *stats;   // each may be null
    int N;

    __host__ __device__ size_t team_bytes(int) const { return 0; }
    __device__ bool live(size_t col, int K) const { return label_scored(labels[col], K); }
    __device__ int label(size_t col) const { return labels[col]; }
    __device__ Early early(size_t col, const float* x) const { return Early{x[labels[col]]}; }
    __device__ void write(size_t col, float lp, float h, float m, float s) const {
        if (logp) logp[col] = lp;
        if (ENTROPY) entropy[col] = h;
        if (stats) {
            stats[col] = m;
            stats[static_cast<size_t>(N) + col] = s;
        }
    }
    __device__ void idle(size_t col) const { write(col, 0.f, 0.f, 0.f, 0.f); }
    template <class T>
    __device__ Grad finish(const T& lead, char*, const Early& e, size_t col, const ColumnSums& c) const {
        const float lp = static_cast<float>(log_prob(e.x, c));
        const float h = ENTROPY ? static_cast<float>(entropy_of(c)) : 0.f;
        if (lead.rank == 0) write(col, lp, h, c.m, static_cast<float>(c.s));
        return Grad{};
    }
    template <class T>
    __device__ void correct(const T&, char*, size_t, float, const Grad&, float*, const Span&) const {}
};

// d_i = g*(delta_i - e_i/s) from the maximum and the sum of the forward call: no reduction
// is left, every element is read and written once.  A team of G threads takes 16*G
// logits of a column.
constexpr int kBwdBlock = 256, kBwdQuads = 4;
template <int G, bool NT>
__global__ __launch_bounds__(kBwdBlock) void logprob_bwd_kernel(float* d, const float* g, const float* x,
                                                                const int32_t* labels, const float* stats, int K,
                                                                int N, int chunks, size_t ld, size_t ldd,
                                                                ExpScale scale) {
    constexpr int kTeams = kBwdBlock / G, kSpan = 4 * G * kBwdQuads;
    const Team<G> team{static_cast<int>(threadIdx.x % G)};
    const size_t piece = static_cast<size_t>(blockIdx.x) * kTeams + threadIdx.x / G;
    const size_t col = kTeams > 1 ? piece : piece / chunks;
    if (col >= static_cast<size_t>(N)) return;
    const int begin = kTeams > 1 ? 0 : static_cast<int>(piece % chunks) * kSpan;
    const int len = K - begin < kSpan ? K - begin : kSpan;
    const float* p = x + col * ld + begin;
    float* out = d + col * ldd + begin;
    const Span span = span_of<(G > 4)>(out, len);
    float* const to = out + span.skew;
    const int label = labels[col];
    const float up = g[col], m = stats[col], s = stats[static_cast<size_t>(N) + col];
    const bool live = label_scored(label, K) && s != 0.f && up != 0.f;
    if (!live) {
        for (int q = team.rank; q < span.quads; q += G) store_quad<NT>(to + 4 * q, Quad(0.f));
        if (team.rank < span.odd) out[span.single(team.rank)] = 0.f;
        return;
    }
    Quad v[kBwdQuads];
#pragma unroll
    for (int k = 0; k < kBwdQuads; ++k) {
        const int q = team.rank + k * G;
        if (q < span.quads) v[k] = load_quad<NT>(p + span.skew + 4 * q);
    }
    const float last = team.rank < span.odd ? p[span.single(team.rank)] : 0.f;
    const bool mine = label >= begin && label < begin + len;
    Grad f{static_cast<float>(-static_cast<double>(up) / static_cast<double>(s)), 0.f, up, 0.f};
    if (mine) {
        f.x = p[label - begin];
        if constexpr (kTeams == 1) __syncthreads();   // the gradient may replace the logits
        else team.sync();
    }
    auto value = [&](float y) { return exp_shifted(y - m, scale) * f.a; };
#pragma unroll
    for (int k = 0; k < kBwdQuads; ++k) {
        const int q = team.rank + k * G;
        if (q < span.quads)
            store_quad<NT>(to + 4 * q, Quad{value(v[k].x), value(v[k].y), value(v[k].z), value(v[k].w)});
    }
    if (team.rank < span.odd) out[span.single(team.rank)] = value(last);
    if (mine) correct_label<false>(team, label - begin, span, m, f, scale, out);
}

int logprobs(float* logp, float* entropy, float* stats, float* scratch, const float* x, const int32_t* labels, int K,
             int N, size_t ld) {
    if (entropy)
        return launch_token_kernel(LogprobHead<true>{exp_scale(1.0), labels, logp, entropy, stats, N}, TokenSums{},
                                   scratch, nullptr, x, K, N, ld, ld);
    return launch_token_kernel(LogprobHead<false>{exp_scale(1.0), labels, logp, nullptr, stats, N}, TokenSums{}, scratch,
                               nullptr, x, K, N, ld, ld);
}

template <int G>
int launch_bwd(float* d, const float* g, const float* x, const int32_t* labels, const float* stats, int K, int N,
               size_t ld, size_t ldd) {
    constexpr int kTeams = kBwdBlock / G, kSpan = 4 * G * kBwdQuads;
    const int chunks = kTeams > 1 ? 1 : (K + kSpan - 1) / kSpan;
    const size_t blocks = (static_cast<size_t>(N) * chunks + kTeams - 1) / kTeams;
    const bool nt = streams_past_cache(static_cast<size_t>(K) * N * 2 * sizeof(float));
    auto kernel = nt ? logprob_bwd_kernel<G, true> : logprob_bwd_kernel<G, false>;
    kernel<<<static_cast<unsigned>(blocks), kBwdBlock, 0, stream()>>>(d, g, x, labels, stats, K, N, chunks, ld, ldd,
                                                                      exp_scale(1.0));
    return launch_rc();
}

int logprobs_bwd(float* d, const float* g, const float* x, const int32_t* labels, const float* stats, int K, int N,
                 size_t ld, size_t ldd) {
    if (K <= 64) return launch_bwd<4>(d, g, x, labels, stats, K, N, ld, ldd);
    if (K <= 256) return launch_bwd<16>(d, g, x, labels, stats, K, N, ld, ldd);
    if (K <= 1024) return launch_bwd<64>(d, g, x, labels, stats, K, N, ld, ldd);
    return launch_bwd<256>(d, g, x, labels, stats, K, N, ld, ldd);
}

// ── paired log ratios ────────────────────────────────────────────────────
// R_s = beta * sum over the scored tokens of sequence s of (logp - ref) [/ their number],
// h = R_chosen - R_rejected.  The slope dl/dh scales both sequences' gradients, so every
// log-probability of a pair is needed before the first gradient of it can be written:
// logprobs over the columns, this kernel over the pairs, logprobs_bwd over the columns.
enum PreferenceKind { kSigmoid = 0, kHinge = 1, kSquared = 2 };

constexpr int kPairsPerLaunch = 64;
struct PairBegins {
    int at[2 * kPairsPerLaunch + 1];
};
constexpr int kPairBlock = 256;
__global__ __launch_bounds__(kPairBlock) void preference_pair_kernel(
    float* g, float* rewards, double* losses, const float* x, const int32_t* labels, const float* stats,
    const float* ref, PairBegins begins, int K, int N, size_t ld, int kind, float beta, float smoothing, int average,
    float scale) {
    __shared__ double slots[4][kPairBlock / kWave];
    const Team<kPairBlock> team{static_cast<int>(threadIdx.x)};
    const int pair = blockIdx.x;
    double reward[2], share[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int lo = begins.at[2 * pair + k], hi = begins.at[2 * pair + k + 1];
        double gain = 0.0, count = 0.0;
        for (int n = lo + team.rank; n < hi; n += kPairBlock) {
            const int label = labels[n];
            const float s = stats[static_cast<size_t>(N) + n];
            if (!label_scored(label, K) || s == 0.f) continue;
            const ColumnSums c{stats[n], static_cast<double>(s), 0.0, 0.0};
            gain += log_prob(x[static_cast<size_t>(n) * ld + label], c) - (ref ? static_cast<double>(ref[n]) : 0.0);
            count += 1.0;
        }
        gain = team.reduce(gain, AddOp{}, slots[2 * k]);
        count = team.reduce(count, AddOp{}, slots[2 * k + 1]);
        share[k] = average ? (count > 0.0 ? 1.0 / count : 0.0) : 1.0;
        reward[k] = static_cast<double>(beta) * gain * share[k];
    }
    const double h = reward[0] - reward[1];
    double loss, slope;   // of h; the comparisons are written so that a NaN stays one
    if (kind == kSigmoid) {
        const double z = exp(-fabs(h)), tail = log1p(z);
        const double down = (h >= 0.0 ? z : 1.0) / (1.0 + z), up = (h >= 0.0 ? 1.0 : z) / (1.0 + z);   // sigma(-h), sigma(h)
        const double sm = static_cast<double>(smoothing);
        loss = (1.0 - sm) * (tail + (h >= 0.0 ? 0.0 : -h)) + sm * (tail + (h >= 0.0 ? h : 0.0));
        slope = -(1.0 - sm) * down + sm * up;
    } else if (kind == kHinge) {
        loss = h >= 1.0 ? 0.0 : 1.0 - h;
        slope = h >= 1.0 ? 0.0 : (h < 1.0 ? -1.0 : h);
    } else {
        const double off = (h - 0.5) / static_cast<double>(beta);
        loss = off * off;
        slope = 2.0 * off / static_cast<double>(beta);
    }
    if (team.rank == 0) {
        rewards[2 * pair] = static_cast<float>(reward[0]);
        rewards[2 * pair + 1] = static_cast<float>(reward[1]);
        losses[pair] = loss;
    }
    if (!g) return;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const double v = (k ? -slope : slope) * share[k] * static_cast<double>(beta) * static_cast<double>(scale);
        for (int n = begins.at[2 * pair + k] + team.rank; n < begins.at[2 * pair + k + 1]; n += kPairBlock)
            g[n] = static_cast<float>(v);
    }
}

}  // namespace
}  // namespace jz

using namespace jz;

JZ_API size_t jzhip_token_scratch_floats(int N, int top) {
    if (N <= 0 || top < 0) return 0;
    return (static_cast<size_t>(8) + static_cast<size_t>(top)) * static_cast<size_t>(N) + kScratchFixed;
}

JZ_API int jzhip_token_logprobs(float* logp, float* entropy, float* stats, float* scratch, const float* logits,
                                const int32_t* labels, int K, int N, int ld) {
    if (!token_args_ok(logits, nullptr, scratch, K, N, ld, ld) || !labels || !scratch || (!logp && !entropy && !stats))
        return -1;
    return logprobs(logp, entropy, stats, scratch, logits, labels, K, N, static_cast<size_t>(ld));
}

JZ_API int jzhip_token_logprobs_bwd(float* dlogits, const float* dlogp, const float* logits, const int32_t* labels,
                                    const float* stats, int K, int N, int ld, int ldd) {
    if (!token_args_ok(logits, dlogits, nullptr, K, N, ld, ldd) || !dlogits || !dlogp || !labels || !stats) return -1;
    return logprobs_bwd(dlogits, dlogp, logits, labels, stats, K, N, static_cast<size_t>(ld),
                        static_cast<size_t>(ldd));
}

JZ_API int jzhip_preference_loss(float* loss_out, float* rewards, float* logp, float* stats, float* dlogits,
                                 float* scratch, const float* logits, const int32_t* labels, const float* ref_logp,
                                 const int* seq_begin, int pairs, int K, int ld, int ldd, int kind, float beta,
                                 float smoothing, int average, float scale) {
    if (!loss_out || !rewards || !logp || !stats || !scratch || !labels || !seq_begin || pairs <= 0) return -1;
    if (pairs > (1 << 18)) return -1;   // the pairs' losses fill half of the fixed part of the scratch
    if (kind < kSigmoid || kind > kSquared || !(beta > 0.f) || !(smoothing >= 0.f && smoothing < 0.5f)) return -1;
    if (kind != kSigmoid && smoothing != 0.f) return -1;
    if (seq_begin[0] != 0) return -1;
    for (int i = 0; i < 2 * pairs; ++i)
        if (seq_begin[i + 1] < seq_begin[i]) return -1;
    const int N = seq_begin[2 * pairs];
    if (!token_args_ok(logits, dlogits, scratch, K, N, ld, ldd)) return -1;
    double* losses = reinterpret_cast<double*>(scratch);
    float* g = scratch + kScratchFixed;
    const size_t ldx = static_cast<size_t>(ld);
    int rc = logprobs(logp, nullptr, stats, scratch, logits, labels, K, N, ldx);
    for (int at = 0; rc == 0 && at < pairs; at += kPairsPerLaunch) {
        const int n = pairs - at < kPairsPerLaunch ? pairs - at : kPairsPerLaunch;
        PairBegins begins = {};
        for (int i = 0; i <= 2 * n; ++i) begins.at[i] = seq_begin[2 * at + i];
        preference_pair_kernel<<<n, kPairBlock, 0, stream()>>>(dlogits ? g : nullptr, rewards + 2 * at, losses + at,
                                                               logits, labels, stats, ref_logp, begins, K, N, ldx,
                                                               kind, beta, smoothing, average, scale);
        rc = launch_rc();
    }
    if (rc == 0 && dlogits) rc = logprobs_bwd(dlogits, g, logits, labels, stats, K, N, ldx, static_cast<size_t>(ldd));
    if (rc) return rc;
    token_fold_kernel<double><<<1, kFoldBlock, 0, stream()>>>(loss_out, losses, pairs, 0, static_cast<double>(scale));
    return launch_rc();
}
