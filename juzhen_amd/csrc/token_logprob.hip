// Log-probabilities of one label per token, their gradient, and the paired
// log-ratio (preference) loss built on the two.
#include "token_loss.hpp"

namespace jz {
namespace {

// EXACT: log p in 64 bits as well, for a loss over many tokens.
template <bool ENTROPY, bool EXACT>
struct LogprobHead {
    static constexpr bool kEntropy = ENTROPY, kRest = false, kTeacher = false, kWrites = false;
    static constexpr int kSums = 0;
    struct Early {
        float x;   // the label's logit
    };
    ExpScale scale;
    const int32_t* labels;
    float *logp, *entropy, *stats;   // each may be null
    int N;
    double* exact;                   // EXACT

    __host__ __device__ size_t team_bytes(int) const { return 0; }
    __device__ bool live(size_t col, int K) const { return label_scored(labels[col], K); }
    __device__ int label(size_t col) const { return labels[col]; }
    __device__ Early early(size_t col, const float* x) const { return Early{x[labels[col]]}; }
    __device__ void write(size_t col, double lp, float h, float m, float s) const {
        if (logp) logp[col] = static_cast<float>(lp);
        if (EXACT) exact[col] = lp;
        if (ENTROPY) entropy[col] = h;
        if (stats) {
            stats[col] = m;
            stats[static_cast<size_t>(N) + col] = s;
        }
    }
    __device__ void idle(size_t col) const { write(col, 0.0, 0.f, 0.f, 0.f); }
    template <class T>
    __device__ Grad finish(const T& lead, char*, const Early& e, size_t col, const ColumnSums& c) const {
        const double lp = log_prob(e.x, c);
        const float h = ENTROPY ? static_cast<float>(entropy_of(c)) : 0.f;
        if (lead.rank == 0) write(col, lp, h, c.m, static_cast<float>(c.s));
        return Grad{};
    }
    template <class T>
    __device__ void correct(const T&, char*, size_t, float, const Grad&, float*) const {}
};

// d_i = g*(delta_i - e_i/s) from the maximum and the sum of the forward call: no reduction
// is left, every element is read and written once.  A team takes NV*G quads of a column,
// from quad `base` on; the one that begins at 0 its single logits as well.  Long columns are
// cut into workgroups of 512 threads with one quad each, which keeps the accesses in flight
// closest together (32000 x 4194, a quarter of the tokens unscored: 151 us, 2 quads 173; 256
// threads with 1, 2, 4 quads 149, 158, 176, but 163 to 151 at 50001 x 2684).
constexpr int kBwdBlock = 256, kBwdLong = 512, kBwdTeams = 1024;   // kBwdTeams: up to so many logits a wave or less
struct BwdArgs {
    float* d;
    const float *g, *x;
    const int32_t* labels;
    const float* stats;
    int K, N;
    size_t ld, ldd;
    ExpScale scale;
    int first = 0;   // column of the launch's first workgroup
};
template <int G, int NV, bool NT>
__device__ __forceinline__ void bwd_span(const BwdArgs& a, const Team<G>& team, size_t col, int base) {
    const float* p = a.x + col * a.ld;
    float* out = a.d + col * a.ldd;
    const Span span = span_of<(G > 4)>(out, a.K);
    const int singles = base == 0 ? span.odd : 0;
    const int label = a.labels[col];
    const float up = a.g[col], m = a.stats[col], s = a.stats[static_cast<size_t>(a.N) + col];
    const bool live = label_scored(label, a.K) && s != 0.f && up != 0.f;
    if (!live) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int q = base + team.rank + k * G;
            if (q < span.quads) store_quad<NT>(out + span.skew + 4 * static_cast<size_t>(q), Quad(0.f));
        }
        if (team.rank < singles) out[span.single(team.rank)] = 0.f;
        return;
    }
    Quad v[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int q = base + team.rank + k * G;
        if (q < span.quads) v[k] = load_quad<NT>(p + span.skew + 4 * static_cast<size_t>(q));
    }
    const float last = team.rank < singles ? p[span.single(team.rank)] : 0.f;
    const int quad = (label - span.skew) / 4;
    const bool mine = label < span.skew || quad >= span.quads ? base == 0 : quad >= base && quad < base + NV * G;
    Grad f{static_cast<float>(-static_cast<double>(up) / static_cast<double>(s)), 0.f, up, 0.f};
    if (mine) {
        f.x = p[label];
        team.sync();   // the gradient may replace the logits
    }
    auto value = [&](float y) { return exp_shifted(y - m, a.scale) * f.a; };
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int q = base + team.rank + k * G;
        if (q < span.quads)
            store_quad<NT>(out + span.skew + 4 * static_cast<size_t>(q),
                           Quad{value(v[k].x), value(v[k].y), value(v[k].z), value(v[k].w)});
    }
    if (team.rank < singles) out[span.single(team.rank)] = value(last);
    if (mine) {
        team.sync();
        if (team.rank == 0) correct_label<false>(label, m, f, a.scale, out);
    }
}

// The sum of the pairs' losses, which the gradient's first workgroup adds up on the way.
struct PairTotal {
    float* out;   // null: none
    const double* losses;
    int pairs;
    double scale;
};
// G <= 64: a column per team; else `chunks` workgroups per column
template <int G, bool NT>
__global__ __launch_bounds__(G > kWave ? G : kBwdBlock) void logprob_bwd_kernel(BwdArgs a, PairTotal total,
                                                                                FastDiv chunks) {
    constexpr int kBlock = G > kWave ? G : kBwdBlock, kTeams = kBlock / G;
    __shared__ double slots[kBlock / kWave];
    if (total.out && blockIdx.x == 0) fold_parts<kBlock>(total.out, total.losses, total.pairs, total.scale, slots);
    const Team<G> team{static_cast<int>(threadIdx.x % G)};
    const int n = kTeams > 1 ? static_cast<int>(blockIdx.x * kTeams + threadIdx.x / G) : static_cast<int>(fdiv(blockIdx.x, chunks));
    if (kTeams > 1 && n >= a.N) return;
    const int base = kTeams > 1 ? 0 : static_cast<int>(blockIdx.x - n * chunks.d) * G;
    bwd_span<G, (kTeams > 1 ? kGroupQuads : 1), NT>(a, team, static_cast<size_t>(a.first) + n, base);
}

template <bool ENTROPY, bool EXACT>
int logprobs(float* logp, float* entropy, float* stats, double* exact, float* scratch, const float* x,
             const int32_t* labels, int K, int N, size_t ld) {
    return launch_token_kernel(LogprobHead<ENTROPY, EXACT>{exp_scale(1.0), labels, logp, entropy, stats, N, exact},
                               TokenSums{}, scratch, nullptr, x, K, N, ld, ld);
}

template <int G>
int launch_bwd(BwdArgs a, PairTotal total) {
    constexpr int kBlock = G > kWave ? G : kBwdBlock, kTeams = kBlock / G;
    const int chunks = kTeams > 1 ? 1 : (a.K / 4 + G - 1) / G;
    const bool nt = streams_past_cache(static_cast<size_t>(a.K) * a.N * 2 * sizeof(float));
    auto kernel = nt ? logprob_bwd_kernel<G, true> : logprob_bwd_kernel<G, false>;
    // A thread per quad: what a launch may have (2^32 threads) is 2^34 logits.  Columns beyond go in
    // launches of their own.  (Columns of small teams are few enough: kMaxTokens.)
    const int most = kTeams > 1 ? a.N : static_cast<int>(kMaxThreads / kBlock) / chunks;
    for (; a.first < a.N; a.first += most) {
        const int n = a.N - a.first < most ? a.N - a.first : most;
        const unsigned blocks = static_cast<unsigned>((static_cast<size_t>(n) * chunks + kTeams - 1) / kTeams);
        kernel<<<blocks, kBlock, 0, stream()>>>(a, total, make_fastdiv(chunks));
        const int rc = launch_rc();
        if (rc) return rc;
        total.out = nullptr;
    }
    return 0;
}
int logprobs_bwd(const BwdArgs& a, const PairTotal& total) {
    if (a.K <= 64) return launch_bwd<4>(a, total);
    if (a.K <= 256) return launch_bwd<16>(a, total);
    if (a.K <= kBwdTeams) return launch_bwd<64>(a, total);
    return launch_bwd<kBwdLong>(a, total);
}

// ── paired log ratios ────────────────────────────────────────────────────
// R_s = beta * sum over the scored tokens of sequence s of (logp - ref) [/ their number],
// h = R_chosen - R_rejected.  The slope dl/dh scales both sequences' gradients, so every
// log-probability of a pair is needed before the first gradient of it can be written:
// logprobs over the columns, this kernel over the pairs, logprobs_bwd over the columns.
// The second read is what this costs, 12 bytes per logit instead of 8, at 5.9 TB/s (4939 x
// 32000: 70 + 6 + 185 us).  It cannot come cheaper out of the memory-side cache, which is no
// faster than the memory (a copy of 128 MB 7.2 TB/s, of 1 GB 6.5): pairs taken in groups that
// fit it 366 us in all, the gradient's sweep from the last column back no change.
enum PreferenceKind { kSigmoid = 0, kHinge = 1, kSquared = 2 };

constexpr int kPairsPerLaunch = 64;
struct PairBegins {
    int at[2 * kPairsPerLaunch + 1];
};
struct PairArgs {
    float* g;   // dl/dlogp of every token, or null
    float* rewards;
    double* losses;
    const double* logp;
    const int32_t* labels;
    const float *stats, *ref;   // ref may be null
    PairBegins begins;
    int K, N, kind, average;
    float beta, smoothing, scale;
};
// One pair by one team; slots: 4*kWaves values in LDS.  token(n, v): whether token n is scored, and its
// log-probability; put(n, g): its dl/dlogp.
template <class T, class Token, class Put>
__device__ __forceinline__ void take_pair(const PairArgs& a, const T& team, int pair, double* slots, double* loss_out,
                                          Token token, Put put) {
    double reward[2], share[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int lo = a.begins.at[2 * pair + k], hi = a.begins.at[2 * pair + k + 1];
        double gain = 0.0, count = 0.0;
        for (int n = lo + team.rank; n < hi; n += T::kSize) {
            double v;
            if (!token(n, v)) continue;
            gain += v - (a.ref ? static_cast<double>(a.ref[n]) : 0.0);
            count += 1.0;
        }
        gain = team.reduce(gain, AddOp{}, slots + 2 * k * T::kWaves);
        count = team.reduce(count, AddOp{}, slots + (2 * k + 1) * T::kWaves);
        share[k] = a.average ? (count > 0.0 ? 1.0 / count : 0.0) : 1.0;
        reward[k] = static_cast<double>(a.beta) * gain * share[k];
    }
    const double h = reward[0] - reward[1];
    double loss, slope;   // of h; the comparisons are written so that a NaN stays one
    if (a.kind == kSigmoid) {
        const double z = exp64(-fabs(h)), tail = z < 1e-5 ? z - 0.5 * z * z : log64(1.0 + z);   // log(1 + z)
        const double down = (h >= 0.0 ? z : 1.0) / (1.0 + z), up = (h >= 0.0 ? 1.0 : z) / (1.0 + z);   // sigma(-h), sigma(h)
        const double sm = static_cast<double>(a.smoothing);
        // -h, h: of the terms -log sigma(h) = tail + max(-h, 0), -log sigma(-h) = tail + max(h, 0); what has
        // no part is left out (h is infinite where a label has probability 0)
        loss = tail + (h >= 0.0 ? (sm != 0.0 ? sm * h : 0.0) : (1.0 - sm) * -h);
        slope = -(1.0 - sm) * down + sm * up;
    } else if (a.kind == kHinge) {
        loss = h >= 1.0 ? 0.0 : 1.0 - h;
        slope = h >= 1.0 ? 0.0 : (h < 1.0 ? -1.0 : h);
    } else {
        const double off = (h - 0.5) / static_cast<double>(a.beta);
        loss = off * off;
        slope = 2.0 * off / static_cast<double>(a.beta);
    }
    if (team.rank == 0) {
        a.rewards[2 * pair] = static_cast<float>(reward[0]);
        a.rewards[2 * pair + 1] = static_cast<float>(reward[1]);
        *loss_out = loss;
    }
    if (!a.g) return;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const double v = (k ? -slope : slope) * share[k] * static_cast<double>(a.beta) * static_cast<double>(a.scale);
        for (int n = a.begins.at[2 * pair + k] + team.rank; n < a.begins.at[2 * pair + k + 1]; n += T::kSize)
            put(n, static_cast<float>(v));
    }
}
constexpr int kPairBlock = 1024;
__global__ __launch_bounds__(kPairBlock) void preference_pair_kernel(PairArgs a) {
    __shared__ double slots[4 * kPairBlock / kWave];
    take_pair(
        a, Team<kPairBlock>{static_cast<int>(threadIdx.x)}, blockIdx.x, slots, a.losses + blockIdx.x,
        [&](int n, double& v) {
            v = a.logp[n];
            return label_scored(a.labels[n], a.K) && a.stats[static_cast<size_t>(a.N) + n] != 0.f;
        },
        [&](int n, float g) { a.g[n] = g; });
}

// Short sequences over few classes: one workgroup keeps every column in registers from the
// log-probabilities to the gradient, with the pairs between two barriers.  The work is less
// than the launches and the round trips to memory of the general way (2 pairs, 90 tokens x 256:
// 4 launches 16 us; one workgroup that reads again for the gradient 10 us; this 6 us).
constexpr int kSmallBlock = 1024, kSmallRounds = 2;
template <int G>
__global__ __launch_bounds__(kSmallBlock, 4) void preference_small_kernel(LogprobHead<false, true> head, PairArgs pairs,
                                                                          BwdArgs a, PairTotal total) {
    using Head = LogprobHead<false, true>;
    constexpr int kTeams = kSmallBlock / G;
    __shared__ double logp[kSmallRounds * kTeams], losses[kPairsPerLaunch];
    __shared__ float up[kSmallRounds * kTeams];
    __shared__ bool scored[kSmallRounds * kTeams];
    const Team<G> team{static_cast<int>(threadIdx.x % G)};
    const int slot = threadIdx.x / G;
    Quad v[kSmallRounds][kGroupQuads];
    float last[kSmallRounds], picked[kSmallRounds], group[kSmallRounds];
    int label[kSmallRounds];
    ColumnSums c[kSmallRounds];
    bool live[kSmallRounds];
    Span span[kSmallRounds];
#pragma unroll
    for (int r = 0; r < kSmallRounds; ++r) {
        const int n = slot + r * kTeams;
        label[r] = n < a.N ? a.labels[n] : -1;
    }
#pragma unroll
    for (int r = 0; r < kSmallRounds; ++r) {
        const float* p = a.x + (slot + r * kTeams) * a.ld;
        live[r] = label_scored(label[r], a.K);
        span[r] = span_of<(G > 4)>(p, a.K);
        last[r] = -INFINITY;
        picked[r] = 0.f;
#pragma unroll
        for (int k = 0; k < kGroupQuads; ++k) {
            const int q = team.rank + k * G;
            v[r][k] = Quad(-INFINITY);
            if (live[r] && q < span[r].quads) v[r][k] = load_quad<false>(p + span[r].skew + 4 * q);
        }
        if (live[r]) picked[r] = p[label[r]];
        if (live[r] && team.rank < span[r].odd) last[r] = p[span[r].single(team.rank)];
    }
#pragma unroll
    for (int r = 0; r < kSmallRounds; ++r) {
        const int n = slot + r * kTeams;
        if (n >= a.N) continue;
        c[r] = ColumnSums{-INFINITY, 0.0, 0.0};
        const Group g = take_group<Head>(v[r], head.scale, [](int) { return 0u; });
        group[r] = g.m;
        add_group<Head>(c[r], g, head.scale);
        if (team.rank < span[r].odd) add_group<Head>(c[r], take_one(last[r]), head.scale);
        scale_sums<Head>(c[r], team.reduce(c[r].m, LargerOp{}, static_cast<float*>(nullptr)), head.scale);
        c[r].s = team.reduce(c[r].s, AddOp{}, static_cast<double*>(nullptr));
        live[r] = live[r] && !(c[r].m == -INFINITY && c[r].s == c[r].s);
        const double lp = live[r] ? log_prob(picked[r], c[r]) : 0.0;
        if (team.rank == 0) {
            head.write(n, lp, 0.f, live[r] ? c[r].m : 0.f, live[r] ? static_cast<float>(c[r].s) : 0.f);
            logp[n] = lp;
            scored[n] = live[r];
        }
        __builtin_amdgcn_sched_barrier(0);   // one round's registers at a time
    }
    __syncthreads();
    const Team<kWave> wave{static_cast<int>(threadIdx.x % kWave)};
    for (int p = threadIdx.x / kWave; p < total.pairs; p += kSmallBlock / kWave)
        take_pair(
            pairs, wave, p, nullptr, losses + p,
            [&](int n, double& x) {
                x = logp[n];
                return scored[n];
            },
            [&](int n, float g) { up[n] = g; });
    __syncthreads();
    if (threadIdx.x < kWave) fold_parts<kWave>(total.out, losses, total.pairs, total.scale, nullptr);
    if (!a.d) return;
#pragma unroll
    for (int r = 0; r < kSmallRounds; ++r) {
        const int n = slot + r * kTeams;
        if (n >= a.N) continue;
        float* out = a.d + n * a.ldd;
        const float g = live[r] ? up[n] : 0.f;
        const bool write = live[r] && g != 0.f;
        // (a maximum of -inf that is scored holds a NaN)
        const float f = write ? static_cast<float>(-static_cast<double>(g) / c[r].s) : 0.f;
        const float fg = write ? (c[r].m == -INFINITY ? 1.f : exp_shifted(group[r] - c[r].m, head.scale)) * f : 0.f;
#pragma unroll
        for (int k = 0; k < kGroupQuads; ++k) {
            const int q = team.rank + k * G;
            const Quad e = v[r][k];
            if (q < span[r].quads)
                store_quad<false>(out + span[r].skew + 4 * q,
                                  write ? Quad{e.x * fg, e.y * fg, e.z * fg, e.w * fg} : Quad(0.f));
        }
        if (team.rank < span[r].odd)
            out[span[r].single(team.rank)] = write ? exp_shifted(last[r] - c[r].m, head.scale) * f : 0.f;
        team.sync();
        if (write && team.rank == 0) correct_label<false>(label[r], c[r].m, Grad{f, 0.f, g, picked[r]}, head.scale, out);
    }
}
template <int G>
int launch_small(const LogprobHead<false, true>& head, const PairArgs& pairs, const BwdArgs& bwd, const PairTotal& total) {
    preference_small_kernel<G><<<1, kSmallBlock, 0, stream()>>>(head, pairs, bwd, total);
    return launch_rc();
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
    auto run = entropy ? logprobs<true, false> : logprobs<false, false>;
    return run(logp, entropy, stats, nullptr, scratch, logits, labels, K, N, static_cast<size_t>(ld));
}

JZ_API int jzhip_token_logprobs_bwd(float* dlogits, const float* dlogp, const float* logits, const int32_t* labels,
                                    const float* stats, int K, int N, int ld, int ldd) {
    if (!token_args_ok(logits, dlogits, nullptr, K, N, ld, ldd) || !dlogits || !dlogp || !labels || !stats) return -1;
    return logprobs_bwd(BwdArgs{dlogits, dlogp, logits, labels, stats, K, N, static_cast<size_t>(ld),
                                static_cast<size_t>(ldd), exp_scale(1.0)},
                        PairTotal{});
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
    double* exact = reinterpret_cast<double*>(scratch + kScratchFixed);
    float* g = dlogits ? scratch + kScratchFixed + 2 * static_cast<size_t>(N) : nullptr;
    const size_t ldx = static_cast<size_t>(ld);
    const BwdArgs bwd{dlogits, g, logits, labels, stats, K, N, ldx, static_cast<size_t>(ldd), exp_scale(1.0)};
    const PairTotal total{loss_out, losses, pairs, static_cast<double>(scale)};
    PairArgs args{g, rewards, losses, exact, labels, stats, ref_logp, {}, K, N, kind, average, beta, smoothing, scale};
    auto begins = [&](int at, int n) {
        for (int i = 0; i <= 2 * n; ++i) args.begins.at[i] = seq_begin[2 * at + i];
        args.rewards = rewards + 2 * at;
        args.losses = losses + at;
    };
    if (K <= 1024 && pairs <= kPairsPerLaunch) {
        const int lanes = K <= 64 ? 4 : K <= 256 ? 16 : 64;
        if (N <= kSmallRounds * kSmallBlock / lanes) {
            begins(0, pairs);
            const LogprobHead<false, true> head{exp_scale(1.0), labels, logp, nullptr, stats, N, exact};
            if (lanes == 4) return launch_small<4>(head, args, bwd, total);
            if (lanes == 16) return launch_small<16>(head, args, bwd, total);
            return launch_small<64>(head, args, bwd, total);
        }
    }
    int rc = logprobs<false, true>(logp, nullptr, stats, exact, scratch, logits, labels, K, N, ldx);
    for (int at = 0; rc == 0 && at < pairs; at += kPairsPerLaunch) {
        const int n = pairs - at < kPairsPerLaunch ? pairs - at : kPairsPerLaunch;
        begins(at, n);
        preference_pair_kernel<<<n, kPairBlock, 0, stream()>>>(args);
        rc = launch_rc();
    }
    if (rc) return rc;
    if (dlogits) return logprobs_bwd(bwd, total);
    // in the order of the gradient's first workgroup
    if (K <= kBwdTeams) token_fold_kernel<kBwdBlock><<<1, kBwdBlock, 0, stream()>>>(loss_out, losses, pairs, 0, total.scale);
    else token_fold_kernel<kBwdLong><<<1, kBwdLong, 0, stream()>>>(loss_out, losses, pairs, 0, total.scale);
    return launch_rc();
}
