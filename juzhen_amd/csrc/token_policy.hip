// Clipped policy-gradient loss over the logits of sampled tokens, with a KL term
// against a reference model and an entropy bonus; value and gradient in one pass.
//
//   r = exp(logp - old),  f = r*A,  c = clamp(r, 1 - lo, 1 + hi)*A,  u = ref - logp
//   L = w * ( -min(f, c) + kl*(e^u - u - 1) - ent*H )
//   G = dL/dlogp = w * ( -[f <= c] f - kl*(e^u - 1) )
//   d_i = G*(delta_i - p_i) + w*ent*p_i*(log p_i + H)
// With log p_i = t_i - log s the second line is e_i*(a + b*t_i) plus G at the label, so the
// whole gradient is one more sweep over the exponentials.
#include "token_loss.hpp"

namespace jz {
namespace {

template <bool ENTROPY>
struct PolicyHead {
    static constexpr bool kEntropy = ENTROPY, kRest = false, kTeacher = false, kWrites = true;
    static constexpr int kSums = 4;
    struct Early {
        float x, old, ref, adv, w;   // x: the label's logit
    };
    ExpScale scale;
    const int32_t* labels;
    const float *old_logp, *ref_logp, *advantage, *weight;   // ref_logp, weight may be null
    float* logp;                                             // may be null
    TokenParts to;
    float clip_low, clip_high, kl_coef, entropy_coef;

    __host__ __device__ size_t team_bytes(int) const { return 0; }
    __device__ bool live(size_t col, int K) const {
        return label_scored(labels[col], K) && !(weight && weight[col] == 0.f);
    }
    __device__ int label(size_t col) const { return labels[col]; }
    __device__ Early early(size_t col, const float* x) const {
        return Early{x[labels[col]], old_logp[col], ref_logp ? ref_logp[col] : 0.f, advantage[col],
                     weight ? weight[col] : 1.f};
    }
    __device__ void write(size_t col, float lp, double loss, double kl, double cut, double h) const {
        if (logp) logp[col] = lp;
        to.at(col, 0) = loss;
        to.at(col, 1) = kl;
        to.at(col, 2) = cut;
        to.at(col, 3) = h;
    }
    __device__ void idle(size_t col) const { write(col, 0.f, 0.0, 0.0, 0.0, 0.0); }
    template <class T>
    __device__ Grad finish(const T& lead, char*, const Early& e, size_t col, const ColumnSums& c) const {
        const double w = static_cast<double>(e.w), adv = static_cast<double>(e.adv);
        const double logs = log64(c.s);
        const double lp = (static_cast<double>(e.x) - static_cast<double>(c.m)) - logs;
        const double ratio = exp64(lp - static_cast<double>(e.old));
        const double low = 1.0 - static_cast<double>(clip_low), high = 1.0 + static_cast<double>(clip_high);
        const double held = (ratio < low ? low : ratio > high ? high : ratio) * adv;
        const double open = ratio * adv;
        const bool cut = open > held;   // a NaN counts as not cut and stays one
        double kl = 0.0, g = cut ? 0.0 : -open;
        double loss = -(cut ? held : open), h = 0.0;
        if (ref_logp) {
            const double u = static_cast<double>(e.ref) - lp;
            const ExpTail em = exp_tail64(u);
            kl = em.tail;
            if (kl_coef != 0.f) {
                g -= static_cast<double>(kl_coef) * em.minus1;
                loss += static_cast<double>(kl_coef) * kl;
            }
        }
        const double inv = 1.0 / c.s;
        double a = -g * w, b = 0.0;
        if constexpr (ENTROPY) {
            h = logs - c.et * inv;
            loss -= static_cast<double>(entropy_coef) * h;
            b = static_cast<double>(entropy_coef) * w;
            a += b * (h - logs);
        }
        if (lead.rank == 0)
            write(col, static_cast<float>(lp), w * loss, w * kl, cut ? w : 0.0, w * h);
        return Grad{static_cast<float>(a * inv), static_cast<float>(b * inv), static_cast<float>(g * w), e.x};
    }
    template <class T>
    __device__ void correct(const T& lead, char*, size_t col, float m, const Grad& f, float* out) const {
        if (lead.rank == 0) correct_label<ENTROPY>(labels[col], m, f, scale, out);
    }
};

}  // namespace
}  // namespace jz

using namespace jz;

JZ_API int jzhip_policy_loss(float* sums, float* logp, float* dlogits, float* scratch, const float* logits,
                             const int32_t* labels, const float* old_logp, const float* ref_logp,
                             const float* advantage, const float* weight, int K, int N, int ld, int ldd,
                             float clip_low, float clip_high, float kl_coef, float entropy_coef) {
    if (!token_args_ok(logits, dlogits, scratch, K, N, ld, ldd) || !sums || !scratch || !labels || !old_logp || !advantage)
        return -1;
    if (!(clip_low >= 0.f && clip_low <= 1.f) || !(clip_high >= 0.f) || !(kl_coef >= 0.f) || !(entropy_coef >= 0.f))
        return -1;
    if (kl_coef != 0.f && !ref_logp) return -1;
    const size_t ldx = static_cast<size_t>(ld), ldg = static_cast<size_t>(ldd);
    double* part = reinterpret_cast<double*>(scratch + kScratchFixed);   // the 8 floats a token
    const TokenSums totals{sums, part, 4};
    const TokenParts to{part, static_cast<size_t>(N)};
    if (entropy_coef != 0.f)
        return launch_token_kernel(PolicyHead<true>{exp_scale(1.0), labels, old_logp, ref_logp, advantage, weight,
                                                    logp, to, clip_low, clip_high, kl_coef, entropy_coef},
                                   totals, scratch, dlogits, logits, K, N, ldx, ldg);
    return launch_token_kernel(PolicyHead<false>{exp_scale(1.0), labels, old_logp, ref_logp, advantage, weight, logp,
                                                 to, clip_low, clip_high, kl_coef, 0.f},
                               totals, scratch, dlogits, logits, K, N, ldx, ldg);
}
