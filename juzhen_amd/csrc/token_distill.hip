// Distillation from a teacher of which, per token, the `top` largest logits are known:
// the divergence of the student from the teacher and its gradient in one pass.
//
// Classes g of a token: the teacher's entries, and where the teacher's normaliser is given
// everything else as one more class.  With u_j = teacher_j / T and p = softmax(x / T)
//   q_j = exp(u_j - lse)  (lse: the teacher's, or over its entries),  q_rest = max(0, 1 - sum q_j)
//   P_j = p_(id_j),  P_rest = sum of the p_i that are no entry
//   L   = w * T^2 * sum_g q_g log(q_g / P_g)
//   d_i = w * T * (Q p_i - q_g(i) p_i / P_g(i)),  Q = sum_g q_g
// P_rest is summed over its own members: 1 - sum P_j would lose it where the entries cover
// nearly all of the student's mass, and the gradient divides by it.
#include "token_loss.hpp"

namespace jz {
namespace {

constexpr int kMaxTop = 512;

struct DistillShared {
    int id[kMaxTop];       // -1: no entry
    int keep[kMaxTop];
    float x[kMaxTop];      // teacher's logit, then the student's
    double lq[kMaxTop];    // log q_j
    float a_known, scale_q;   // gradient of an entry: e*a_known - scale_q*q
};

template <bool REST>
struct DistillHead {
    static constexpr bool kEntropy = false, kRest = REST;
    using Shared = DistillShared;
    ExpScale scale;
    const float* teacher;
    const int32_t* ids;
    const float *lse, *weight;   // lse set iff REST; weight may be null
    float *token_loss, *part;    // token_loss may be null
    size_t ldt;
    int top;
    float temperature;

    __device__ bool live(size_t col, int) const { return !(weight && weight[col] == 0.f); }
    __device__ void write(size_t col, float each, float loss) const {
        if (token_loss) token_loss[col] = each;
        part[col] = loss;
    }
    __device__ void idle(size_t col) const { write(col, 0.f, 0.f); }
    // The teacher's distribution; false where it has none.
    template <class T>
    __device__ bool prologue(const T& team, Shared& sh, size_t col, int K) const {
        for (int j = team.rank; j < top; j += T::kSize) {
            const int id = ids[col * ldt + j];
            sh.id[j] = id >= 0 && id < K ? id : -1;
            sh.x[j] = teacher[col * ldt + j];
        }
        team.sync();
        float big = -INFINITY;
        bool some = false, nan = false;
        for (int j = team.rank; j < top; j += T::kSize) {
            bool keep = sh.id[j] >= 0;
            for (int i = 0; i < j && keep; ++i) keep = sh.id[i] != sh.id[j];   // an id counts once
            sh.keep[j] = keep;
            if (!keep) continue;
            some = true;
            nan |= sh.x[j] != sh.x[j];
            big = fmaxf(big, sh.x[j]);
        }
        team.sync();
        for (int j = team.rank; j < top; j += T::kSize)
            if (!sh.keep[j]) sh.id[j] = -1;
        const double T_ = static_cast<double>(temperature);
        if constexpr (REST) {
            const double all = static_cast<double>(lse[col]);
            for (int j = team.rank; j < top; j += T::kSize) sh.lq[j] = static_cast<double>(sh.x[j]) / T_ - all;
            some = team.any(some);
        } else {
            big = team.max(big);
            some = big != -INFINITY || team.any(nan);
            double z = 0.0;
            for (int j = team.rank; j < top; j += T::kSize)
                if (sh.id[j] >= 0) z += exp((static_cast<double>(sh.x[j]) - static_cast<double>(big)) / T_);
            z = log(team.sum(z));
            for (int j = team.rank; j < top; j += T::kSize)
                sh.lq[j] = (static_cast<double>(sh.x[j]) - static_cast<double>(big)) / T_ - z;
        }
        team.sync();
        return some;
    }
    __device__ bool known(const Shared& sh, int i) const {
        bool k = false;
        for (int j = 0; j < top; ++j) k |= sh.id[j] == i;
        return k;
    }
    template <class T>
    __device__ Coef finish(const T& team, Shared& sh, size_t col, const ColumnSums& c, const float* x) const {
        const double T_ = static_cast<double>(temperature), s = static_cast<double>(c.s), logs = log(s);
        const double w = weight ? static_cast<double>(weight[col]) : 1.0;
        double Q = 0.0, each = 0.0;
        for (int j = team.rank; j < top; j += T::kSize) {
            if (sh.id[j] < 0) continue;
            const double q = exp(sh.lq[j]);
            const float xj = x[sh.id[j]];
            sh.x[j] = xj;
            Q += q;
            // an entry of no mass adds nothing, whatever the student gives it; a NaN stays one
            if (q != 0.0) each += q * (sh.lq[j] - ((static_cast<double>(xj) - static_cast<double>(c.m)) / T_ - logs));
        }
        Q = team.sum(Q);
        each = team.sum(each);
        double out = 0.0;   // what the rest subtracts
        if constexpr (REST) {
            const double left = static_cast<double>(c.rest);
            double r = 1.0 - Q;
            r = r < 0.0 ? 0.0 : r;
            if (r != 0.0) each += r * (log(r) - log(left / s));
            Q += r;
            out = left > 0.0 ? r / left : Q / s;
        }
        each *= T_ * T_;
        if (team.rank == 0) {
            sh.a_known = static_cast<float>(T_ * w * (Q / s));
            sh.scale_q = static_cast<float>(T_ * w);
            write(col, static_cast<float>(each), static_cast<float>(w * each));
        }
        team.sync();
        return Coef{static_cast<float>(T_ * w * (Q / s - out)), 0.f};
    }
    template <class T>
    __device__ void correct(const T& team, Shared& sh, size_t, const ColumnSums& c, const Coef&, float* out) const {
        for (int j = team.rank; j < top; j += T::kSize)
            if (sh.id[j] >= 0)
                out[sh.id[j]] = exp_shifted(sh.x[j] - c.m, scale) * sh.a_known -
                                static_cast<float>(static_cast<double>(sh.scale_q) * exp(sh.lq[j]));
    }
};

}  // namespace
}  // namespace jz

using namespace jz;

JZ_API int jzhip_distill_topk(float* loss_out, float* token_loss, float* dlogits, float* scratch,
                              const float* logits, const float* teacher, const int32_t* ids, const float* teacher_lse,
                              const float* weight, int K, int top, int N, int ld, int ldd, int ldt,
                              float temperature) {
    if (!token_args_ok(logits, dlogits, scratch, K, N, ld, ldd) || !loss_out || !scratch || !teacher || !ids) return -1;
    if (top <= 0 || top > kMaxTop || ldt < top) return -1;
    if (!(temperature >= 1e-3f && temperature <= 1e3f)) return -1;
    const size_t ldx = static_cast<size_t>(ld), ldg = static_cast<size_t>(ldd), ldq = static_cast<size_t>(ldt);
    int rc;
    if (teacher_lse)
        rc = launch_token_kernel(DistillHead<true>{exp_scale(temperature), teacher, ids, teacher_lse, weight,
                                                   token_loss, scratch, ldq, top, temperature},
                                 dlogits, logits, K, N, ldx, ldg);
    else
        rc = launch_token_kernel(DistillHead<false>{exp_scale(temperature), teacher, ids, nullptr, weight, token_loss,
                                                    scratch, ldq, top, temperature},
                                 dlogits, logits, K, N, ldx, ldg);
    if (rc) return rc;
    token_fold_kernel<float><<<1, kFoldBlock, 0, stream()>>>(loss_out, scratch, N, 0, 1.0);
    return launch_rc();
}
