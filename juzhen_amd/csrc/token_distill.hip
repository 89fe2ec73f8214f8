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

// One of a column's entries, in LDS.
struct Entry {
    double lq;   // log q_j
    int id;      // -1: none
    float x;     // the teacher's logit, then the student's
};

template <bool REST>
struct DistillHead {
    static constexpr bool kEntropy = false, kRest = REST, kTeamwork = true, kWrites = true;
    ExpScale scale;
    const float* teacher;
    const int32_t* ids;
    const float *lse, *weight;   // lse set iff REST; weight may be null
    float *token_loss, *part;    // token_loss may be null
    float* picked;               // students' logits of the entries for a later kernel, or null
    size_t ldt;
    int top;
    float temperature;

    // entries, then one bit per logit (K = 0: the entries alone)
    __host__ __device__ size_t team_bytes(int K) const {
        return sizeof(Entry) * static_cast<size_t>(top) + (REST ? (static_cast<size_t>(K) + 127) / 128 * 16 : 0);
    }
    __device__ unsigned* bits(char* own) const { return reinterpret_cast<unsigned*>(own + sizeof(Entry) * top); }
    template <class T>
    __device__ void mark(const T& team, unsigned* all, size_t col, int begin, int len) const {
        for (int j = team.rank; j < top; j += T::kSize) {
            const int at = ids[col * ldt + j];
            if (at >= begin && at < begin + len) atomicOr(&all[(at - begin) >> 5], 1u << ((at - begin) & 31));
        }
    }
    __device__ bool live(size_t col, int) const { return !(weight && weight[col] == 0.f); }
    __device__ int label(size_t) const { return -1; }
    __device__ void write(size_t col, float each, float loss) const {
        if (token_loss) token_loss[col] = each;
        part[col] = loss;
    }
    __device__ void idle(size_t col) const { write(col, 0.f, 0.f); }
    // The teacher's distribution; false where it has none.
    template <class T>
    __device__ bool prologue(const T& team, char* own, size_t col, int K) const {
        Entry* e = reinterpret_cast<Entry*>(own);
        for (int j = team.rank; j < top; j += T::kSize) {
            const int id = ids[col * ldt + j];
            e[j].id = id >= 0 && id < K ? id : -1;
            e[j].x = teacher[col * ldt + j];
        }
        team.sync();
        float big = -INFINITY;
        bool some = false, nan = false;
        for (int j = team.rank; j < top; j += T::kSize) {
            const int id = e[j].id;
            bool keep = id >= 0;
            for (int i = 0; i < j; ++i) keep = keep && e[i].id != id;   // an id counts once
            e[j].lq = keep ? 1.0 : 0.0;
            if (!keep) continue;
            some = true;
            nan |= e[j].x != e[j].x;
            big = fmaxf(big, e[j].x);
        }
        team.sync();   // everyone has compared
        const double T_ = static_cast<double>(temperature);
        if constexpr (REST) {
            const double all = static_cast<double>(lse[col]);
            for (int j = team.rank; j < top; j += T::kSize) {
                if (e[j].lq == 0.0) e[j].id = -1;
                e[j].lq = static_cast<double>(e[j].x) / T_ - all;
            }
            some = team.any(some);
        } else {
            big = team.max(big);
            some = big != -INFINITY || team.any(nan);
            double z = 0.0;
            for (int j = team.rank; j < top; j += T::kSize) {
                if (e[j].lq == 0.0) e[j].id = -1;
                e[j].lq = (static_cast<double>(e[j].x) - static_cast<double>(big)) / T_;
                if (e[j].id >= 0) z += exp(e[j].lq);
            }
            z = log(team.sum(z));
            for (int j = team.rank; j < top; j += T::kSize) e[j].lq -= z;
        }
        return some;
    }
    template <class T>
    __device__ Grad finish(const T& team, char* own, size_t col, const ColumnSums& c, const float* x) const {
        Entry* e = reinterpret_cast<Entry*>(own);
        const double T_ = static_cast<double>(temperature), logs = one_at_a_time(log(c.s));
        const double w = weight ? static_cast<double>(weight[col]) : 1.0;
        double Q = 0.0, each = 0.0;
        for (int j = team.rank; j < top; j += T::kSize) {
            if (e[j].id < 0) continue;
            const double q = one_at_a_time(exp(e[j].lq));
            const float xj = x[e[j].id];
            e[j].x = xj;
            if (picked) picked[col * top + j] = xj;
            Q += q;
            // an entry of no mass adds nothing, whatever the student gives it; a NaN stays one
            if (q != 0.0) each += q * (e[j].lq - ((static_cast<double>(xj) - static_cast<double>(c.m)) / T_ - logs));
        }
        Q = team.sum(Q);
        each = team.sum(each);
        double out = 0.0;   // what the rest subtracts
        if constexpr (REST) {
            double r = 1.0 - Q;
            r = r < 0.0 ? 0.0 : r;
            if (r != 0.0) {
                const double logr = one_at_a_time(log(r));
                each += r * (logr - one_at_a_time(log(c.rest / c.s)));
            }
            Q += r;
            out = c.rest > 0.0 ? r / c.rest : Q / c.s;
        }
        each *= T_ * T_;
        if (team.rank == 0) write(col, static_cast<float>(each), static_cast<float>(w * each));
        return Grad{static_cast<float>(T_ * w * (Q / c.s - out)), 0.f, static_cast<float>(T_ * w * (Q / c.s)),
                    static_cast<float>(T_ * w)};
    }
    // The entries of a column whose prologue has run again, as finish left them.
    template <class T>
    __device__ void restore(const T& team, char* own, size_t col, const Grad&) const {
        Entry* e = reinterpret_cast<Entry*>(own);
        for (int j = team.rank; j < top; j += T::kSize)
            if (e[j].id >= 0) e[j].x = picked[col * top + j];
    }
    // f.g: Q*T*w/s, f.x: T*w
    template <class T>
    __device__ void correct(const T& team, char* own, size_t, float m, const Grad& f, float* out, int) const {
        const Entry* e = reinterpret_cast<const Entry*>(own);
        team.sync();   // behind the sweep that wrote these elements as any other
        for (int j = team.rank; j < top; j += T::kSize)
            if (e[j].id >= 0)
                out[e[j].id] = exp_shifted(e[j].x - m, scale) * f.g -
                               static_cast<float>(static_cast<double>(f.x) * exp(e[j].lq));
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
    if (top <= 0 || top > kMaxTop || top > K || ldt < top) return -1;
    if (!(temperature >= 1e-3f && temperature <= 1e3f)) return -1;
    const size_t ldx = static_cast<size_t>(ld), ldg = static_cast<size_t>(ldd), ldq = static_cast<size_t>(ldt);
    float* part = scratch + kScratchFixed;
    float* picked = part + static_cast<size_t>(8) * N;
    int rc;
    if (teacher_lse)
        rc = launch_token_kernel(DistillHead<true>{exp_scale(temperature), teacher, ids, teacher_lse, weight,
                                                   token_loss, part, picked, ldq, top, temperature},
                                 scratch, dlogits, logits, K, N, ldx, ldg);
    else
        rc = launch_token_kernel(DistillHead<false>{exp_scale(temperature), teacher, ids, nullptr, weight, token_loss,
                                                    part, picked, ldq, top, temperature},
                                 scratch, dlogits, logits, K, N, ldx, ldg);
    if (rc) return rc;
    token_fold_kernel<float><<<1, kFoldBlock, 0, stream()>>>(loss_out, part, N, 0, 1.0);
    return launch_rc();
}
