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
    double lq;   // the teacher's logit, then log q_j
    int id;      // -1: none
    float x;     // the student's logit
};

template <bool REST>
struct DistillHead {
    static constexpr bool kEntropy = false, kRest = REST, kTeacher = true, kWrites = true;
    struct Early {
        float w;
    };
    ExpScale scale;
    const float* teacher;
    const int32_t* ids;
    const float *lse, *weight;   // lse set iff REST; weight may be null
    float *token_loss, *part;    // token_loss may be null
    float* picked;               // the student's logits of the entries for a later kernel, or null
    size_t ldt;
    int top;
    float temperature;

    // entries, then one bit per logit (K = 0: the entries alone)
    __host__ __device__ size_t team_bytes(int K) const {
        return sizeof(Entry) * static_cast<size_t>(top) + (static_cast<size_t>(K) + 127) / 128 * 16;
    }
    __device__ unsigned* bits(char* own) const { return reinterpret_cast<unsigned*>(own + sizeof(Entry) * top); }
    // The entries among the logits [begin, begin + len).
    template <class T>
    __device__ void mark(const T& team, unsigned* all, size_t col, int begin, int len) const {
        for (int j = team.rank; j < top; j += T::kSize) {
            const int at = ids[col * ldt + j];
            if (at >= begin && at < begin + len) atomicOr(&all[(at - begin) >> 5], 1u << ((at - begin) & 31));
        }
    }
    __device__ bool live(size_t col, int) const { return !(weight && weight[col] == 0.f); }
    __device__ int label(size_t) const { return -1; }
    __device__ Early early(size_t col, const float*) const { return Early{weight ? weight[col] : 1.f}; }
    __device__ void write(size_t col, float each, float loss) const {
        if (token_loss) token_loss[col] = each;
        part[col] = loss;
    }
    __device__ void idle(size_t col) const { write(col, 0.f, 0.f); }
    // The teacher's distribution, by one wave or less; false where it has none.  all: one bit per
    // logit, cleared, left with the entries marked (null: not kept).  x: the student's column (null:
    // its logits at the entries are in `picked`).
    template <class T>
    __device__ bool prologue(const T& lead, char* own, unsigned* all, size_t col, int K, const float* x) const {
        Entry* e = reinterpret_cast<Entry*>(own);
        bool twice = all == nullptr;
        float big = -INFINITY;
        for (int j = lead.rank; j < top; j += T::kSize) {
            const int id = ids[col * ldt + j];
            const bool is = id >= 0 && id < K;
            const float t = teacher[col * ldt + j];
            e[j].id = is ? id : -1;
            e[j].lq = static_cast<double>(t);
            e[j].x = !is ? 0.f : x ? x[id] : picked[col * top + j];
            if (!is) continue;
            big = fmaxf(big, t);
            if (all) {
                const unsigned bit = 1u << (id & 31);
                twice |= (atomicOr(&all[id >> 5], bit) & bit) != 0u;
            }
        }
        lead.sync();
        if (lead.lanes(twice ? 1.f : 0.f, LargerOp{}) != 0.f) {
            // An id counts once, the first time: the later ones are dropped.  From the back, so that
            // each is compared with ids that are still there.
            const int rounds = (top + T::kSize - 1) / T::kSize;
            big = -INFINITY;
            for (int r = rounds - 1; r >= 0; --r) {
                const int j = lead.rank + r * T::kSize;
                bool drop = false;
                if (j < top)
                    for (int i = 0; i < j; ++i) drop |= e[i].id == e[j].id;
                lead.sync();
                if (j < top && drop) e[j].id = -1;
                lead.sync();
                if (j < top && e[j].id >= 0) big = fmaxf(big, static_cast<float>(e[j].lq));
            }
        }
        const double over = 1.0 / static_cast<double>(temperature);
        float some = 0.f;
        if constexpr (REST) {
            const double norm = static_cast<double>(lse[col]);
            for (int j = lead.rank; j < top; j += T::kSize) {
                e[j].lq = e[j].lq * over - norm;
                if (e[j].id >= 0) some = 1.f;
            }
            some = lead.lanes(some, LargerOp{});
        } else {
            big = lead.lanes(big, LargerOp{});
            double z = 0.0;
            for (int j = lead.rank; j < top; j += T::kSize) {
                const double t = e[j].lq, u = (t - static_cast<double>(big)) * over;
                e[j].lq = u;
                if (e[j].id < 0) continue;
                z += exp64(u);
                if (big != -INFINITY || t != t) some = 1.f;
            }
            z = log64(lead.lanes(z, AddOp{}));
            some = lead.lanes(some, LargerOp{});
            for (int j = lead.rank; j < top; j += T::kSize) e[j].lq -= z;
        }
        lead.sync();
        return some != 0.f;
    }
    template <class T>
    __device__ Grad finish(const T& lead, char* own, const Early& early, size_t col, const ColumnSums& c) const {
        const Entry* e = reinterpret_cast<const Entry*>(own);
        const double T_ = static_cast<double>(temperature), over = 1.0 / T_, logs = log64(c.s);
        const double w = static_cast<double>(early.w);
        double Q = 0.0, each = 0.0;
        for (int j = lead.rank; j < top; j += T::kSize) {
            if (e[j].id < 0) continue;
            const double q = exp64(e[j].lq);
            if (picked) picked[col * top + j] = e[j].x;
            Q += q;
            // an entry of no mass adds nothing, whatever the student gives it; a NaN stays one
            if (q != 0.0)
                each += q * (e[j].lq - ((static_cast<double>(e[j].x) - static_cast<double>(c.m)) * over - logs));
        }
        Q = lead.lanes(Q, AddOp{});
        each = lead.lanes(each, AddOp{});
        const double inv = 1.0 / c.s;
        double out = 0.0;   // what the rest subtracts
        if constexpr (REST) {
            double r = 1.0 - Q;
            r = r < 0.0 ? 0.0 : r;
            if (r != 0.0) each += r * (log64(r) - log64(c.rest * inv));
            Q += r;
            out = c.rest > 0.0 ? r / c.rest : Q * inv;
        }
        each *= T_ * T_;
        if (lead.rank == 0) write(col, static_cast<float>(each), static_cast<float>(w * each));
        return Grad{static_cast<float>(T_ * w * (Q * inv - out)), 0.f, static_cast<float>(T_ * w * (Q * inv)),
                    static_cast<float>(T_ * w)};
    }
    // f.g: Q*T*w/s, f.x: T*w
    template <class T>
    __device__ void correct(const T& team, char* own, size_t, float m, const Grad& f, float* out, int) const {
        const Entry* e = reinterpret_cast<const Entry*>(own);
        for (int j = team.rank; j < top; j += T::kLanes)
            if (e[j].id >= 0)
                out[e[j].id] = exp_shifted(e[j].x - m, scale) * f.g -
                               static_cast<float>(static_cast<double>(f.x) * exp64(e[j].lq));
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
    float* picked = K > kMaxWhole ? part + static_cast<size_t>(8) * N : nullptr;
    const TokenSums totals{loss_out, part, 1};
    if (teacher_lse)
        return launch_token_kernel(DistillHead<true>{exp_scale(temperature), teacher, ids, teacher_lse, weight,
                                                     token_loss, part, picked, ldq, top, temperature},
                                   totals, scratch, dlogits, logits, K, N, ldx, ldg);
    return launch_token_kernel(DistillHead<false>{exp_scale(temperature), teacher, ids, nullptr, weight, token_loss,
                                                  part, picked, ldq, top, temperature},
                               totals, scratch, dlogits, logits, K, N, ldx, ldg);
}
