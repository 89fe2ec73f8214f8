// Distillation from a teacher of which, per token, the `top` largest logits are known:
// the divergence of the student from the teacher and its gradient in one pass.
//
// Classes g of a token: the teacher's entries, and where the teacher's normaliser is given
// everything else as one more class.  With u_j = teacher_j / T and p = softmax(x / T)
//   q_j = exp(u_j - lse)  (lse: the teacher's, or over its entries),  q_rest = max(0, 1 - sum q_j)
//   P_j = p_(id_j),  P_rest = sum of the p_i that are no entry
//   L   = w * T^2 * sum_g q_g log(q_g / P_g)
//   d_i = w * T * (Q p_i - q_g(i) p_i / P_g(i)),  Q = sum_g q_g
// P_rest is summed over its own members, relative to the largest of them: 1 - sum P_j, and a sum
// relative to the column's maximum, would lose it where the student gives the entries nearly all
// of its mass (logits 87 T above the others: exp underflows), and the gradient divides by it.  The
// sweep leaves the entries out, and finish() adds them in 64 bits: with m', s' of the rest,
//   M = max(m', entries),  S = s' exp((m' - M)/T) + sum_j exp((x_j - M)/T)
//   log P_rest = (m' - M)/T + log s' - log S
//   d_i = e'_i * w T (Q exp((m' - M)/T)/S - q_rest/s'),  e'_i = exp((x_i - m')/T)   (i in the rest)
#include "token_loss.hpp"

#include <cfloat>

namespace jz {
namespace {

constexpr int kMaxTop = 512;

// A column's entries in LDS.
struct Entries {
    double *lq, *q;   // the teacher's logit, then log q_j; q_j (64 bits: the divergence is a small difference)
    float* x;         // the student's logit
    int* id;          // -1: none
    static constexpr size_t kBytes = 2 * sizeof(double) + sizeof(float) + sizeof(int);
    __device__ Entries(char* own, int top)
        : lq(reinterpret_cast<double*>(own)), q(lq + top), x(reinterpret_cast<float*>(q + top)),
          id(reinterpret_cast<int*>(x + top)) {}
};

template <bool REST>
struct DistillHead {
    static constexpr bool kEntropy = false, kRest = REST, kTeacher = true, kWrites = true;
    static constexpr int kSums = 1;
    struct Early {
        float w;
        // from the prologue: REST: maximum and sum of the student's entries; sum of the q_j
        float m;
        double s, Q;
    };
    ExpScale scale;
    const float* teacher;
    const int32_t* ids;
    const float *lse, *weight;   // lse set iff REST; weight may be null
    float* token_loss;           // may be null
    TokenParts to;
    float* picked;               // gradients at the entries, for a later kernel where the column is cut into chunks
    size_t ldt;
    int top;
    float temperature;
    bool chunked = false;

    // entries, then one bit per logit and a word more (K = 0: the entries alone)
    __host__ __device__ size_t entry_bytes() const { return (Entries::kBytes * static_cast<size_t>(top) + 15) / 16 * 16; }
    __host__ __device__ size_t team_bytes(int K) const {
        return entry_bytes() + (K ? (static_cast<size_t>(K) + 159) / 128 * 16 : 0);
    }
    __device__ unsigned* bits(char* own) const { return reinterpret_cast<unsigned*>(own + entry_bytes()); }
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
    __device__ Early early(size_t col, const float*) const { return Early{weight ? weight[col] : 1.f, -INFINITY, 0.0, 0.0}; }
    __device__ void write(size_t col, double each, double loss) const {
        if (token_loss) token_loss[col] = static_cast<float>(each);
        to.at(col, 0) = loss;
    }
    __device__ void idle(size_t col) const { write(col, 0.0, 0.0); }
    // The teacher's distribution, by one wave or less; false where it has none.  all: one bit per
    // logit, cleared, left with the entries marked (null: not kept).
    template <class T>
    __device__ bool prologue(const T& lead, char* own, unsigned* all, size_t col, int K, const float* x,
                             Early& early) const {
        const Entries e(own, top);
        bool twice = all == nullptr;
        float big = -INFINITY;
        for (int j = lead.rank; j < top; j += T::kSize) {
            const int id = ids[col * ldt + j];
            const bool is = id >= 0 && id < K;
            const float t = teacher[col * ldt + j];
            e.id[j] = is ? id : -1;
            e.lq[j] = static_cast<double>(t);
            if (!is) continue;
            e.x[j] = x[id];
            if (REST) early.m = fmaxf(early.m, e.x[j]);
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
                    for (int i = 0; i < j; ++i) drop |= e.id[i] == e.id[j];
                lead.sync();
                if (j < top && drop) e.id[j] = -1;
                lead.sync();
                if (j < top && e.id[j] >= 0) big = fmaxf(big, static_cast<float>(e.lq[j]));
            }
        }
        const double over = 1.0 / static_cast<double>(temperature);
        float some = 0.f;
        double Q = 0.0;
        if constexpr (REST) {
            const double norm = static_cast<double>(lse[col]);
            early.m = lead.lanes(early.m, LargerOp{});
            const double shift = early.m == -INFINITY ? 0.0 : static_cast<double>(early.m);
            for (int j = lead.rank; j < top; j += T::kSize) {
                if (e.id[j] < 0) continue;
                early.s += exp64((static_cast<double>(e.x[j]) - shift) * over);
                const double u = e.lq[j] * over - norm, q = exp64(u);
                e.lq[j] = u;
                e.q[j] = q;
                Q += q;
                some = 1.f;
            }
            Q = lead.lanes(Q, AddOp{});
            early.s = lead.lanes(early.s, AddOp{});
        } else {
            big = lead.lanes(big, LargerOp{});
            double z = 0.0;
            for (int j = lead.rank; j < top; j += T::kSize) {
                if (e.id[j] < 0) continue;
                const double t = e.lq[j], u = (t - static_cast<double>(big)) * over, q = exp64(u);
                e.lq[j] = u;
                e.q[j] = q;
                z += q;
                if (big != -INFINITY || t != t) some = 1.f;
            }
            z = lead.lanes(z, AddOp{});
            const double logz = log64(z), inv = 1.0 / z;
            for (int j = lead.rank; j < top; j += T::kSize) {
                if (e.id[j] < 0) continue;
                e.lq[j] -= logz;
                e.q[j] *= inv;
            }
            Q = z * inv;   // 1, or NaN
        }
        early.Q = Q;
        return lead.lanes(some, LargerOp{}) != 0.f;
    }
    // f.g: Q*T*w/s, f.x: T*w, f.b: the maximum of the whole column
    __device__ float entry_gradient(const Entries& e, int j, const Grad& f) const {
        return static_cast<float>(static_cast<double>(exp_shifted(e.x[j] - f.b, scale) * f.g) - static_cast<double>(f.x) * e.q[j]);
    }
    template <class T>
    __device__ Grad finish(const T& lead, char* own, const Early& early, size_t col, const ColumnSums& c) const {
        const Entries e(own, top);
        const double T_ = static_cast<double>(temperature), over = 1.0 / T_;
        const double w = static_cast<double>(early.w);
        float big = c.m;
        double s = c.s, below = 1.0;   // below: what the rest's exponentials are to those relative to `big`
        if constexpr (REST) {
            big = fmaxf(c.m, early.m);
            const bool higher = c.m >= early.m;
            const double f = exp64(-fabs((static_cast<double>(c.m) - static_cast<double>(early.m)) * over));
            below = c.m == -INFINITY ? 0.0 : higher ? 1.0 : f;
            s = c.s * below + early.s * (early.m == -INFINITY ? 0.0 : higher && c.m != early.m ? f : 1.0);
        }
        const double logs = log64(s);
        double Q = early.Q, each = 0.0;
        for (int j = lead.rank; j < top; j += T::kSize) {
            // an entry of no mass adds nothing, whatever the student gives it; a NaN stays one
            if (e.id[j] < 0 || e.q[j] == 0.0) continue;
            each += e.q[j] *
                    (e.lq[j] - ((static_cast<double>(e.x[j]) - static_cast<double>(big)) * over - logs));
        }
        each = lead.lanes(each, AddOp{});
        const double inv = 1.0 / s;
        double out = 0.0;   // what the rest subtracts
        if constexpr (REST) {
            double r = 1.0 - Q;
            r = r < 0.0 ? 0.0 : r;
            // the type's lowest value beside larger logits is a mask
            const double rest = c.m == -FLT_MAX && big > c.m ? 0.0 : c.s;
            if (r != 0.0)
                each += r * (log64(r) - ((static_cast<double>(c.m) - static_cast<double>(big)) * over + log64(rest) - logs));
            Q += r;
            if (rest > 0.0) out = r / rest;
        }
        each *= T_ * T_;
        if (lead.rank == 0) write(col, each, w * each);
        const Grad f{static_cast<float>(T_ * w * (Q * below * inv - out)), big, static_cast<float>(T_ * w * (Q * inv)),
                     static_cast<float>(T_ * w)};
        if (chunked)
            for (int j = lead.rank; j < top; j += T::kSize)
                if (e.id[j] >= 0) picked[col * top + j] = entry_gradient(e, j, f);
        return f;
    }
    template <class T>
    __device__ void correct(const T& lead, char* own, size_t, float, const Grad& f, float* out) const {
        const Entries e(own, top);
        for (int j = lead.rank; j < top; j += T::kSize)
            if (e.id[j] >= 0) out[e.id[j]] = entry_gradient(e, j, f);
    }
    // The entries among the logits [begin, begin + len), whose gradients `picked` holds.
    template <class T>
    __device__ void correct_chunk(const T& team, char* own, size_t col, int begin, int len, float* out) const {
        int* id = reinterpret_cast<int*>(own);
        for (int j = team.rank; j < top; j += T::kSize) id[j] = ids[col * ldt + j];
        team.sync();
        for (int j = team.rank; j < top; j += T::kSize) {
            if (id[j] < begin || id[j] >= begin + len) continue;
            bool first = true;
            for (int i = 0; i < j; ++i) first &= id[i] != id[j];
            if (first) out[id[j] - begin] = picked[col * top + j];
        }
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
    double* part = reinterpret_cast<double*>(scratch + kScratchFixed);
    float* picked = scratch + kScratchFixed + static_cast<size_t>(8) * N;   // behind the 8 floats a token
    const TokenSums totals{loss_out, part, 1};
    const TokenParts to{part, static_cast<size_t>(N)};
    if (teacher_lse)
        return launch_token_kernel(DistillHead<true>{exp_scale(temperature), teacher, ids, teacher_lse, weight,
                                                     token_loss, to, picked, ldq, top, temperature},
                                   totals, scratch, dlogits, logits, K, N, ldx, ldg);
    return launch_token_kernel(DistillHead<false>{exp_scale(temperature), teacher, ids, nullptr, weight, token_loss,
                                                  to, picked, ldq, top, temperature},
                               totals, scratch, dlogits, logits, K, N, ldx, ldg);
}
