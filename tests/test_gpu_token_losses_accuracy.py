"""Losses on logits: how near the results are, element by element.

Bounds, with u = 2^-24, t = x - m and C = 2 log K + 8.  An exponential is off by (2 |t| + 4) u relative:
the difference t, its product with log2(e) and the hardware's 2^v (below 2 u), once relative to the largest of a
thread's sixteen logits and once for that one; a tree of sixteen fp32 additions adds 4 u, everything further is
64 bits.  As sum e |t| / sum e <= log K, a column's sum of exponentials is off by C u relative.  Exponentials
that are 1 are counted apart and exact: with s = 1 + b (one largest logit), log s is off by b/s C u.
  log p, entropy            the same absolute, and half a step of the result
  off-label gradient        p_i |up| (2 |t_i| + 4 + C + 8) u: 8 for the coefficient's and the products' roundings;
                            |up| 2^-118 for what lies below 2^-126
  at the label              up - up p: up u more
Values of a loss are sums in 64 bits of 64-bit terms, rounded once."""
import ctypes as C_

import numpy as np
import pytest

import token_loss_reference as ref
from test_gpu_token_losses import SENTINEL, columns, grad_buffer, kept, same, scratch, take
from util import dev_empty, dptr, to_dev, to_host

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F = np.float32
TINY = 2.0 ** -118

# every way a column is cut (lanes of a wave, one wave, workgroups that keep it or half of it, chunks)
CUTS = [(5, 40), (40, 40), (100, 40), (200, 20), (300, 20), (900, 20), (1500, 20), (3000, 9), (6000, 9), (12000, 5), (30000, 5),
        (40000, 3), (50001, 70), (70000, 100), (140001, 3), (5001, 530), (12001, 520), (20001, 515), (40000, 600)]


def bound(K):
    return 2 * np.log(K) + 8


def parts(x):
    """p, t, the share of all but the largest."""
    x = x.astype(np.float64)
    t = x - x.max(1, keepdims=True)
    e = np.exp(t)
    s = e.sum(1)
    return e / s[:, None], t, np.log(s), (s - 1.0) / s


@pytest.mark.parametrize("K,N", CUTS)
def test_log_probabilities_of_likely_tokens(gpu, K, N):
    """A label that holds all but 1e-6 to a half of the mass: log p is as exact as that rest of it."""
    print(f"likely K {K} N {N}", flush=True)
    r = np.random.default_rng(K)
    x = r.normal(0, 1, (N, K)).astype(F)
    labels = r.integers(0, K, N).astype(np.int32)
    rest = 10.0 ** r.uniform(-6, -0.3, N)
    x[np.arange(N), labels] = (np.log(np.exp(x.astype(np.float64)).sum(1)) - np.log(rest)).astype(F)
    some = np.arange(N)[:12]
    p, t, logs, b = parts(x[some])
    lp, h, _, _ = ref.logprobs(x[some], labels[some])
    tol = 1.05 * b * bound(K) * U + (np.abs(lp) + 1e-8) * U
    dx, dl, sc = columns(x, K), to_dev(labels), scratch(N)
    out, ent, alone = dev_empty(N), dev_empty(N), dev_empty(N)
    gpu.token_logprobs(dptr(out), dptr(ent), None, dptr(sc), dptr(dx), dptr(dl), K, N, K)
    same(to_host(out)[some], lp, tol, "logp")
    # of the e_i t_i an element below the largest: its own exponential, t_i and the product
    same(to_host(ent)[some], h, tol + (np.sum(p * np.abs(t) * (2 * np.abs(t) + 8 + bound(K)), 1) + np.abs(h)) * U, "entropy")
    gpu.token_logprobs(dptr(alone), None, None, dptr(sc), dptr(dx), dptr(dl), K, N, K)
    same(to_host(alone)[some], lp, tol, "logp alone")
    zero = kept(to_dev(np.zeros(N, F)))
    for e in (0.0, 0.01):
        gpu.policy_loss(kept(dev_empty(4)), dptr(out), kept(dev_empty(N * K)), dptr(sc), dptr(dx), dptr(dl), zero, None, zero,
                        None, K, N, K, K, 0.2, 0.2, 0.0, e)
        same(to_host(out)[some], lp, tol, "logp beside a policy loss")
    # distillation from one entry that is the label: the loss is -log p
    ids, one = kept(to_dev(labels)), kept(to_dev(np.ones(N, F)))
    gpu.distill_topk(kept(dev_empty(1)), dptr(out), None, dptr(sc), dptr(dx), one, ids, None, None, K, 1, N, K, K, 1, 1.0)
    same(to_host(out)[some], -lp, tol, "distillation")


@pytest.mark.parametrize("K,N,off", [(K, N, off) for off in (0, 1, 3) for K, N in CUTS if N <= 100 or off == 0])
def test_gradients_element_by_element(gpu, K, N, off):
    """Relative to each element, at any alignment."""
    print(f"elements K {K} N {N} off {off}", flush=True)
    r = np.random.default_rng(K + off)
    ld, top = K + off, min(4, K - 1)
    x = r.normal(0, 3, (N, K)).astype(F)
    labels = r.integers(0, K, N).astype(np.int32)
    labels[1] = -1
    x[2, : K // 2] -= F(60.0)
    flat = np.full(N * ld + off, np.nan, F)
    flat[off:].reshape(N, ld)[:, :K] = x
    base, d, sc = to_dev(flat), to_dev(np.full(N * ld + off, SENTINEL, F)), scratch(N, top)
    px, pd = C_.c_void_p(base.data_ptr() + 4 * off), C_.c_void_p(d.data_ptr() + 4 * off)
    dl = to_dev(labels)
    some = np.concatenate([np.arange(min(N, 6)), [N - 1]])
    xs, ls = x[some], labels[some]
    live = ls >= 0
    p, t, logs, _ = parts(xs)
    H = np.where(live, ref.logprobs(xs, ls)[1], 0.0)
    c = bound(K)
    rel = 2 * np.minimum(np.abs(t), 100.0) + 12 + c
    hit = np.zeros(xs.shape, bool)
    hit[np.flatnonzero(live), ls[live]] = True

    def check(want, tol, what):
        got = to_host(d)[off:].reshape(N, ld)
        assert (got[:, K:] == SENTINEL).all()
        same(got[some, :K], want, tol, what)
        d.fill_(float(SENTINEL))

    up = r.normal(0, 1, N).astype(F)
    du = to_dev(up)
    g = np.where(live, np.abs(up[some]), 0.0)[:, None]
    stats = dev_empty(2 * N)
    gpu.token_logprobs(None, None, dptr(stats), dptr(sc), px, dptr(dl), K, N, ld)
    gpu.token_logprobs_bwd(pd, dptr(du), px, dptr(dl), dptr(stats), K, N, ld, ld)
    check(ref.logprobs_bwd(xs, ls, up[some].astype(np.float64)), g * (p * rel + 2 * hit) * U + g * TINY, "log-probabilities")

    lp = np.where(labels >= 0, x[np.arange(N), np.maximum(labels, 0)] - np.log(np.exp(x.astype(np.float64)).sum(1)), 0.0)
    old, rlp = (lp + 0.1).astype(F), (lp - 0.3).astype(F)
    w = (r.random(N) + 0.5).astype(F)
    args = [to_dev(v) for v in (old, rlp, up, w)]
    for kl, ent in ((0.0, 0.0), (0.1, 0.02)):
        klf, entf = float(F(kl)), float(F(ent))
        _, _, want, G = ref.policy(xs, ls, old[some], rlp[some] if kl else None, up[some], w[some], 0.0, float(F(0.5)), klf, entf)
        do, dr, da, dw = (dptr(v) for v in args)
        gpu.policy_loss(kept(dev_empty(4)), None, pd, dptr(sc), px, dptr(dl), do, dr if kl else None, da, dw, K, N, ld, ld, 0.0,
                        0.5, kl, ent)
        ww = np.where(live, w[some], 0.0)[:, None]
        G, gerr = np.abs(G)[:, None], ww * 2 * (np.abs(up[some])[:, None] + klf) * c      # ratio and e^gap follow log p: C u
        tol = p * (G * rel + gerr) + hit * (2 * G + gerr)
        # p (log p + H): the two cancel; H is off by C (1 + log K) u at most
        tol += ww * entf * p * (np.abs(t) + logs[:, None] + H[:, None] + 1) * (rel + c * (1 + np.log(K)))
        check(want, tol * U + ww * TINY * (1 + g), f"policy {kl}")

    begin = [0, N // 2, N]
    gpu.preference_loss(kept(dev_empty(1)), kept(dev_empty(2)), kept(dev_empty(N)), dptr(stats), pd, dptr(sc), px, dptr(dl),
                        None, (C_.c_int * 3)(*begin), 1, K, ld, ld, 1, 0.25, 0.0, 1, 1.0)
    n_scored = [int((labels[a:b] >= 0).sum()) for a, b in zip(begin, begin[1:])]
    R = [0.25 * lp[a:b][labels[a:b] >= 0].sum() / max(1, k) for a, b, k in zip(begin, begin[1:], n_scored)]
    assert abs(R[0] - R[1] - 1.0) > 1e-3
    slope = -1.0 if R[0] - R[1] < 1.0 else 0.0
    pref = np.array([slope * (1 if n < N // 2 else -1) * 0.25 / max(1, n_scored[0 if n < N // 2 else 1]) for n in some])
    g2 = np.where(live, np.abs(pref), 0.0)[:, None]
    check(ref.logprobs_bwd(xs, ls, np.where(live, pref, 0.0)), g2 * (p * rel + 2 * hit) * U + g2 * TINY, "preference")

    ids = np.stack([r.choice(K, top, replace=False) for _ in range(N)]).astype(np.int32)
    tea = r.normal(0, 1, (N, top)).astype(F)
    lse = (np.log(np.exp(tea.astype(np.float64)).sum(1)) + 0.25).astype(F)
    dt, di, dz, dw = (to_dev(v.reshape(-1)) for v in (tea, ids, lse, w))
    known = np.zeros(xs.shape, bool)
    np.put_along_axis(known, ids[some].astype(np.int64), True, 1)
    for tail in (False, True):
        _, _, want = ref.distill(xs, tea[some], ids[some], lse[some] if tail else None, w[some], 1.0)
        gpu.distill_topk(kept(dev_empty(1)), None, pd, dptr(sc), px, dptr(dt), dptr(di), dptr(dz) if tail else None, dptr(dw), K,
                         top, N, ld, ld, top, 1.0)
        ww = w[some][:, None].astype(np.float64)
        share = np.where(known, 0.0, p / np.where(known, 0.0, p).sum(1, keepdims=True))
        tol = ww * ((p + (share if tail else 0.0)) * rel + known * 4)
        check(want, tol * U + 2 * ww * TINY, f"distillation {tail}")


def test_values_of_losses_that_cancel(gpu):
    """Terms of 64 bits, summed in 64 bits: with weights that nearly cancel the result is the small difference.
    One class: log p = 0, the ratio exp(-old) is 1 and a term -w A, 48 bits long; then equal columns, whose
    per-token divergence is one number, under weights of both signs."""
    r = np.random.default_rng(1)
    for N in (64, 3000, 20000):
        w = r.normal(0, 1, N).astype(F)
        adv = r.normal(0, 1, N).astype(F)
        wa = w.astype(np.float64) * adv
        adv[-1] = F(-wa[:-1].sum() / w[-1]) if abs(w[-1]) > 1e-3 else adv[-1]
        want = -np.sum(w.astype(np.float64) * adv)
        out, sc = dev_empty(4), scratch(N)
        x, lab, z = kept(to_dev(np.zeros(N, F))), kept(to_dev(np.zeros(N, np.int32))), kept(to_dev(np.zeros(N, F)))
        gpu.policy_loss(dptr(out), None, None, dptr(sc), x, lab, z, None, kept(to_dev(adv)), kept(to_dev(w)), 1, N, 1, 1, 0.2,
                        0.2, 0.0, 0.0)
        assert abs(to_host(out)[0] - want) <= U * abs(want) + 1e-13 * np.abs(wa).sum()
        # a reference 1 away: e^-1 of KL per token, under the same weights, minus their mean in the last one
        w[-1] = F(-w[:-1].astype(np.float64).sum())
        total, kl = w.astype(np.float64).sum(), np.exp(-1.0)
        gpu.policy_loss(dptr(out), None, None, dptr(sc), x, lab, z, kept(to_dev(np.full(N, -1, F))), z, kept(to_dev(w)), 1, N, 1,
                        1, 0.2, 0.2, 0.25, 0.0)
        assert abs(to_host(out)[1] - total * kl) <= U * abs(total) + 1e-9 * abs(total) + 1e-13 * np.abs(w).sum()
        K = 50
        row, ids = r.normal(0, 1, K).astype(F), np.array([3, 7], np.int32)
        tea = np.array([1.0, 0.5], F)
        for lse in (None, np.full(N, 1.6, F)):
            gpu.distill_topk(dptr(out), None, None, dptr(sc), kept(to_dev(np.tile(row, N))), kept(to_dev(np.tile(tea, N))),
                             kept(to_dev(np.tile(ids, N))), None if lse is None else kept(to_dev(lse)), kept(to_dev(w)), K, 2, N, K,
                             K, 2, 1.0)
            each = ref.distill(row[None], tea[None], ids[None], None if lse is None else lse[:1], None, 1.0)[1][0]
            assert abs(to_host(out)[0] - each * total) <= (2 * bound(K) + 1 + each) * U * abs(total) + 1e-13 * np.abs(w).sum() * each


def test_rewards_of_long_answers(gpu):
    """The sum of 1000 small differences of log-probabilities.  An exponential's error is (3 roundings, |t| up to 12
    where it has weight, twice) 14 u rms and independent of the others', log s averages it over the logits that share
    the mass: under 2 u rms per token, six deviations of their sum 12 sqrt(1000) u, and a tenth of a u per token for
    what is common to them.  (An exponential with one-part log2(e) is off by 1.3e-8 t, 1.2 u per token here.)"""
    K, n = 32000, 1000
    r = np.random.default_rng(3)
    x = r.normal(0, 2, (2 * n, K)).astype(F)
    labels = r.integers(0, K, 2 * n).astype(np.int32)
    lp = np.concatenate([ref.logprobs(x[a:a + 250], labels[a:a + 250])[0] for a in range(0, 2 * n, 250)])
    rlp = lp.astype(F)
    want = np.array([np.sum(lp[:n] - rlp[:n]), np.sum(lp[n:] - rlp[n:])])
    rew, N = dev_empty(2), 2 * n
    gpu.preference_loss(kept(dev_empty(1)), dptr(rew), kept(dev_empty(N)), kept(dev_empty(2 * N)), None, kept(scratch(N)),
                        kept(columns(x, K)), kept(to_dev(labels)), kept(to_dev(rlp)), (C_.c_int * 3)(0, n, N), 1, K, K, K, 0, 1.0,
                        0.0, 0, 1.0)
    assert np.max(np.abs(to_host(rew) - want)) <= (12 * np.sqrt(n) + 0.1 * n) * U + U * np.abs(want).max()


@pytest.mark.parametrize("K", [8, 32, 200, 500])
@pytest.mark.parametrize("T", [1.0, 2.0])
def test_divergence_of_nearly_equal_distributions(gpu, K, T):
    """A student 1e-2 away from a teacher all of whose classes are known: the divergence, 5e-5, is what is left of
    terms of 1e-2.  With the normaliser given every exponential is a 64-bit one: exp is off by 2e-13 (its series'
    first dropped term), log by 5e-13, and they meet weights that sum to 1; the result is rounded once."""
    N = 48
    r = np.random.default_rng(K)
    t = r.normal(0, 1.5, (N, K)).astype(F)
    x = (t + r.normal(0, 1e-2, (N, K))).astype(F)
    ids = np.tile(r.permutation(K).astype(np.int32), (N, 1))
    tea = np.take_along_axis(t, ids.astype(np.int64), 1)
    # a normaliser just below the true one: nothing is left for a class that the student has no mass for
    lse = np.nextafter((np.log(np.exp(t.astype(np.float64) / T).sum(1))).astype(F), F(-100)) - F(1e-6)
    token = ref.distill(x, tea, ids, lse, None, T)[1]
    assert np.all(np.abs(token) < 1e-2 * T * T)
    tok = dev_empty(N)
    gpu.distill_topk(kept(dev_empty(1)), dptr(tok), None, kept(scratch(N, K)), kept(columns(x, K)), kept(to_dev(tea.reshape(-1))),
                     kept(to_dev(ids.reshape(-1))), kept(to_dev(lse)), None, K, K, N, K, K, K, T)
    same(to_host(tok), token, 2e-12 * T * T + U * np.abs(token), "token loss")
