"""Losses on logits (log-probabilities, policy, preference, distillation) on the device against
the float64 restatement in token_loss_reference.py.

Tolerances, with u = 2^-24 (half a step of fp32): an exponential is off by (|t| + 4) u relative,
a thread adds at most 128 of them one after another and a tree of at most 20 levels joins the rest,
so the sum of a column is off by D u, D(K) = 32 + min(K, 32768) / 256 (sum e|t| / sum e stays under
log K + 1 <= 14).  log p is then off by D u absolute, everything behind it runs in 64 bits and is
rounded once.  An element of the gradient is the upstream value times p or 1 - p, p off by
(D + |t| + 4) u with p |t| <= 0.37: (D + 8) u times the upstream value, absolute."""
import ctypes as C

import numpy as np
import pytest

import token_loss_reference as ref
from util import _KEEP, dev_empty, dptr, to_dev, to_host

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F = np.float32

# one of each regime and its borders, odd ones among them: (K, N, padding of the logits, of the gradient)
SHAPES = [(1, 1, 0, 0), (2, 3, 0, 0), (3, 70, 1, 0), (13, 33, 0, 0), (16, 4, 0, 4), (63, 17, 0, 0), (64, 300, 0, 0),
          (65, 129, 3, 1), (128, 9, 0, 0), (130, 64, 0, 0), (256, 96, 0, 0), (257, 31, 1, 0), (512, 5, 0, 0),
          (1000, 40, 0, 0), (1024, 16, 0, 8), (1025, 7, 0, 0), (4096, 6, 0, 0), (4099, 300, 2, 0), (8200, 5, 0, 0),
          (16385, 4, 0, 3), (32000, 300, 0, 0), (32771, 3, 0, 0), (50001, 2, 0, 0), (65537, 260, 0, 0), (98309, 2, 1, 0),
          (131072, 3, 0, 0), (131077, 2, 0, 0), (200003, 5, 0, 1),
          # enough columns for several workgroups on a CU
          (5001, 530, 0, 0), (12000, 520, 1, 1), (20001, 515, 0, 2), (45000, 513, 0, 0)]


def D(K):
    return 32 + min(K, 32768) / 256


def D_of(x):
    return D(x.shape[1])


def logits(K, N, seed, special=True):
    """Logits (N, K), labels; from N = 16 on the columns that go wrong most easily are among them."""
    r = np.random.default_rng(seed)
    x = r.normal(0, 3, (N, K)).astype(F)
    labels = r.integers(0, K, N).astype(np.int32)
    for n in range(0, N, 2):
        x[n, labels[n]] += F(9.0)
    labels[3::7] = -1
    x[5::11] += F(200.0)                       # far from zero
    x[4::9, :K // 2] = F(-np.inf)              # part of the vocabulary masked, two ways
    x[6::9, K // 3:] = F(ref.LOWEST)
    if special and N >= 16:
        labels[8] = K                          # not a label
        labels[9], x[9] = -5, F(np.nan)        # prompt tokens may hold anything
        labels[10], x[10, :] = -1, F(np.inf)
        x[11] = F(-np.inf)                     # nothing left
        labels[12], x[12] = 0, F(ref.LOWEST)   # the lowest value everywhere: uniform
        labels[13] = 0
        x[13, 0] = F(-np.inf) if K > 1 else x[13, 0]
        labels[14], x[14, K // 2] = K - 1, F(np.nan)
        labels[15], x[15] = 0, F(np.nan)
    return x, labels


def columns(a, ld):
    """(N, K) -> device column-major with leading dimension ld, padding NaN."""
    N, K = a.shape
    full = np.full((N, ld), np.nan, F)
    full[:, :K] = a
    return to_dev(full.reshape(-1))


SENTINEL = F(-7.25)


def kept(t):
    """Pointer to a tensor that nothing else holds: alive until the test ends."""
    _KEEP.append(t)
    return dptr(t)



def grad_buffer(N, ldd):
    return to_dev(np.full(N * ldd, SENTINEL, F))


def take(dev, N, K, ldd):
    got = to_host(dev).reshape(N, ldd)
    assert np.all(got[:, K:] == SENTINEL)
    return got[:, :K].astype(np.float64)


def scratch(N, top=0):
    from juzhen_amd import capi
    return to_dev(np.full(capi.load().jzhip_token_scratch_floats(N, top), np.nan, F))


def same(got, want, tol, what):
    """Equal NaNs and infinities, the rest within tol (absolute, broadcast)."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    odd = ~np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    assert np.array_equal(got[odd & ~np.isnan(want)], want[odd & ~np.isnan(want)]), what
    off = np.where(odd, 0.0, np.abs(np.where(odd, 0.0, got) - np.where(odd, 0.0, want)))
    tol = np.broadcast_to(tol, off.shape)
    worst = np.unravel_index(np.argmax(off - tol), off.shape) if off.size else None
    assert off.size == 0 or off[worst] <= tol[worst], (what, worst, off[worst], tol[worst])


def fin(a):
    return np.where(np.isfinite(a), a, 0.0)


@pytest.mark.parametrize("K,N,pad,padd", SHAPES)
def test_logprobs_and_gradient(gpu, K, N, pad, padd):
    print(f"logprobs K {K} N {N}", flush=True)
    x, labels = logits(K, N, K + N)
    ld, ldd = K + pad, K + padd
    dx, dl = columns(x, ld), to_dev(labels)
    lp, h, m, s = ref.logprobs(x, labels)
    out, ent, stats = dev_empty(N), dev_empty(N), dev_empty(2 * N)
    sc = scratch(N)
    gpu.token_logprobs(dptr(out), dptr(ent), dptr(stats), dptr(sc), dptr(dx), dptr(dl), K, N, ld)
    same(to_host(out), lp, D(K) * U + 2 * U * np.abs(fin(lp)), "logp")
    same(to_host(ent), h, (16 * D(K) + 2 * np.log(K)) * U, "entropy")
    st = to_host(stats).reshape(2, N)
    same(st[0], m, 0.0, "maximum")
    same(st[1], s, D(K) * U * fin(s), "sum")
    # each output alone gives the same bits
    one = dev_empty(N)
    gpu.token_logprobs(dptr(one), None, None, dptr(sc), dptr(dx), dptr(dl), K, N, ld)
    assert np.array_equal(to_host(one), to_host(out), equal_nan=True)
    two = dev_empty(2 * N)
    gpu.token_logprobs(None, None, dptr(two), dptr(sc), dptr(dx), dptr(dl), K, N, ld)
    assert np.array_equal(to_host(two), to_host(stats), equal_nan=True)

    up = np.random.default_rng(N).normal(0, 1, N).astype(F)
    up[2::5] = 0.0
    want = ref.logprobs_bwd(x, labels, up.astype(np.float64))
    d, du = grad_buffer(N, ldd), to_dev(up)
    gpu.token_logprobs_bwd(dptr(d), dptr(du), dptr(dx), dptr(dl), dptr(stats), K, N, ld, ldd)
    got = take(d, N, K, ldd)
    same(got, want, (np.abs(up) * (D(K) + 8) * U)[:, None], "gradient")
    # over the logits themselves
    gpu.token_logprobs_bwd(dptr(dx), dptr(du), dptr(dx), dptr(dl), dptr(stats), K, N, ld, ld)
    inplace = to_host(dx).reshape(N, ld)
    assert np.all(np.isnan(inplace[:, K:]))
    assert np.array_equal(inplace[:, :K].astype(np.float64), got, equal_nan=True)


def policy_inputs(x, labels, seed):
    """Ratios well off the clipping borders, so that both sides of a comparison agree on them."""
    N = len(x)
    r = np.random.default_rng(seed)
    lp, _, _, _ = ref.logprobs(x, labels)
    steps = np.array([0.0, 0.05, -0.05, 0.15, -0.15, 0.4, -0.4, 1.0])
    drift = steps[r.integers(0, len(steps), N)] + r.uniform(-0.01, 0.01, N)
    old = (fin(lp) - drift).astype(F)
    rlp = (fin(lp) + r.normal(0, 0.3, N)).astype(F)
    adv = r.normal(0, 1, N).astype(F)
    w = (r.random(N) / N).astype(F)
    w[1::6] = 0.0
    dead = ~ref.scored(x, labels)
    old[dead], rlp[dead], adv[dead] = np.nan, np.nan, np.nan
    return old, rlp, adv, w


@pytest.mark.parametrize("K,N,pad,padd", SHAPES)
@pytest.mark.parametrize("beta,ent,weighted", [(0.0, 0.0, True), (0.1, 0.0, True), (0.05, 0.02, False)])
def test_policy(gpu, K, N, pad, padd, beta, ent, weighted):
    print(f"policy K {K} N {N} kl {beta} entropy {ent}", flush=True)
    x, labels = logits(K, N, 3 * K + N)
    if N > 13 and K > 1:
        labels[13] = 1                # a label of probability 0 makes the ratio's log infinite: its own test below
    if N > 15:
        x[14], x[15] = x[0], x[2]     # NaN columns too
    old, rlp, adv, w = policy_inputs(x, labels, K)
    lo, hi, b, e = (float(F(v)) for v in (0.2, 0.28, beta, ent))
    live = ref.scored(x, labels) & (w != 0 if weighted else True)
    zero = live & ~np.isfinite(ref.logprobs(x, labels)[0])
    labels[zero] = -1
    sums, lp, want, up = ref.policy(x, labels, old, rlp if beta else None, adv, w if weighted else None, lo, hi, b, e)
    ld, ldd = K + pad, K + padd
    dx, d = columns(x, ld), grad_buffer(N, ldd)
    args = [to_dev(v) for v in (labels, old, rlp, adv, w)]
    out, lps, sc = dev_empty(4), dev_empty(N), scratch(N)
    dl, do, dr, da, dw = (dptr(t) for t in args)
    rest = (dl, do, dr if beta else None, da, dw if weighted else None, K, N, ld)
    tail = (0.2, 0.28, beta, ent)
    gpu.policy_loss(dptr(out), dptr(lps), dptr(d), dptr(sc), dptr(dx), *rest, ldd, *tail)
    same(to_host(lps), lp, D(K) * U + 2 * U * np.abs(lp), "logp")
    got = take(d, N, K, ldd)
    ww = np.where(live, w if weighted else 1.0, 0.0)
    # |r A| shifts with log p by D u relative: part of the upstream value's own error
    tol = (np.abs(up) * (2 * D(K) + 16) + ww * (b * D(K) * 4 + np.abs(adv.astype(np.float64)) * 0 + e * 32 * D(K))) * U
    same(got, want, np.where(live, fin(tol), 0.0)[:, None], "gradient")
    scale = np.sum(fin(np.abs(up) + ww * (1 + b + e * 16) * 4))
    same(to_host(out), sums, 4 * D(K) * U * scale, "sums")
    # values alone; then over the logits
    out2 = dev_empty(4)
    gpu.policy_loss(dptr(out2), None, None, dptr(sc), dptr(dx), *rest, ldd, *tail)
    assert np.array_equal(to_host(out2), to_host(out))
    gpu.policy_loss(dptr(out2), None, dptr(dx), dptr(sc), dptr(dx), *rest, ld, *tail)
    assert np.array_equal(to_host(dx).reshape(N, ld)[:, :K].astype(np.float64), got)


@pytest.mark.parametrize("K", [5, 700, 5000, 40000, 140000])
def test_policy_nan_and_zero_probability(gpu, K):
    """A NaN logit reaches its own column and the sums and nothing else; a label of probability 0 has
    ratio 0 and an infinite KL term; an advantage or weight of an unscored token is not looked at."""
    print(f"policy specials K {K}", flush=True)
    N = 4
    x, labels = logits(K, N, K, special=False)
    labels[:] = [1, 2, 3, -1]
    x[:, :] = np.where(np.isfinite(x), x, 0)
    x[1, 0] = np.nan
    x[2, 3] = -np.inf
    old = np.full(N, -3.0, F)
    adv = np.array([1.0, 1.0, 1.0, np.nan], F)
    ds = [to_dev(v) for v in (labels, old, adv)]
    out, lps, sc = dev_empty(4), dev_empty(N), scratch(N)
    for beta in (0.0, 0.5):
        d = grad_buffer(N, K)
        sums, lp, want, up = ref.policy(x, labels, old, old if beta else None, adv, None, float(F(0.2)), float(F(0.28)), beta, 0.0)
        gpu.policy_loss(dptr(out), dptr(lps), dptr(d), dptr(sc), kept(columns(x, K)), dptr(ds[0]), dptr(ds[1]),
                        dptr(ds[1]) if beta else None, dptr(ds[2]), None, K, N, K, K, 0.2, 0.28, beta, 0.0)
        got = take(d, N, K, K)
        assert np.isnan(to_host(out)[0]) and np.isnan(got[1]).all() and np.isnan(to_host(lps)[1])
        assert to_host(lps)[2] == -np.inf and (got[3] == 0).all()
        same(got[0], want[0], np.abs(up[0]) * (2 * D(K) + 16) * U + beta * D(K) * 4 * U, "clean column")
        if not beta:
            assert (got[2] == 0).all()


PAIRS = [(1, [3, 2]), (2, [1, 0, 0, 5]), (3, [4, 4, 9, 1, 0, 0]), (70, [1 + (7 * i) % 3 for i in range(140)])]


@pytest.mark.parametrize("K", [3, 700, 140000])
def test_policy_infinite_kl(gpu, K):
    """A sampled token that the policy or the reference excludes: ratio 0 or not, KL infinite, gradient of the
    KL term -inf times (1 - p) or its limit kl_coef, and the other tokens as ever."""
    print(f"policy infinite kl K {K}", flush=True)
    x = np.random.default_rng(K).normal(0, 1, (3, K)).astype(F)
    labels = np.array([0, 1, 2], np.int32)
    x[0, 0] = -np.inf
    lp = ref.logprobs(x, labels)[0]
    old, rlp, adv = np.full(3, -2.0, F), np.array([-2.0, -np.inf, lp[2] - 0.3], F), np.array([1.0, 1.0, -1.0], F)
    lo, b = float(F(0.2)), float(F(0.1))
    sums, lps, want, up = ref.policy(x, labels, old, rlp, adv, None, lo, lo, b, 0.0)
    out, one, d, sc = dev_empty(4), dev_empty(3), grad_buffer(3, K), scratch(3)
    gpu.policy_loss(dptr(out), dptr(one), dptr(d), dptr(sc), kept(columns(x, K)), kept(to_dev(labels)), kept(to_dev(old)),
                    kept(to_dev(rlp)), kept(to_dev(adv)), None, K, 3, K, K, 0.2, 0.2, 0.1, 0.0)
    got = take(d, 3, K, K)
    assert to_host(out)[0] == np.inf and to_host(out)[1] == np.inf
    same(to_host(one), lps, D(K) * U + 2 * U * np.abs(fin(lps)), "logp")
    same(got[1:], want[1:], (np.abs(up[1:]) * (2 * D(K) + 16) + b * 4 * D(K))[:, None] * U, "gradient")
    assert up[0] == -np.inf


@pytest.mark.parametrize("K", [1, 13, 256, 1000, 5003, 33001, 140001])
@pytest.mark.parametrize("pairs,lengths", PAIRS)
@pytest.mark.parametrize("kind,sm,average", [(0, 0.0, 0), (0, 0.1, 1), (1, 0.0, 0), (2, 0.0, 1)])
def test_preference(gpu, K, pairs, lengths, kind, sm, average):
    if K > 30000 and pairs > 3:
        pairs, lengths = 3, [7, 2, 3, 9, 4, 1]
    print(f"preference K {K} pairs {pairs} kind {kind}", flush=True)
    begin = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    N, extra = int(begin[-1]), 2
    x, labels = logits(K, N + extra, 5 * K + N, special=False)
    labels[(N + 1) // 2] = -1
    if K > 1:
        x[:, :] = np.where(np.isneginf(x) & (np.arange(K) == labels[:, None]), F(-2), x)   # labels have a probability
    lp = ref.logprobs(x, labels)[0]
    rlp = (lp + np.random.default_rng(N).normal(0, 0.4, N + extra)).astype(F)
    rlp[~ref.scored(x, labels)] = np.nan
    beta, scale = float(F(0.3)), 1.0 / pairs
    loss, R, lp, want, up = ref.preference(x[:N], labels[:N], rlp[:N], begin, kind, beta, float(F(sm)), average,
                                           float(F(scale)))
    h = R[0::2] - R[1::2]
    assert kind != 1 or np.all(np.abs(h - 1.0) > 1e-3)      # the hinge's corner is not among them
    ldd = K + 1
    dx, d = columns(x, K), grad_buffer(N + extra, ldd)
    dl, dr = to_dev(labels), to_dev(rlp)
    out, rew, lps, stats, sc = dev_empty(1), dev_empty(2 * pairs), grad_buffer(N + extra, 1), dev_empty(2 * N), scratch(N)
    cb = (C.c_int * len(begin))(*begin.tolist())
    rest = (dptr(dl), dptr(dr), cb, pairs, K, K)
    tail = (kind, 0.3, sm, average, scale)
    gpu.preference_loss(dptr(out), dptr(rew), dptr(lps), dptr(stats), dptr(d), dptr(sc), dptr(dx), *rest, ldd, *tail)
    got = to_host(d).reshape(N + extra, ldd)
    assert (got[N:] == SENTINEL).all() and (got[:, K:] == SENTINEL).all()
    assert (to_host(lps)[N:] == SENTINEL).all()
    same(to_host(lps)[:N], lp, D(K) * U + 2 * U * np.abs(lp), "logp")
    count = max(lengths)
    err_R = beta * (1 if average else count) * D(K) * U          # every log p off by D u
    same(to_host(rew), R, err_R + 2 * U * np.abs(R), "rewards")
    curve = {0: 1.0, 1: 0.0, 2: 2.0 / beta ** 2}[kind]           # |d slope / d h|
    top_slope = {0: 1.0, 1: 1.0, 2: 2.0 * (np.abs(h).max() + 0.5) / beta ** 2}[kind]
    same(to_host(out), [loss], scale * pairs * (top_slope * 2 * err_R + 4 * U * (1 + abs(loss))) + 2 * U * abs(loss), "loss")
    tol = np.abs(up) * (D(K) + 8) * U + beta * scale * curve * 2 * err_R
    same(got[:N, :K], want, tol[:, None], "gradient")
    out2 = dev_empty(1)
    gpu.preference_loss(dptr(out2), dptr(rew), dptr(lps), dptr(stats), None, dptr(sc), dptr(dx), *rest, ldd, *tail)
    assert np.array_equal(to_host(out2), to_host(out))
    gpu.preference_loss(dptr(out2), dptr(rew), dptr(lps), dptr(stats), dptr(dx), dptr(sc), dptr(dx), *rest, K, *tail)
    inplace = to_host(dx).reshape(N + extra, K)
    assert np.array_equal(inplace[:N], got[:N, :K]) and np.array_equal(inplace[N:], x[N:], equal_nan=True)


def teacher_inputs(K, N, top, seed, T, tail):
    r = np.random.default_rng(seed)
    ids = np.stack([r.choice(K, top, replace=False) for _ in range(N)]).astype(np.int32)
    t = np.sort(r.normal(3, 2, (N, top)), axis=1)[:, ::-1].astype(F)
    w = (r.random(N) + 0.1).astype(F)
    ids[2::5, top // 2:] = -1                # fewer known
    w[1::7] = 0.0
    if N >= 16:
        ids[8] = -1                          # none known
        if top > 2:
            ids[10, 2] = ids[10, 0]          # twice the same
            t[10, 2] = F(np.nan)             # and only the first counts
            t[12, 1:] = F(-np.inf)
            ids[13, 0] = K
        w[9], t[9] = 0.0, F(np.nan)
    lse = None
    if tail:
        known = np.zeros(N)
        for n in range(N):
            seen = {}
            for j, i in enumerate(ids[n]):
                if 0 <= i < K and i not in seen:
                    seen[i] = float(t[n, j])
            v = np.array(list(seen.values()) or [0.0]) / T
            known[n] = np.logaddexp.reduce(v)
        lse = (known - np.log1p(-r.uniform(0.02, 0.3, N))).astype(F)
        if N >= 16:
            lse[14] = F(known[14] - 0.1)     # a normaliser below the entries': nothing is left over
    return t, ids, lse, w


@pytest.mark.parametrize("K,N,pad,padd", SHAPES)
@pytest.mark.parametrize("top,T,tail,weighted", [(1, 1.0, False, False), (5, 2.0, False, True), (40, 1.0, True, True),
                                                 (512, 0.7, True, False)])
def test_distill(gpu, K, N, pad, padd, top, T, tail, weighted):
    top = min(top, max(1, K // 2))
    print(f"distill K {K} N {N} top {top} T {T} tail {tail}", flush=True)
    x, labels = logits(K, N, 7 * K + N)
    x[np.isnan(x).any(1) | np.isposinf(x).any(1)] = 1.0
    t, ids, lse, w = teacher_inputs(K, N, top, K + top, float(F(T)), tail)
    if not weighted:
        t[np.isnan(t)] = 0.0
    # an entry of probability 0 makes the loss infinite: its own test below
    for n in range(N):
        if not np.all(np.isneginf(x[n])):
            good = ids[n][(ids[n] >= 0) & (ids[n] < K)]
            dead = good[x[n, good] < -1e30]
            x[n, dead] = x[n][x[n] > -1e30].min() if (x[n] > -1e30).any() else x[n, dead]
    total, token, want = ref.distill(x, t, ids, lse, w if weighted else None, float(F(T)))
    ok = np.isfinite(token)
    ldt = top + 3
    ft, fi = np.full((N, ldt), np.nan, F), np.zeros((N, ldt), np.int32)
    ft[:, :top], fi[:, :top] = t, ids
    ld, ldd = K + pad, K + padd
    dx, d, sc = columns(x, ld), grad_buffer(N, ldd), scratch(N, top)
    dt, di, dw = to_dev(ft.reshape(-1)), to_dev(fi.reshape(-1)), to_dev(w)
    dz = to_dev(lse) if tail else None
    out, tok = dev_empty(1), dev_empty(N)
    rest = (dptr(dt), dptr(di), dptr(dz) if tail else None, dptr(dw) if weighted else None, K, top, N, ld)
    gpu.distill_topk(dptr(out), dptr(tok), dptr(d), dptr(sc), dptr(dx), *rest, ldd, ldt, T)
    got = take(d, N, K, ldd)
    ww = np.abs(w) if weighted else np.ones(N)
    # Q <= 1.2 by construction; the rest's share r/P_rest carries both sums' errors
    same(got, want, (T * ww * 4 * (D(K) + 16) * U)[:, None], "gradient")
    terms = 4 * np.abs(fin(token)) + 40 * T * T          # sum q |log q - log p|: entries under 40 each
    same(to_host(tok), token, terms * 2 * U + 2.4 * T * T * D(K) * U, "token loss")
    if ok.all():
        same(to_host(out), [total], np.sum(ww * (terms * 4 * U + 2.4 * T * T * D(K) * U)), "loss")
    out2 = dev_empty(1)
    gpu.distill_topk(dptr(out2), None, None, dptr(sc), dptr(dx), *rest, ldd, ldt, T)
    assert np.array_equal(to_host(out2), to_host(out), equal_nan=True)
    gpu.distill_topk(dptr(out2), None, dptr(dx), dptr(sc), dptr(dx), *rest, ld, ldt, T)
    assert np.array_equal(to_host(dx).reshape(N, ld)[:, :K].astype(np.float64), got, equal_nan=True)


@pytest.mark.parametrize("K", [6, 700, 5000, 40000, 140000])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_specials(gpu, K, tail):
    """All mass known, an entry the student excludes, an all-masked teacher, NaN on either side."""
    print(f"distill specials K {K} tail {tail}", flush=True)
    N, top = 6, 4
    r = np.random.default_rng(K)
    x = r.normal(0, 2, (N, K)).astype(F)
    ids = np.tile(np.arange(top, dtype=np.int32), (N, 1))
    t = r.normal(0, 1, (N, top)).astype(F)
    lse = np.logaddexp.reduce(t.astype(np.float64), axis=1).astype(F)       # nothing left but rounding
    lse[0] += F(0.2)
    x[1, 0] = -np.inf                  # excluded by the student: infinite loss, finite gradient
    t[2] = -np.inf                     # no teacher (without the tail: not scored)
    lse[2] = 0.0
    t[3, 1] = np.nan
    x[4, K - 1] = np.nan
    x[5, top:] = -np.inf               # the student has no mass outside the entries
    lse[5] = F(np.logaddexp.reduce(t[5].astype(np.float64)) - 0.01)
    total, token, want = ref.distill(x, t, ids, lse if tail else None, None, 1.0)
    d, out, tok, sc = grad_buffer(N, K), dev_empty(1), dev_empty(N), scratch(N, top)
    gpu.distill_topk(dptr(out), dptr(tok), dptr(d), dptr(sc), kept(columns(x, K)), kept(to_dev(t.reshape(-1))),
                     kept(to_dev(ids.reshape(-1))), kept(to_dev(lse)) if tail else None, None, K, top, N, K, K, top, 1.0)
    got = take(d, N, K, K)
    assert np.isnan(to_host(out)[0])
    same(to_host(tok), token, 40 * 4 * U + 2.4 * D(K) * U, "token loss")
    same(got, want, 4 * (D(K) + 16) * U, "gradient")
    assert np.isnan(got[3]).any() and np.isnan(got[4]).all() and np.isinf(to_host(tok)[1])
    if not tail:
        assert (got[2] == 0).all() and to_host(tok)[2] == 0


def test_gradients_against_differences_of_the_losses(gpu):
    """Central differences of the float64 values along a random direction: h^2 f''' ~ 1e-8 at h = 1e-4,
    the device gradient's own error (D + 8) u |v| ~ 1e-5."""
    K, N, h = 300, 12, 1e-4
    x, labels = logits(K, N, 1, special=False)
    x[np.abs(x) > 1e30] = -4.0
    v = np.random.default_rng(2).normal(0, 1, (N, K))
    dx, dl, sc, d = columns(x, K), to_dev(labels), scratch(N, 4), dev_empty(N * K)

    def slope(f):
        return (f(x.astype(np.float64) + h * v) - f(x.astype(np.float64) - h * v)) / (2 * h)

    def close(want):
        got = np.sum(v * to_host(d).reshape(N, K).astype(np.float64))
        assert abs(got - want) <= 2e-5 * max(1.0, abs(want)) + 2e-5, (got, want)

    old, rlp, adv, w = policy_inputs(x, labels, 3)
    gpu.policy_loss(kept(dev_empty(4)), None, dptr(d), dptr(sc), dptr(dx), dptr(dl), kept(to_dev(old)), kept(to_dev(rlp)),
                    kept(to_dev(adv)), kept(to_dev(w)), K, N, K, K, 0.2, 0.28, 0.1, 0.05)
    close(slope(lambda y: ref.policy(y, labels, old, rlp, adv, w, 0.2, 0.28, 0.1, 0.05)[0][0]))
    begin = [0, 4, 7, 7, 12]
    gpu.preference_loss(kept(dev_empty(1)), kept(dev_empty(4)), kept(dev_empty(N)), kept(dev_empty(2 * N)), dptr(d),
                        dptr(sc), dptr(dx), dptr(dl), kept(to_dev(rlp)), (C.c_int * 5)(*begin), 2, K, K, K, 0, 0.5, 0.1,
                        0, 0.5)
    close(slope(lambda y: ref.preference(y, labels, rlp, begin, 0, 0.5, float(F(0.1)), 0, 0.5)[0]))
    for tail in (False, True):
        t, ids, lse, w2 = teacher_inputs(K, N, 4, 5, 2.0, tail)
        gpu.distill_topk(kept(dev_empty(1)), None, dptr(d), dptr(sc), dptr(dx), kept(to_dev(t.reshape(-1))),
                         kept(to_dev(ids.reshape(-1))), kept(to_dev(lse)) if tail else None, kept(to_dev(w2)), K, 4, N, K,
                         K, 4, 2.0)
        close(slope(lambda y: ref.distill(y, t, ids, lse, w2, 2.0)[0]))


@pytest.mark.parametrize("K,N", [(256, 512), (5003, 40), (140001, 3)])
def test_recorded_and_replayed_on_two_streams(gpu, K, N):
    """Two recorded steps with their own scratch, replayed several times on two streams at once with
    eager calls in between: every replay gives the eager bits."""
    from juzhen_amd import capi
    lib = capi.load()
    print(f"replay K {K} N {N}", flush=True)
    sets = []
    for seed in (1, 2):
        x, labels = logits(K, N, seed, special=False)
        x[np.abs(x) > 1e30] = -4.0
        old, rlp, adv, w = policy_inputs(x, labels, seed)
        t, ids, lse, w2 = teacher_inputs(K, N, 3, seed, 1.0, True)
        labels[N // 2:] = np.maximum(labels[N // 2:], 0)
        g = dict(x=columns(x, K), labels=to_dev(labels), old=to_dev(np.nan_to_num(old)), rlp=to_dev(np.nan_to_num(rlp)),
                 adv=to_dev(np.nan_to_num(adv)), w=to_dev(w), t=to_dev(np.nan_to_num(t).reshape(-1)),
                 ids=to_dev(ids.reshape(-1)), lse=to_dev(lse), sc=scratch(N, 3), out=dev_empty(7), logp=dev_empty(N),
                 stats=dev_empty(2 * N), d=dev_empty(3 * N * K), rew=dev_empty(2))
        sets.append(g)

    def step(g):
        p = {k: v.data_ptr() for k, v in g.items()}
        gpu.policy_loss(p["out"], p["logp"], p["d"], p["sc"], p["x"], p["labels"], p["old"], p["rlp"], p["adv"], p["w"],
                        K, N, K, K, 0.2, 0.28, 0.1, 0.01)
        gpu.preference_loss(p["out"] + 16, p["rew"], p["logp"], p["stats"], p["d"] + 4 * N * K, p["sc"], p["x"],
                            p["labels"], p["rlp"], (C.c_int * 3)(0, N // 3, N), 1, K, K, K, 0, 0.1, 0.0, 1, 1.0)
        gpu.distill_topk(p["out"] + 20, None, p["d"] + 8 * N * K, p["sc"], p["x"], p["t"], p["ids"], p["lse"], p["w"], K,
                         3, N, K, K, 3, 1.0)

    def results(g):
        return [to_host(g[k]).copy() for k in ("out", "logp", "stats", "d", "rew")]

    eager = []
    for g in sets:
        g["out"].zero_()
        step(g)
        gpu.synchronize()
        eager.append(results(g))
    graphs, streams = [], []
    for g in sets:
        h = C.c_void_p()
        assert lib.jzhip_graph_begin() == 0
        try:
            step(g)
        finally:
            assert lib.jzhip_graph_end(C.byref(h)) == 0
        graphs.append(h)
        s = C.c_void_p()
        assert lib.jzhip_stream_create(C.byref(s)) == 0
        streams.append(s)
    import torch
    try:
        for _ in range(4):
            for g in sets:
                for k in ("out", "logp", "stats", "d", "rew"):
                    g[k].fill_(3.0)
                g["out"][6] = 0.0
            torch.cuda.synchronize()
            for h, s in zip(graphs, streams):
                assert lib.jzhip_set_stream(s) == 0
                assert lib.jzhip_graph_launch(h) == 0
            assert lib.jzhip_set_stream(None) == 0
            torch.cuda.synchronize()
            for g, want in zip(sets, eager):
                for a, b in zip(results(g), want):
                    assert np.array_equal(a, b, equal_nan=True)
            step(sets[0])      # eager work between the replays
            torch.cuda.synchronize()
    finally:
        assert lib.jzhip_set_stream(None) == 0
        for h in graphs:
            assert lib.jzhip_graph_destroy(h) == 0
        for s in streams:
            assert lib.jzhip_stream_destroy(s) == 0


@pytest.mark.parametrize("K,N", [(256, 33), (5003, 9), (140001, 2)])
def test_another_stream_sees_its_own_order(gpu, K, N):
    """On a stream of its own, behind work of that stream that makes the inputs."""
    import torch
    from juzhen_amd import capi
    lib = capi.load()
    x, labels = logits(K, N, 4, special=False)
    lp = ref.logprobs(x, labels)[0]
    dx, dl, out, sc = columns(x, K), to_dev(labels), dev_empty(N), scratch(N)
    late = torch.zeros_like(dx)
    torch.cuda.synchronize()
    s = C.c_void_p()
    assert lib.jzhip_stream_create(C.byref(s)) == 0
    try:
        assert lib.jzhip_set_stream(s) == 0
        gpu.copy(dptr(late), dptr(dx), N * K)
        gpu.token_logprobs(dptr(out), None, None, dptr(sc), dptr(late), dptr(dl), K, N, K)
        gpu.synchronize()
    finally:
        lib.jzhip_set_stream(None)
        lib.jzhip_stream_destroy(s)
    same(to_host(out), lp, D(K) * U + 2 * U * np.abs(fin(lp)), "logp")


def test_no_workspace_is_made(gpu):
    from juzhen_amd import capi
    lib = capi.load()
    before = lib.jzhip_workspace_bytes()
    K, N = 140001, 3
    x, labels = logits(K, N, 9, special=False)
    gpu.token_logprobs(kept(dev_empty(N)), None, None, kept(scratch(N)), kept(columns(x, K)), kept(to_dev(labels)), K, N, K)
    gpu.synchronize()
    assert lib.jzhip_workspace_bytes() == before


REGIMES = [(5, 40), (100, 40), (300, 20), (900, 20), (1500, 20), (3000, 9), (6000, 9), (12000, 5), (30000, 5), (40000, 3),
           (40000, 600), (70000, 100), (70000, 3)]


def everything(gpu, g, K, N, ld, top=4):
    """One call of each entry point on a set of buffers; returns what they wrote."""
    p = {k: v if isinstance(v, int) else v.data_ptr() for k, v in g.items()}
    gpu.token_logprobs(p["logp"], p["ent"], p["stats"], p["sc"], p["x"], p["labels"], K, N, ld)
    res = [to_host(g[k]).copy() for k in ("logp", "ent", "stats")]
    d = g["d"]

    def done():
        gpu.synchronize()
        res.append(take(d, N, K, ld) if g["off"] == 0 else to_host(d).reshape(-1)[g["off"]:g["off"] + N * ld].reshape(N, ld)[:, :K].astype(np.float64))
        d.fill_(float(SENTINEL))

    dp_ = p["d"] + 4 * g["off"]
    gpu.token_logprobs_bwd(dp_, p["up"], p["x"], p["labels"], p["stats"], K, N, ld, ld)
    done()
    for e in (0.0, 0.02):
        gpu.policy_loss(p["sums"], None, dp_, p["sc"], p["x"], p["labels"], p["old"], p["old"], p["up"], p["w"], K, N, ld, ld,
                        0.2, 0.2, 0.1, e)
        done()
        res.append(to_host(g["sums"]).copy())
    cb = (C.c_int * 3)(0, N // 3, N)
    gpu.preference_loss(p["sums"], p["rew"], p["logp"], p["stats"], dp_, p["sc"], p["x"], p["labels"], p["old"], cb, 1, K, ld,
                        ld, 0, 0.1, 0.0, 0, 1.0)
    done()
    res += [to_host(g["sums"])[:1].copy(), to_host(g["rew"]).copy()]
    for z in (None, p["lse"]):
        gpu.distill_topk(p["sums"], None, dp_, p["sc"], p["x"], p["t"], p["ids"], z, p["w"], K, top, N, ld, ld, top, 1.5)
        done()
        res.append(to_host(g["sums"])[:1].copy())
    return res


def buffers(K, N, ld, off, labels, seed=1, top=4):
    r = np.random.default_rng(seed)
    flat = np.full(N * ld + off, np.nan, F)
    x = r.normal(0, 2, (N, K)).astype(F)
    flat[off:].reshape(N, ld)[:, :K] = x
    t, ids, lse, w = teacher_inputs(K, N, top, 3, 1.5, True)
    lse[~np.isfinite(lse)] = 5.0
    base = to_dev(flat)
    g = dict(base=base, labels=to_dev(labels), up=to_dev(r.normal(0, 1, N).astype(F)), old=to_dev(np.full(N, -3.0, F)),
             w=to_dev(np.abs(r.normal(0, 1, N)).astype(F)), t=to_dev(np.nan_to_num(t).reshape(-1)), ids=to_dev(ids.reshape(-1)),
             lse=to_dev(lse), sc=scratch(N, top), logp=dev_empty(N), ent=dev_empty(N), stats=dev_empty(2 * N),
             sums=dev_empty(4), rew=dev_empty(2), d=to_dev(np.full(N * ld + off, SENTINEL, F)), off=off)
    g["x"] = base.data_ptr() + 4 * off
    return g, x


@pytest.mark.parametrize("K,N", REGIMES)
def test_any_alignment_and_the_same_bits_again(gpu, K, N):
    """Buffers that begin at any multiple of 4 bytes hold the same numbers to rounding, and a call
    repeated gives the same bits."""
    print(f"alignment K {K} N {N}", flush=True)
    labels = np.random.default_rng(K).integers(-1, K, N).astype(np.int32)
    labels[0], labels[-1] = 0, K - 1
    first = None
    for off in (0, 1, 2, 3):
        for ld in (K, K + 2):
            g, x = buffers(K, N, ld, off, labels)
            got = everything(gpu, g, K, N, ld)
            if (off, ld) in ((0, K), (3, K + 2)):
                for a, b in zip(got, everything(gpu, g, K, N, ld)):
                    assert np.array_equal(a, b, equal_nan=True)
            tail = to_host(g["d"])
            assert (tail == SENTINEL).all()
            if first is None:
                first = got
                want = ref.logprobs(x, labels)[0]
                same(got[0], want, D(K) * U + 2 * U * np.abs(want), "logp")
                continue
            for i, (a, b) in enumerate(zip(got, first)):
                a, b = a.astype(np.float64), b.astype(np.float64)
                scale = np.max(np.abs(b)) + 1.0
                assert np.max(np.abs(a - b)) <= 64 * D(K) * U * scale, (i, off, ld)


@pytest.mark.parametrize("K,N", REGIMES)
def test_nothing_scored(gpu, K, N):
    """All prompt: every loss but the pairs' is 0, every gradient is 0, nothing is NaN."""
    labels = np.full(N, -1, np.int32)
    labels[::2] = K
    g, _ = buffers(K, N, K, 0, labels)
    import torch
    g["base"].fill_(float("nan"))
    g["old"].fill_(float("nan"))
    g["w"].fill_(0.0)
    for r, want in zip(everything(gpu, g, K, N, K), [0] * 9 + [np.log(2.0)] + [0] * 5):
        if want:
            assert np.abs(r - want).max() <= 4 * U
        else:
            assert not r.any()
    assert torch.isnan(g["base"]).all()
