"""Distillation with the teacher's normaliser where the student gives the logits outside the entries
next to nothing: their mass is far below what fp32, or even a 64-bit softmax, can hold beside the
entries', its logarithm and the shares of it are ordinary numbers.

The restatement works on logarithms in float64.  Bounds, with u = 2^-24 and t = (x - max)/T: an
exponential is off by (2 |t| + 4) u relative (the difference, its product with log2(e)/T, the
hardware's 2^v, once within a thread's group of sixteen and once for the group), a tree of sixteen adds
4 u, and sum e |t| / sum e <= log K: the sum over the rest is off by C u, C = 2 log K + 8, an element
of its distribution by (2 |t_i| + 4 + C + 8) u relative (8: the coefficients' roundings and the last
products).  Quantities of a column are formed in 64 bits: a token's loss is off by what log P_rest and
log s are, T^2 C u each, and by its own rounding.  Nothing below 2^-126 is kept (floor)."""
import numpy as np
import pytest

import token_loss_reference as ref
from test_gpu_token_losses import SENTINEL, columns, grad_buffer, kept, same, scratch, take
from util import dev_empty, dptr, to_dev, to_host

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F = np.float32
TOP = 4


def lse64(v):
    m = np.max(v)
    return m if not np.isfinite(m) else m + np.log(np.sum(np.exp(v - m)))


def distill64(x, t, ids, lse, w, T):
    """Per-token loss, gradient, and per element what an error of the rest's share and of p scale with."""
    N, K = x.shape
    token, d, near = np.zeros(N), np.zeros((N, K)), np.zeros((N, K))
    for n in range(N):
        v = x[n].astype(np.float64) / T
        lx = v - lse64(v)
        at = ids[n]
        lq = t[n].astype(np.float64) / T - float(lse[n])
        q = np.exp(lq)
        r = max(0.0, 1.0 - q.sum())
        out = np.ones(K, bool)
        out[at] = False
        left = lse64(lx[out])
        token[n] = T * T * (np.sum(q * (lq - lx[at])) + (r * (np.log(r) - left) if r else 0.0))
        share = np.where(out, np.exp(np.where(out, lx - left, 0.0)), 0.0)
        Q = q.sum() + r
        d[n] = T * w[n] * (Q * np.exp(lx) - r * share)
        d[n, at] -= T * w[n] * q
        top_all, top_rest = v.max(), v[out].max()
        far = np.where(out, top_rest - v, top_all - v)         # |t| of the exponential that stands for the element
        far = np.minimum(far, 100.0)                           # (below 2^-126: the floor)
        C = 2 * np.log(K) + 8
        near[n] = T * w[n] * ((Q * np.exp(lx) + r * share) * (2 * far + 12 + C))
        near[n, at] += T * w[n] * q * 4
    return token, d, near


def inputs(K, N, T, seed):
    """Entries `gap` above the rest (column 0: none, 1: below the rest), the last entry always among the rest."""
    r = np.random.default_rng(seed)
    x = r.normal(0, 1.5 * T, (N, K)).astype(F)
    ids = np.stack([np.sort(r.choice(K, TOP, replace=False)) for _ in range(N)]).astype(np.int32)
    r.permuted(ids, axis=1, out=ids)
    for n in range(N):
        gap = (0.0, -110 * T, 60 * T, 120 * T, 600 * T)[n % 5]
        x[n, ids[n, :TOP - 1]] = F(gap) + r.normal(0, T, TOP - 1).astype(F)
    t = (r.normal(0, 1, (N, TOP)) * T).astype(F)
    lse = np.array([lse64(t[n].astype(np.float64) / T) + 0.3 for n in range(N)]).astype(F)
    w = (r.random(N) + 0.5).astype(F)
    return x, t, ids, lse, w


# one of each way a column is cut: lanes of a wave, one wave, workgroups that keep all of it or half, chunks
CUTS = [(6, 40), (40, 7), (100, 9), (200, 9), (400, 9), (900, 9), (1500, 9), (3000, 9), (6001, 9), (12001, 6), (30000, 6),
        (50001, 5), (50001, 70), (70000, 70), (140001, 5)]
LARGE = [(6001, 520), (12000, 515), (20001, 513)]


@pytest.mark.parametrize("K,N,T", [(K, N, T) for T in (1.0, 0.1, 0.05, 1e-3) for K, N in CUTS] +
                         [(K, N, T) for T in (1.0, 1e-3) for K, N in LARGE] + [(1300001, 65, 0.1)])
def test_rest_far_below_the_entries(gpu, K, N, T):
    print(f"rest K {K} N {N} T {T}", flush=True)
    Tf = float(F(T))
    x, t, ids, lse, w = inputs(K, N, Tf, K + int(1 / T))
    some = np.arange(N) if K <= 10 ** 6 else np.array([0, 1, 2, 3, 4, N - 1])
    token, want, near = distill64(x[some], t[some], ids[some], lse[some], w[some].astype(np.float64), Tf)
    assert np.isfinite(token).all()
    dx, d, tok, out, sc = columns(x, K), grad_buffer(N, K + 1), dev_empty(N), dev_empty(1), scratch(N, TOP)
    gpu.distill_topk(dptr(out), dptr(tok), dptr(d), dptr(sc), dptr(dx), kept(to_dev(t.reshape(-1))),
                     kept(to_dev(ids.reshape(-1))), kept(to_dev(lse)), kept(to_dev(w)), K, TOP, N, K, K + 1, TOP, T)
    got = to_host(tok)
    assert np.isfinite(got).all() and np.isfinite(to_host(out)).all()
    same(got[some], token, (2 * (2 * np.log(K) + 8) * Tf * Tf + 2 * np.abs(token)) * U, "token loss")
    same(take(d, N, K, K + 1)[some], want, near * U + 2.0 ** -118 * w[some][:, None], "gradient")
    # in place
    gpu.distill_topk(dptr(out), dptr(tok), dptr(dx), dptr(sc), dptr(dx), kept(to_dev(t.reshape(-1))),
                     kept(to_dev(ids.reshape(-1))), kept(to_dev(lse)), kept(to_dev(w)), K, TOP, N, K, K, TOP, T)
    assert np.array_equal(to_host(tok), got)
    same(to_host(dx).reshape(N, K)[some].astype(np.float64), want, near * U + 2.0 ** -118 * w[some][:, None], "in place")


@pytest.mark.parametrize("K,N", [(9, 4), (700, 4), (5000, 4), (50001, 70), (140001, 4)])
def test_rest_masked_or_alone(gpu, K, N):
    """The rest all -inf or all of the type's lowest value has no mass: infinite loss, gradient 0 there; the
    entries all masked and the rest not: the token counts; all of it the lowest value: uniform."""
    print(f"rest masked K {K}", flush=True)
    x, t, ids, lse, w = inputs(K, N, 1.0, K)
    rest = np.ones((N, K), bool)
    for n in range(N):
        rest[n, ids[n]] = False
        x[n, ids[n]] = F(n)
    x[0, rest[0]] = F(-np.inf)
    x[1, rest[1]] = F(ref.LOWEST)
    x[2, ids[2]] = F(-np.inf)
    x[3] = F(ref.LOWEST)
    d, tok, out, sc = grad_buffer(N, K), dev_empty(N), dev_empty(1), scratch(N, TOP)
    gpu.distill_topk(dptr(out), dptr(tok), dptr(d), dptr(sc), kept(columns(x, K)), kept(to_dev(t.reshape(-1))),
                     kept(to_dev(ids.reshape(-1))), kept(to_dev(lse)), None, K, TOP, N, K, K, TOP, 1.0)
    got, each = take(d, N, K, K), to_host(tok)
    q = np.exp(t.astype(np.float64) - lse[:, None])
    r = 1.0 - q.sum(1)
    for n in (0, 1):
        assert each[n] == np.inf and (got[n][rest[n]] == 0).all()
        p = np.full(TOP, 1.0 / TOP)                            # four equal entries and nothing else
        same(got[n][ids[n]], p - q[n], 16 * U, "entries")
    assert each[2] == np.inf                                   # entries of probability 0
    same(got[2][ids[2]], -q[2], 4 * U, "excluded entries")
    share = np.exp(x[2][rest[2]].astype(np.float64) - lse64(x[2][rest[2]].astype(np.float64)))
    same(got[2][rest[2]], share * (1.0 - r[2]), share * (60 + 4 * np.log(K)) * U, "the rest alone")
    left = (K - TOP) / K
    want = np.sum(q[3] * (np.log(q[3]) + np.log(K))) + r[3] * (np.log(r[3]) - np.log(left))
    same(each[3], want, (2 * (2 * np.log(K) + 8) + 4 * abs(want)) * U, "uniform")
    same(got[3][rest[3]], np.full(K - TOP, 1.0 / K - r[3] / (K - TOP)), (1.0 / K + r[3] / (K - TOP)) * (20 + 2 * np.log(K)) * U, "uniform")
    same(got[3][ids[3]], 1.0 / K - q[3], 32 * U, "uniform")


def test_shared_memory_of_any_size_in_any_order(gpu):
    """A bit per logit: 88, 138 and 75 KB of LDS one after another, and from two threads at once, give what each
    gives alone."""
    import threading
    N, T = 70, 1.0
    calls = {}
    for K in (700001, 1100003, 600001):
        r = np.random.default_rng(K)
        x = np.zeros((N, K), F)
        x[:, :1000] = r.normal(0, 2, (N, 1000))
        ids = np.tile(np.array([1, 5, 999, K - 1], np.int32), (N, 1))
        t = r.normal(0, 1, (N, TOP)).astype(F)
        lse = np.array([lse64(v.astype(np.float64)) + 0.3 for v in t]).astype(F)
        calls[K] = [columns(x, K), to_dev(t.reshape(-1)), to_dev(ids.reshape(-1)), to_dev(lse), scratch(N, TOP), dev_empty(1), dev_empty(N)]
        some = [0, N - 1]
        calls[K].append(distill64(x[some], t[some], ids[some], lse[some], np.ones(N), T)[0])
    import torch
    torch.cuda.synchronize()

    def run(K):
        x, t, ids, lse, sc, out, tok, _ = calls[K]
        gpu.distill_topk(dptr(out), dptr(tok), None, dptr(sc), dptr(x), dptr(t), dptr(ids), dptr(lse), None, K, TOP, N, K, K, TOP, T)

    first = {}
    for K in (700001, 1100003, 600001, 1100003, 700001):
        run(K)
        got = to_host(calls[K][6])
        same(got[[0, N - 1]], calls[K][7], (2 * (2 * np.log(K) + 8) + 2 * np.abs(calls[K][7])) * U, "token loss")
        assert np.array_equal(first.setdefault(K, got), got)
    failed = []

    def guarded(K):
        try:
            run(K)
        except Exception as e:      # reported by the test's own thread
            failed.append(e)

    threads = [threading.Thread(target=guarded, args=(K,)) for K in (700001, 1100003)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    assert not failed
    for K in (700001, 1100003):
        assert np.array_equal(first[K], to_host(calls[K][6]))
