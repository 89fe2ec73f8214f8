"""Losses on logits at sizes where an index could go wrong: matrices of more than 2^32 elements,
columns that no workgroup's LDS has a bit per logit for, groups of columns that are joined over
several launches.  Only the columns that are scored hold numbers; the float64 restatement sees
those alone.  Tolerances as in test_gpu_token_losses.py."""
import ctypes as C

import numpy as np
import pytest

import token_loss_reference as ref
from util import dev_empty, dptr, to_dev, to_host

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F = np.float32


def D(K):
    return 32 + min(K, 32768) / 256


def sparse(K, N, ld, live, seed):
    """Device logits of which the columns `live` are written, their values, and the labels of all columns."""
    import torch
    r = np.random.default_rng(seed)
    x = torch.empty(N * ld, dtype=torch.float32, device="cuda")
    values = r.normal(0, 2, (len(live), K)).astype(F)
    labels = np.full(N, -1, np.int32)
    for i, n in enumerate(live):
        labels[n] = r.integers(0, K)
        values[i, labels[n]] += F(8.0)
        x[n * ld:n * ld + K] = torch.from_numpy(values[i]).cuda()
    return x, values, labels


def scratch(N, top=0):
    import torch
    from juzhen_amd import capi
    return torch.empty(capi.load().jzhip_token_scratch_floats(N, top), dtype=torch.float32, device="cuda")


# (K, N, ld, scored columns): the last columns lie beyond 2^32 elements in the first three
FAR = [(1000, 4300000, 1000, [0, 1, 2147483, 4294968, 4299999]), (65536, 66000, 65537, [0, 32768, 65540, 65999]),
       (200000, 21600, 200001, [0, 10737, 21475, 21599]), (600000, 70, 600000, [0, 1, 33, 69]),
       (1300000, 70, 1300001, [0, 35, 69]), (150000, 64, 150000, [0, 63]), (5000000, 5, 5000000, [0, 4])]


@pytest.mark.parametrize("K,N,ld,live", FAR)
def test_far_offsets_and_long_columns(gpu, K, N, ld, live):
    import torch
    print(f"far K {K} N {N}", flush=True)
    x, values, labels = sparse(K, N, ld, live, K)
    picked = labels[live]
    dl, sc = to_dev(labels), scratch(N, 4)
    lp, h, m, s = ref.logprobs(values, picked)
    out, ent, stats = dev_empty(N), dev_empty(N), dev_empty(2 * N)
    gpu.token_logprobs(dptr(out), dptr(ent), dptr(stats), dptr(sc), dptr(x), dptr(dl), K, N, ld)
    got = to_host(out)
    assert np.max(np.abs(got[live] - lp)) <= D(K) * U + 2 * U * np.abs(lp).max()
    assert np.max(np.abs(to_host(ent)[live] - h)) <= (16 * D(K) + 2 * np.log(K)) * U
    dead = np.ones(N, bool)
    dead[live] = False
    assert not got[dead].any() and not to_host(stats).reshape(2, N)[:, dead].any()

    d = torch.full((N * ld,), 3.0, dtype=torch.float32, device="cuda")

    def check(want, tol):
        rows = d.view(N, ld)
        for i, n in enumerate(live):
            off = np.abs(to_host(rows[n, :K]).astype(np.float64) - want[i])
            assert off.max() <= tol[i], (n, off.max(), tol[i])
        quiet = torch.tensor(np.flatnonzero(dead)[[0, len(live) // 2, -1]] if dead.any() else [], dtype=torch.long, device="cuda")
        assert not rows[quiet, :K].any()
        assert ld == K or bool((rows[:, K:] == 3.0).all())
        assert int(torch.count_nonzero(d.view(N, ld)[-1, :K])) > 0
        d.fill_(3.0)

    up = np.random.default_rng(1).normal(0, 1, N).astype(F)
    gpu.token_logprobs_bwd(dptr(d), dptr(to_keep(up)), dptr(x), dptr(dl), dptr(stats), K, N, ld, ld)
    check(ref.logprobs_bwd(values, picked, up[live].astype(np.float64)), np.abs(up[live]) * (D(K) + 8) * U)

    old, adv = np.zeros(N, F), np.random.default_rng(2).normal(0, 1, N).astype(F)
    old[live] = (lp - 0.1).astype(F)
    for e in (0.0, 0.02):
        sums, _, want, g = ref.policy(values, picked, old[live], None, adv[live], None, float(F(0.2)), float(F(0.2)), 0.0, float(F(e)))
        four = dev_empty(4)
        gpu.policy_loss(dptr(four), None, dptr(d), dptr(sc), dptr(x), dptr(dl), dptr(to_keep(old)), None, dptr(to_keep(adv)),
                        None, K, N, ld, ld, 0.2, 0.2, 0.0, e)
        check(want, (np.abs(g) * (2 * D(K) + 16) + e * 32 * D(K)) * U)
        assert np.max(np.abs(to_host(four) - sums)) <= 4 * D(K) * U * np.sum(np.abs(g) + 4 + 16 * e)

    top = 4
    r = np.random.default_rng(3)
    ids, t, w = np.full((N, top), -1, np.int32), np.zeros((N, top), F), np.zeros(N, F)
    lse = np.zeros(N, F)
    for n in live:
        ids[n], t[n], w[n] = r.choice(K, top, replace=False), r.normal(2, 1, top), 1.0
        lse[n] = F(np.log(np.exp(t[n].astype(np.float64)).sum()) + 0.2)
    ids[live[-1], 3] = ids[live[-1], 1]            # the same twice
    for tail in (False, True):
        total, token, want = ref.distill(values, t[live], ids[live], lse[live] if tail else None, None, 1.0)
        tok, one = dev_empty(N), dev_empty(1)
        gpu.distill_topk(dptr(one), dptr(tok), dptr(d), dptr(sc), dptr(x), dptr(to_keep(t.reshape(-1))),
                         dptr(to_keep(ids.reshape(-1))), dptr(to_keep(lse)) if tail else None, dptr(to_keep(w)), K, top, N,
                         ld, ld, top, 1.0)
        check(want, np.full(len(live), 4 * (D(K) + 16) * U))
        assert np.max(np.abs(to_host(tok)[live] - token)) <= (4 * np.abs(token).max() + 40) * 2 * U + 2.4 * D(K) * U
        assert abs(to_host(one)[0] - total) <= len(live) * ((4 * np.abs(token).max() + 40) * 4 * U + 2.4 * D(K) * U)

    # one pair: the first scored column against the others
    if N <= 100000:
        begin = (C.c_int * 3)(0, live[0] + 1, N)
        loss, R, _, want, g = ref.preference(values, picked, None, [0, 1, len(live)], 0, float(F(0.1)), 0.0, 1, 1.0)
        one, rew, lps = dev_empty(1), dev_empty(2), dev_empty(N)
        gpu.preference_loss(dptr(one), dptr(rew), dptr(lps), dptr(stats), dptr(d), dptr(sc), dptr(x), dptr(dl), None, begin, 1,
                            K, ld, ld, 0, 0.1, 0.0, 1, 1.0)
        check(want, np.abs(g) * (D(K) + 8) * U + 0.1 * D(K) * U)
        assert np.max(np.abs(to_host(rew) - R)) <= 0.1 * D(K) * U + 2 * U * np.abs(R).max()
        assert abs(to_host(one)[0] - loss) <= D(K) * U + 4 * U * (1 + loss)


def test_gradient_over_several_launches(gpu):
    """2^23 + 300 columns of 1025 logits (34 GB), in place: with 512 threads to a column, more threads than a
    launch may have.  All logits 0, sums as of a column of 1025 ones: -g/1025, and g - g/1025 at the label, off by
    the roundings of the sum's quotient, of the exponential (1 ulp) and of the products (4 U |g|)."""
    import torch
    K, N = 1025, (1 << 23) + 300
    print(f"far gradient K {K} N {N}", flush=True)
    x = torch.zeros(N, K, dtype=torch.float32, device="cuda")
    n = torch.arange(N, device="cuda")
    labels = (n % K).to(torch.int32)
    labels[5::1000] = -1
    g = ((n % 7) + 1).to(torch.float32)
    stats = torch.cat([torch.zeros(N, device="cuda"), torch.full((N,), float(K), device="cuda")])
    torch.cuda.synchronize()
    gpu.token_logprobs_bwd(dptr(x), dptr(g), dptr(x), dptr(labels), dptr(stats), K, N, K, K)
    to_host(g[:1])   # waits
    for at in range(0, N, 1 << 20):
        rows, lab, up = x[at:at + (1 << 20)], labels[at:at + (1 << 20)].long(), g[at:at + (1 << 20)]
        up = torch.where(lab >= 0, up, torch.zeros_like(up))
        rows[torch.arange(len(lab), device="cuda"), lab.clamp(min=0)] -= up
        off = torch.maximum((rows.amax(1) + up / K).abs(), (rows.amin(1) + up / K).abs())
        assert bool((off <= 4 * U * up).all()), at


def to_keep(a):
    import util
    t = to_dev(a)
    util._KEEP.append(t)
    return t
