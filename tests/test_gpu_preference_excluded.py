"""The paired log-ratio loss where a scored token has probability 0 (its logit is -inf): the
sequence's reward is -inf, h infinite, and the loss its limit.  A term that the smoothing leaves out
(smoothing 0) is absent, not 0 * inf.  Tolerances as in test_gpu_token_losses.py."""
import ctypes as C

import numpy as np
import pytest

import token_loss_reference as ref
from test_gpu_token_losses import D, U, columns, grad_buffer, kept, same, scratch, take
from util import dev_empty, dptr, to_dev, to_host

pytestmark = pytest.mark.gpu
F = np.float32
LENGTHS = [3, 2]                 # of every pair
BETA = float(F(0.5))


def limits(h, kind, sm):
    """Loss and slope of h; terms with a factor of 0 left out."""
    with np.errstate(all="ignore"):
        if kind == 0:
            each = (1 - sm) * np.logaddexp(0.0, -h) + (sm * np.logaddexp(0.0, h) if sm else 0.0)
            slope = -(1 - sm) / (1 + np.exp(h)) + (sm / (1 + np.exp(-h)) if sm else 0.0)
        elif kind == 1:
            each = np.where(np.isnan(h), h, np.maximum(0.0, 1.0 - h))
            slope = np.where(np.isnan(h), h, np.where(h < 1.0, -1.0, 0.0))
        else:
            each, slope = ((h - 0.5) / BETA) ** 2, 2.0 * (h - 0.5) / BETA ** 2
    return each, slope


def excluded(K, pairs, which):
    """Sequences of small rewards; `which`: {pair: (chosen excluded, rejected excluded)}."""
    N = sum(LENGTHS) * pairs
    r = np.random.default_rng(K + pairs)
    x = r.normal(0, 1, (N, K)).astype(F)
    labels = r.integers(0, K, N).astype(np.int32)
    begin = np.concatenate([[0], np.cumsum(LENGTHS * pairs)]).astype(np.int32)
    for p, sides in which.items():
        for side, off in enumerate(sides):
            if off:
                n = begin[2 * p + side] + 1
                x[n, labels[n]] = F(-np.inf)
    lp = ref.logprobs(x, labels)[0]
    rlp = (np.where(np.isfinite(lp), lp, -2.0) + r.normal(0, 0.1, N)).astype(F)
    return x, labels, begin, lp, rlp


def call(gpu, x, labels, begin, rlp, pairs, K, kind, sm, average):
    N = len(x)
    out, rew, d, sc = dev_empty(1), dev_empty(2 * pairs), grad_buffer(N, K), scratch(N)
    gpu.preference_loss(dptr(out), dptr(rew), kept(dev_empty(N)), kept(dev_empty(2 * N)), dptr(d), dptr(sc), kept(columns(x, K)),
                        kept(to_dev(labels)), kept(to_dev(rlp)), (C.c_int * len(begin))(*begin.tolist()), pairs, K, K, K, kind,
                        BETA, sm, average, 1.0)
    return to_host(out)[0], to_host(rew), take(d, N, K, K)


# one workgroup for all of it; many pairs; long columns; chunks
@pytest.mark.parametrize("K,pairs", [(7, 4), (700, 4), (13, 80), (5003, 4), (140001, 3)])
@pytest.mark.parametrize("kind,sm,average", [(0, 0.0, 0), (0, 0.0, 1), (0, 0.1, 0), (1, 0.0, 0), (2, 0.0, 0)])
@pytest.mark.parametrize("side", ["rejected", "chosen", "both"])
def test_a_label_of_probability_zero(gpu, K, pairs, kind, sm, average, side):
    print(f"preference excluded K {K} pairs {pairs} kind {kind} {side}", flush=True)
    which = {1: (side != "rejected", side != "chosen")}
    x, labels, begin, lp, rlp = excluded(K, pairs, which)
    loss, rew, got = call(gpu, x, labels, begin, rlp, pairs, K, kind, sm, average)
    smf = float(F(sm))
    R = np.zeros(2 * pairs)
    share = np.ones(2 * pairs)
    for s in range(2 * pairs):
        on = slice(begin[s], begin[s + 1])
        share[s] = 1.0 / (begin[s + 1] - begin[s]) if average else 1.0
        R[s] = BETA * share[s] * np.sum(lp[on] - rlp[on].astype(np.float64))
    err = BETA * max(LENGTHS) * D(K) * U
    same(rew, R, err + 2 * U * np.abs(np.where(np.isfinite(R), R, 0)), "rewards")
    with np.errstate(invalid="ignore"):
        h = R[0::2] - R[1::2]
    each, slope = limits(h, kind, smf)
    want = np.sum(each)
    assert (each[1] == 0.0) == (side == "rejected" and (kind == 1 or kind == 0 and not sm))
    steep = np.max(np.abs(slope[np.isfinite(slope)])) + 1.0
    fine = np.sum(each[np.isfinite(each)])
    same(loss, want, pairs * (steep * 2 * err + 4 * U * (1 + fine)), "loss")
    up = np.repeat(np.stack([slope, -slope], 1).reshape(-1) * share * BETA, LENGTHS * pairs)
    curve = {0: 1.0, 1: 0.0, 2: 2.0 / BETA ** 2}[kind]
    # an infinite slope (squared form) leaves its own pair's gradient infinite or NaN, a NaN one NaN
    odd = ~np.isfinite(up)
    grad = ref.logprobs_bwd(x, labels, np.where(odd, 0.0, up))
    tol = np.abs(np.where(odd, 0.0, up)) * (D(K) + 8) * U + BETA * curve * 2 * err
    same(got[~odd], grad[~odd], tol[~odd][:, None], "gradient")
    assert odd.sum() == (sum(LENGTHS) if side == "both" or kind == 2 else 0)
    assert not np.isfinite(got[odd]).any() if kind != 1 else True


def test_values_do_not_depend_on_the_gradient_being_asked_for(gpu):
    """1024 losses whose 64-bit sum depends on its order: 2.25 and two of 2^-24 reach a tie of fp32, two of
    2^-52 decide it if they meet before they meet the rest.  One class, so log p is 0 and h = ref_r - ref_c."""
    pairs, K = 1024, 1
    off = np.zeros(pairs)
    off[0], off[1], off[2], off[512], off[768] = 1.5, 2.0 ** -12, 2.0 ** -12, 2.0 ** -26, 2.0 ** -26
    rlp = np.stack([np.full(pairs, -0.5), off], 1).reshape(-1).astype(F)
    N = 2 * pairs
    begin = (C.c_int * (N + 1))(*range(N + 1))
    x, labels, sc, stats = to_dev(np.zeros(N, F)), to_dev(np.zeros(N, np.int32)), scratch(N), dev_empty(2 * N)
    rew, lps, d, dr = dev_empty(N), dev_empty(N), dev_empty(N), to_dev(rlp)
    losses = []
    for g in (dptr(d), None):
        out = dev_empty(1)
        gpu.preference_loss(dptr(out), dptr(rew), dptr(lps), dptr(stats), g, dptr(sc), dptr(x), dptr(labels), dptr(dr), begin,
                            pairs, K, K, K, 2, 1.0, 0.0, 0, 1.0)
        losses.append(to_host(out)[0])
    assert np.array_equal(to_host(rew)[0::2], np.full(pairs, 0.5, F))
    assert losses[0] == losses[1]
