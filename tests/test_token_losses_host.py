"""Losses on logits, without a GPU: what the entry points refuse, the size of the scratch, and the
float64 restatement the device results are held to against differences of its own values."""
import ctypes as C

import numpy as np
import pytest

import token_loss_reference as ref

INT = C.c_int


@pytest.fixture(scope="module")
def lib():
    from juzhen_amd import capi
    return capi.load()


P = C.c_void_p(1 << 20)      # never looked at: every call here is refused
Q = C.c_void_p(1 << 21)


def test_scratch_size(lib):
    assert lib.jzhip_token_scratch_floats(1, 0) == 8 + (1 << 20)
    assert lib.jzhip_token_scratch_floats(1000, 64) == 72 * 1000 + (1 << 20)
    assert lib.jzhip_token_scratch_floats(1 << 30, 512) == 520 * (1 << 30) + (1 << 20)
    assert lib.jzhip_token_scratch_floats(0, 0) == 0 and lib.jzhip_token_scratch_floats(5, -1) == 0


def test_logprobs_refuses(lib):
    good = [P, None, None, P, P, P, 8, 4, 8]
    for at, bad in ((3, None), (4, None), (5, None), (6, 0), (6, -1), (6, (1 << 28) + 1), (7, 0), (8, 7), (0, None),
                    (3, C.c_void_p((1 << 20) + 4))):
        a = list(good)
        a[at] = bad
        if at == 6 and bad > 0:
            a[8] = bad
        assert lib.jzhip_token_logprobs(*a) == -1, (at, bad)
    good = [P, P, Q, P, P, 8, 4, 8, 8]
    for at, bad in ((0, None), (1, None), (2, None), (3, None), (4, None), (5, 0), (6, 0), (7, 7), (8, 7)):
        a = list(good)
        a[at] = bad
        assert lib.jzhip_token_logprobs_bwd(*a) == -1, (at, bad)
    assert lib.jzhip_token_logprobs_bwd(Q, P, Q, P, P, 8, 4, 8, 9) == -1      # in place needs one leading dimension


def test_policy_refuses(lib):
    good = [P, P, Q, P, P, P, P, P, P, P, 8, 4, 8, 8, 0.2, 0.2, 0.1, 0.0]
    nan = float("nan")
    for at, bad in ((0, None), (3, None), (4, None), (5, None), (6, None), (8, None), (10, 0), (11, 0), (12, 7), (13, 7),
                    (14, -0.1), (14, 1.5), (14, nan), (15, -0.1), (15, nan), (16, -1.0), (16, nan), (17, -1.0), (17, nan),
                    (7, None), (3, C.c_void_p((1 << 20) + 8))):
        a = list(good)
        a[at] = bad
        assert lib.jzhip_policy_loss(*a) == -1, (at, bad)


def test_preference_refuses(lib):
    begin = (INT * 5)(0, 3, 5, 5, 9)
    good = [P, P, P, P, Q, P, P, P, None, begin, 2, 8, 8, 8, 0, 0.1, 0.0, 0, 1.0]
    nan = float("nan")
    for at, bad in ((0, None), (1, None), (2, None), (3, None), (5, None), (6, None), (7, None), (9, None),
                    (9, (INT * 5)(1, 3, 5, 5, 9)), (9, (INT * 5)(0, 3, 2, 5, 9)), (9, (INT * 5)(0, 0, 0, 0, 0)), (10, 0),
                    (10, (1 << 18) + 1), (11, 0), (12, 7), (13, 7), (14, 3), (14, -1), (15, 0.0), (15, -1.0), (15, nan),
                    (16, 0.5), (16, -0.1), (16, nan), (5, C.c_void_p((1 << 20) + 4))):
        a = list(good)
        a[at] = bad
        assert lib.jzhip_preference_loss(*a) == -1, (at, bad)
    a = list(good)
    a[14], a[16] = 1, 0.1          # smoothing belongs to the sigmoid form
    assert lib.jzhip_preference_loss(*a) == -1


def test_distill_refuses(lib):
    good = [P, None, Q, P, P, P, P, None, None, 8, 4, 2, 8, 8, 4, 1.0]
    nan = float("nan")
    for at, bad in ((0, None), (3, None), (4, None), (5, None), (6, None), (9, 0), (10, 0), (10, 513), (10, 9), (11, 0), (12, 7),
                    (13, 7), (14, 3), (15, 0.0), (15, -1.0), (15, nan), (15, 1e-4), (15, 1e4), (3, C.c_void_p((1 << 20) + 4))):
        a = list(good)
        a[at] = bad
        if at == 10 and bad > 0:
            a[14] = bad
        assert lib.jzhip_distill_topk(*a) == -1, (at, bad)


# more columns, or more logits, than a launch has threads for
@pytest.mark.parametrize("K,N", [(8, (1 << 25) + 1), (8, (1 << 31) - 1), (4097, 1 << 24), (1 << 28, 257)])
def test_sizes_beyond_a_launch(lib, K, N):
    begin = (INT * 3)(0, 1, N)
    assert lib.jzhip_token_logprobs(P, None, None, P, P, P, K, N, K) == -1
    assert lib.jzhip_token_logprobs_bwd(P, P, Q, P, P, K, N, K, K) == -1
    assert lib.jzhip_policy_loss(P, P, Q, P, P, P, P, P, P, P, K, N, K, K, 0.2, 0.2, 0.1, 0.0) == -1
    assert lib.jzhip_preference_loss(P, P, P, P, Q, P, P, P, None, begin, 1, K, K, K, 0, 0.1, 0.0, 0, 1.0) == -1
    assert lib.jzhip_distill_topk(P, None, Q, P, P, P, P, None, None, K, 2, N, K, K, 2, 1.0) == -1


def _slope(f, x, v, h=1e-5):
    return (f(x + h * v) - f(x - h * v)) / (2 * h)


@pytest.mark.parametrize("K,N", [(2, 1), (7, 5), (40, 6)])
def test_restatement_against_differences(K, N):
    """d/dh of every value along a random direction, central differences in float64: the error is
    h^2 f''' + eps/h ~ 1e-10 + 1e-11 at h = 1e-5 for values of order one."""
    r = np.random.default_rng(K * 100 + N)
    x, v = r.normal(0, 2, (N, K)), r.normal(0, 1, (N, K))
    labels = r.integers(-1, K, N)
    labels[0] = K - 1
    up = r.normal(0, 1, N)
    live = ref.scored(x, labels)
    got = _slope(lambda y: np.sum((up * ref.logprobs(y, labels)[0])[live]), x, v)
    assert abs(got - np.sum(v * ref.logprobs_bwd(x, labels, up))) < 1e-7
    lp = ref.logprobs(x, labels)[0]
    old, rlp, adv, w = lp + 0.3 * r.normal(0, 1, N), lp + 0.3 * r.normal(0, 1, N), r.normal(0, 1, N), r.random(N)
    args = (labels, old, rlp, adv, w, 0.2, 0.28, 0.1, 0.05)
    assert abs(_slope(lambda y: ref.policy(y, *args)[0][0], x, v) - np.sum(v * ref.policy(x, *args)[2])) < 1e-7
    begin = [0, (N + 1) // 2, N]
    for kind, sm in ((0, 0.0), (0, 0.1), (1, 0.0), (2, 0.0)):
        for average in (0, 1):
            args = (labels, rlp, begin, kind, 0.7, sm, average, 0.5)
            slope = _slope(lambda y: ref.preference(y, *args)[0], x, v)
            assert abs(slope - np.sum(v * ref.preference(x, *args)[3])) < 1e-6, (kind, sm, average)
    top = min(3, K)
    ids = np.stack([r.permutation(K)[:top] for _ in range(N)])
    ids[0, 0] = -1
    t = r.normal(0, 1, (N, top))
    for T in (1.0, 2.0, 0.5):
        for lse in (None, np.log(np.exp(t / T).sum(1) + 1.0)):
            if lse is not None and K == top:
                continue
            args = (t, ids, lse, w, T)
            slope = _slope(lambda y: ref.distill(y, *args)[0], x, v)
            assert abs(slope - np.sum(v * ref.distill(x, *args)[2])) < 1e-6, (T, lse is None)
