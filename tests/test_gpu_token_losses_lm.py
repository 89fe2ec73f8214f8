"""The losses on logits in the place they are for: the character model trained with each of them.

The gradient of the untied head's bias is the sum of dlogits over the tokens and nothing else, so
it checks value, gradient and wiring against the float64 restatement on the model's own logits;
a run scores with the model, moves it, and scores again, as training with a frozen reference does.
An entry of that bias gradient sums N columns that are each off by (D + 8) u times their upstream
value (see test_gpu_token_losses.py), and N rounded additions: (D + 8 + N) u sum |up|."""
import numpy as np
import pytest

import token_loss_reference as ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
V, D_MODEL, HEADS, FF, LAYERS, S, B = 37, 32, 2, 48, 2, 12, 6
N = S * B


@pytest.fixture(scope="module")
def model(gpu):
    from juzhen_amd.lm import CharLM
    m = CharLM(V, D_MODEL, HEADS, FF, LAYERS, S, B, gelu=True, tied=False, adamw=True, lr=1e-2)
    yield m
    m.close()


def start(model, seed=3):
    model.init_random(seed)
    for k in (2, 3):
        for n in model.names:
            model.set(n, np.zeros(model.shape(n)), which=k)
    model.lib.jzlm_set_iteration(model.h, 1)
    r = np.random.default_rng(seed)
    model.set_batch(r.integers(0, V, (B, S + 1)))
    model.forward()
    x = model.logits().T.copy()                        # (N, V)
    labels = r.integers(0, V, N).astype(np.int32)
    labels.reshape(B, S)[:, :S // 4] = -1              # prompts
    return r, x, labels


def head_bias(model):
    return model.get("head_bias", which=1)[:, 0].astype(np.float64)


def check_bias(model, want, up):
    tol = (40 + N) * U * np.sum(up) + 1e-12
    assert np.max(np.abs(head_bias(model) - want.sum(0))) <= tol
    for n in model.names:                              # and every parameter has one
        g = model.get(n, which=1)
        assert np.isfinite(g).all() and np.any(g != 0), n


def test_scores(model):
    r, x, labels = start(model)
    lp = ref.logprobs(x, labels)[0]
    assert np.max(np.abs(model.logprobs(labels) - lp)) <= 40 * U + 2 * U * np.abs(lp).max()
    assert np.any(model.logprobs() != model.logprobs(labels))      # the targets by default


@pytest.mark.parametrize("kl,ent", [(0.0, 0.0), (0.1, 0.02)])
def test_policy_gradient(model, kl, ent):
    r, x, labels = start(model)
    lp = model.logprobs(labels)
    old = (lp - r.choice([0.0, 0.1, -0.1, 0.5, -0.5], N)).astype(np.float32)
    rlp, adv, w = (lp + 0.1 * r.normal(0, 1, N)).astype(np.float32), r.normal(0, 1, N).astype(np.float32), \
        np.full(N, 1.0 / N, np.float32)
    f = lambda v: float(np.float32(v))
    sums, _, d, up = ref.policy(x, labels, old, rlp if kl else None, adv, w, f(0.2), f(0.2), f(kl), f(ent))
    got = model.backward_policy(old, adv, ref_logp=rlp if kl else None, weight=w, labels=labels, kl_coef=kl, entropy_coef=ent)
    scale = np.abs(up) + w * (1 + kl + 16 * ent)
    assert np.max(np.abs(got - sums)) <= 200 * U * np.sum(scale + w * 4)
    assert model.loss() == got[0]
    check_bias(model, d, 4 * scale)


@pytest.mark.parametrize("kind,smoothing,average", [("sigmoid", 0.1, False), ("hinge", 0.0, False), ("squared", 0.0, True)])
def test_preference_gradient(model, kind, smoothing, average):
    r, x, labels = start(model)
    rlp = (model.logprobs(labels) + 0.2 * r.normal(0, 1, N)).astype(np.float32)
    beta = float(np.float32(0.2))
    loss, R, _, d, up = ref.preference(x, labels, rlp, [b * S for b in range(B + 1)], ("sigmoid", "hinge", "squared").index(kind),
                                       beta, float(np.float32(smoothing)), int(average), float(np.float32(2.0 / B)))
    rewards = model.backward_preference(rlp, labels, kind, 0.2, smoothing, average)
    err = beta * S * 40 * U + 2 * U * np.abs(R).max()
    assert np.max(np.abs(rewards - R)) <= err
    steep = {"sigmoid": 1.0, "hinge": 1.0, "squared": 2 * (np.abs(R).max() * 2 + 0.5) / beta ** 2}[kind]
    assert abs(model.loss() - loss) <= 2 * err * steep + 4 * U * (1 + abs(loss))
    check_bias(model, d, np.abs(up) + beta * {"sigmoid": 1.0, "hinge": 0.0, "squared": 2 / beta ** 2}[kind] * 2 * err / U / 40 / N)


@pytest.mark.parametrize("top,tail,T", [(5, False, 2.0), (8, True, 1.0)])
def test_distillation_gradient(model, top, tail, T):
    r, x, labels = start(model)
    ids = np.stack([r.choice(V, top, replace=False) for _ in range(N)]).astype(np.int32)
    ids[::5, -1] = -1
    t = r.normal(1, 1, (N, top)).astype(np.float32)
    lse = (np.log(np.exp(t / T).sum(1)) + 0.2).astype(np.float32) if tail else None
    w = np.full(N, 1.0 / N, np.float32)
    loss, _, d = ref.distill(x, t, ids, lse, w, T)
    model.backward_distill(t, ids, lse, w, T)
    assert abs(model.loss() - loss) <= 400 * U * T * T * (1 + abs(loss))
    check_bias(model, d, 4 * T * w)


def test_refusals_change_nothing(model):
    from juzhen_amd import capi
    r, x, labels = start(model)
    before = {n: model.get(n) for n in model.names}
    z = np.zeros(N, np.float32)
    for call in (lambda: model.backward_policy(z, z, kl_coef=0.1, update=True),              # KL without a reference
                 lambda: model.backward_policy(z, z, clip_low=1.5, update=True),
                 lambda: model.backward_preference(beta=0.0, update=True),
                 lambda: model.backward_preference(kind="hinge", smoothing=0.1, update=True),
                 lambda: model.backward_distill(np.zeros((N, 4)), np.zeros((N, 4)), temperature=0.0, update=True),
                 lambda: model.backward_distill(np.zeros((N, V + 1)), np.zeros((N, V + 1)), update=True)):
        with pytest.raises(capi.JzhipError):
            call()
    for n in model.names:
        assert np.array_equal(model.get(n), before[n])
    model.backward(update=False)                       # and the model still works
    assert np.isfinite(model.loss())


def test_a_run_of_all_of_them(model):
    """Score with the frozen start, distil, then preferences, then a policy update, each a step of the
    optimiser on fresh logits, then cross-entropy again: the steps move the weights and stay finite."""
    r, x, labels = start(model)
    frozen = model.logprobs(labels)
    assert np.array_equal(frozen, model.logprobs(labels))
    p = np.argsort(-x, axis=1)[:, :6].astype(np.int32)
    t = np.take_along_axis(x, p, 1)
    lse = np.log(np.exp(x.astype(np.float64)).sum(1)).astype(np.float32)
    seen = [model.get("head")]
    for step in range(3):
        for call in (lambda: model.backward_distill(t, p, lse, np.full(N, 1.0 / N), 1.0, update=True),
                     lambda: model.backward_preference(frozen, labels, beta=0.5, update=True),
                     lambda: model.backward_policy(model.logprobs(labels), r.normal(0, 1, N), ref_logp=frozen,
                                                   weight=np.full(N, 1.0 / N), labels=labels, kl_coef=0.05, update=True)):
            model.forward()
            call()
            assert np.isfinite(model.loss())
            seen.append(model.get("head"))
            assert np.isfinite(seen[-1]).all() and np.any(seen[-1] != seen[-2])
    model.step()
    assert np.isfinite(model.loss())
