"""The losses on logits in float64 numpy: values and gradients from their definitions, column by
column, with the rules for tokens that are not scored.  x is (N, K): one token per row here."""
import numpy as np

LOWEST = np.finfo(np.float32).min


def scored(x, labels):
    K = x.shape[1]
    with np.errstate(invalid="ignore"):
        blank = np.all(x == -np.inf, axis=1)
    return (labels >= 0) & (labels < K) & ~blank


def softmax_parts(x):
    """log softmax and softmax of one column."""
    with np.errstate(all="ignore"):
        m = np.fmax.reduce(x, initial=-np.inf)      # of the numbers: a NaN shows in the sum
        t = x - m
        e = np.exp(t)
        logs = np.log(np.sum(e))
        return t - logs, e / np.sum(e), m, np.sum(e)


def entropy(lq, p):
    with np.errstate(all="ignore"):
        return -np.sum(np.where(p == 0, 0.0, p * lq))


def logprobs(x, labels):
    N = len(x)
    live = scored(x, labels)
    lp, h, m, s = (np.zeros(N) for _ in range(4))
    for n in np.flatnonzero(live):
        lq, p, m[n], s[n] = softmax_parts(x[n].astype(np.float64))
        lp[n], h[n] = lq[labels[n]], entropy(lq, p)
    return lp, h, m, s


def logprobs_bwd(x, labels, up):
    d = np.zeros(x.shape)
    for n in np.flatnonzero(scored(x, labels) & (up != 0)):
        _, p, _, _ = softmax_parts(x[n].astype(np.float64))
        d[n] = -up[n] * p
        d[n, labels[n]] += up[n]
    return d


def policy(x, labels, old, ref, adv, w, lo, hi, beta, ent):
    """sums (4), logp, dlogits, and the entropies' share of the gradient's scale (for tolerances)."""
    N, K = x.shape
    w = np.ones(N) if w is None else w.astype(np.float64)
    sums, lp, d = np.zeros(4), np.zeros(N), np.zeros((N, K))
    up = np.zeros(N)
    with np.errstate(all="ignore"):
        for n in np.flatnonzero(scored(x, labels) & (w != 0)):
            lq, p, _, _ = softmax_parts(x[n].astype(np.float64))
            lp[n] = lq[labels[n]]
            r = np.exp(lp[n] - old[n])
            f, c = r * adv[n], min(max(r, 1.0 - lo), 1.0 + hi) * adv[n]
            cut = f > c
            g, kl, h = (0.0 if cut else -f), 0.0, 0.0
            if ref is not None:
                u = ref[n] - lp[n]
                kl = np.expm1(u) - u
                if beta:
                    g -= beta * np.expm1(u)
            loss = -(c if cut else f) + (beta * kl if beta else 0.0)
            if ent:
                h = entropy(lq, p)
                loss -= ent * h
                d[n] = ent * w[n] * np.where(p == 0, 0.0, p * (lq + h))
            sums += w[n] * np.array([loss, kl, float(cut), h])
            up[n] = g * w[n]
            d[n] -= up[n] * p
            d[n, labels[n]] += up[n]
    return sums, lp, d, up


def preference(x, labels, ref, begin, kind, beta, sm, average, scale):
    lp, _, _, _ = logprobs(x, labels)
    live = scored(x, labels)
    P = (len(begin) - 1) // 2
    R, share = np.zeros(2 * P), np.ones(2 * P)
    for q in range(2 * P):
        on = np.zeros(len(x), bool)
        on[begin[q]:begin[q + 1]] = True
        on &= live
        gain = np.sum(lp[on] - (0.0 if ref is None else ref[on].astype(np.float64)))
        if average:
            share[q] = 1.0 / on.sum() if on.any() else 0.0
        R[q] = beta * gain * share[q]
    h = R[0::2] - R[1::2]
    if kind == 0:
        sp = lambda v: np.logaddexp(0.0, v)
        sig = lambda v: 0.5 * (1.0 + np.tanh(0.5 * v))
        each, slope = (1 - sm) * sp(-h) + sm * sp(h), -(1 - sm) * sig(-h) + sm * sig(h)
    elif kind == 1:
        each, slope = np.maximum(0.0, 1.0 - h), np.where(h < 1.0, -1.0, 0.0)
    else:
        each, slope = ((h - 0.5) / beta) ** 2, 2.0 * (h - 0.5) / beta ** 2
    up = np.zeros(len(x))
    for p in range(P):
        for k, sign in ((0, 1.0), (1, -1.0)):
            q = 2 * p + k
            up[begin[q]:begin[q + 1]] = sign * slope[p] * share[q] * beta * scale
    up = np.where(live, up, 0.0)
    return scale * each.sum(), R, lp, logprobs_bwd(x, labels, up), up


def distill(x, teacher, ids, lse, w, T):
    """Loss, per-token loss, gradient.  teacher, ids: (N, top)."""
    N, K = x.shape
    w = np.ones(N) if w is None else w.astype(np.float64)
    total, token, d = 0.0, np.zeros(N), np.zeros((N, K))
    with np.errstate(all="ignore"):
        for n in range(N):
            if w[n] == 0 or np.all(x[n] == -np.inf):
                continue
            entries = {}
            for j, i in enumerate(ids[n]):
                if 0 <= i < K and i not in entries:
                    entries[int(i)] = float(teacher[n, j])
            if not entries:
                continue
            at = np.array(list(entries))
            u = np.array([entries[i] for i in at]) / T
            if lse is None:
                if np.all(u == -np.inf):
                    continue
                u = u - np.max(u)
                lq = u - np.log(np.sum(np.exp(u)))
            else:
                lq = u - float(lse[n])
            q = np.exp(lq)
            lx, p, _, _ = softmax_parts(x[n].astype(np.float64) / T)
            each = np.sum(np.where(q == 0, 0.0, q * (lq - lx[at])))
            Q, g = q.sum(), np.zeros(K)
            if lse is not None:
                rest = max(0.0, 1.0 - Q)
                others = p.copy()
                others[at] = 0.0
                left = others.sum()
                if rest != 0:
                    each += rest * (np.log(rest) - np.log(left))
                    if left > 0:
                        g -= others * (rest / left)
                    else:
                        g -= others
                Q += rest
            g += p * Q
            g[at] -= q
            token[n] = T * T * each
            total += w[n] * token[n]
            d[n] = T * w[n] * g
    return total, token, d
