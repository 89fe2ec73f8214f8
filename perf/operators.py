"""Losses of a language model over its logits: what is measured, and their plain forms.

Four operators on a vocab x tokens matrix of logits (column-major with leading dimension `ld`,
that is a row-major (tokens, ld) tensor here, of which the first `vocab` entries of a row count):

  logprobs     log-probability of one label per token, and the entropy of its distribution
  logprobs_bwd gradient of the logits from the gradient of those log-probabilities
  policy       clipped policy-gradient loss with a KL term against a reference model and an
               entropy bonus: value, diagnostics and the gradient of the logits
  preference   paired log-ratio loss of chosen and rejected sequences: value, rewards and gradient
  distill      divergence from a teacher of which the largest logits of each token are known

`run` computes them with elementary torch operations, or, where `own` is set, with the entry
points of libjzhip.  A label outside [0, vocab) is a token that is not scored (prompt, padding).
"""
import torch

own = False

LARGEST = 1 << 28          # elements of the largest logits matrix
LARGEST_VOCAB = 1 << 18
KINDS = ("sigmoid", "hinge", "squared")


def listed():
    return [
        # scoring a batch of the character model's configuration (64 sequences of 256 tokens, 256 symbols)
        {"name": "score a character batch", "op": "logprobs", "vocab": 256, "tokens": 16384, "pad": 0},
        # one token while sampling from a model with a large vocabulary
        {"name": "score one token", "op": "logprobs", "vocab": 262144, "tokens": 1, "pad": 0},
        # gradient of a user's own loss on log-probabilities, odd vocabulary, so no column but the first is aligned
        {"name": "log-probability gradient", "op": "logprobs_bwd", "vocab": 50001, "tokens": 1500, "pad": 0},
        # a handful of tokens of the character model: launches and latency
        {"name": "policy, few tokens", "op": "policy", "vocab": 256, "tokens": 64, "pad": 0, "kl": 0.0, "entropy": 0.0},
        # one update of a policy with a word-piece vocabulary, KL to a reference
        {"name": "policy, 32000 words", "op": "policy", "vocab": 32000, "tokens": 4096, "pad": 0, "kl": 0.05,
         "entropy": 0.0},
        # a large vocabulary with padded columns, KL and entropy bonus
        {"name": "policy, 131072 words", "op": "policy", "vocab": 131072, "tokens": 2048, "pad": 64, "kl": 0.02,
         "entropy": 0.01},
        # two short pairs of character sequences
        {"name": "preference, short pairs", "op": "preference", "vocab": 256, "pairs": 2, "longest": 48, "pad": 0,
         "kind": "sigmoid", "smoothing": 0.0, "average": False},
        # a micro-batch of ragged answers
        {"name": "preference, 8 pairs", "op": "preference", "vocab": 32000, "pairs": 8, "longest": 640, "pad": 0,
         "kind": "sigmoid", "smoothing": 0.1, "average": False},
        # one pair of long answers, odd vocabulary, length-normalised squared loss
        {"name": "preference, one long pair", "op": "preference", "vocab": 50001, "pairs": 1, "longest": 2000,
         "pad": 0, "kind": "squared", "smoothing": 0.0, "average": True},
        # a small student
        {"name": "distill, few words", "op": "distill", "vocab": 1000, "tokens": 512, "top": 8, "pad": 0,
         "tail": False, "temperature": 1.0},
        # the usual form: the teacher's 64 largest, renormalised, temperature 2
        {"name": "distill, 32000 words", "op": "distill", "vocab": 32000, "tokens": 4096, "top": 64, "pad": 0,
         "tail": False, "temperature": 2.0},
        # the teacher's normaliser is known too, so the rest of its mass counts as one class
        {"name": "distill with the rest", "op": "distill", "vocab": 100003, "tokens": 1024, "top": 32, "pad": 1,
         "tail": True, "temperature": 1.0},
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], uniform over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(("logprobs", "logprobs_bwd", "policy", "preference", "distill"))
    vocab = _spread(rng, 16, LARGEST_VOCAB)
    case = {"op": op, "vocab": vocab, "pad": rng.choice((0, 0, 1, 8))}
    most = LARGEST // (vocab + case["pad"]) // 2
    if op == "preference":
        case["pairs"] = _spread(rng, 1, 16)
        case["longest"] = _spread(rng, 1, max(1, min(2000, most // (2 * case["pairs"]))))
        case["kind"] = rng.choice(KINDS)
        case["smoothing"] = rng.choice((0.0, 0.1)) if case["kind"] == "sigmoid" else 0.0
        case["average"] = rng.random() < 0.4
        return case
    case["tokens"] = _spread(rng, 1, min(16384, most))
    if op == "policy":
        case["kl"] = rng.choice((0.0, 0.05))
        case["entropy"] = rng.choice((0.0, 0.0, 0.01))
    if op == "distill":
        case["top"] = _spread(rng, 1, min(256, vocab // 2))
        case["tail"] = rng.random() < 0.5
        case["temperature"] = rng.choice((1.0, 2.0, 0.7))
    return case


# ── inputs ────────────────────────────────────────────────────────────────

BETA = 0.1
CLIP = (0.2, 0.28)


def _lengths(case):
    """Ragged lengths of the 2 * pairs sequences, the longest among them."""
    longest = case["longest"]
    return [longest if i == 1 else 1 + (longest * (37 * i + 11) // 17) % longest for i in range(2 * case["pairs"])]


def _tokens(case):
    return sum(_lengths(case)) if case["op"] == "preference" else case["tokens"]


def _scored(case):
    """How many tokens have a label: the rest is prompt."""
    if case["op"] == "preference":
        return sum(n - n // 4 for n in _lengths(case))
    n = case["tokens"]
    return n if case["op"] == "distill" else n - sum(1 for i in range(n) if _is_prompt(i))


def _is_prompt(i):
    return i % 64 >= 48


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    V, N, op = case["vocab"], _tokens(case), case["op"]
    ld = V + case["pad"]

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    logits = normal(N, ld)
    logits.mul_(2.0)
    labels = torch.randint(0, V, (N,), device=dev, generator=g)
    # most sampled tokens are likely ones
    likely = torch.rand(N, device=dev, generator=g) < 0.75
    rows = torch.arange(N, device=dev)
    logits[rows, labels] += torch.where(likely, 10.0 + normal(N), torch.zeros((), device=dev))
    if op == "preference":
        prompt = torch.cat([torch.arange(n) < n // 4 for n in _lengths(case)]).to(dev)
    else:
        prompt = torch.arange(N, device=dev) % 64 >= 48
    state = {"case": case, "V": V, "N": N, "ld": ld, "logits": logits,
             "labels": torch.where(prompt, -1, labels).to(torch.int32)}
    if op in ("policy", "preference"):
        # the same tokens under the sampling policy and the reference: near the present one
        now = torch.log_softmax(logits[:, :V], 1)[rows, labels]
        state["ref_logp"] = torch.where(prompt, 0.0, now + 0.1 * normal(N))
    if op == "policy":
        state["old_logp"] = torch.where(prompt, 0.0, now + 0.08 * normal(N))
        state["advantage"] = normal((N + 63) // 64).repeat_interleave(64)[:N].contiguous()
        state["weight"] = torch.full((N,), 1.0 / _scored(case), device=dev)
        state["sums"] = torch.empty(4, device=dev)
    if op == "logprobs_bwd":
        state["dlogp"] = normal(N) / N
        # what the forward call left: the largest logit and the sum of exponentials
        big = logits[:, :V].amax(1)
        total = torch.exp(logits[:, :V] - big[:, None]).sum(1)
        state["stats"] = torch.cat([big, total])
    if op == "preference":
        begin = [0]
        for n in _lengths(case):
            begin.append(begin[-1] + n)
        state["begin"] = begin
        state["rewards"] = torch.empty(2 * case["pairs"], device=dev)
    if op == "distill":
        top, T = case["top"], case["temperature"]
        step = V // top
        start = torch.randint(0, V, (N, 1), device=dev, generator=g)
        jump = torch.randint(0, step, (N, top), device=dev, generator=g)
        ids = (start + torch.arange(top, device=dev) * step + jump) % V
        teacher = 10.0 - 2.0 * torch.log1p(torch.arange(top, device=dev)) + 0.5 * normal(N, top)
        logits.scatter_add_(1, ids, 0.7 * teacher + 0.5 * normal(N, top))
        known = torch.logsumexp(teacher.double() / T, 1)
        rest = 0.02 + 0.2 * torch.rand(N, device=dev, generator=g).double()
        if top > 1:      # some tokens come with fewer entries
            ids[7::8, top // 2:] = -1
            known[7::8] = torch.logsumexp(teacher[7::8, :top // 2].double() / T, 1)
        state["ids"] = ids.to(torch.int32).contiguous()
        state["teacher"] = teacher.contiguous()
        state["teacher_lse"] = (known - torch.log1p(-rest)).float() if case["tail"] else None
        state["weight"] = torch.full((N,), 1.0 / N, device=dev)
        state["weight"][3::16] = 0.0     # padding
        state["token_loss"] = torch.empty(N, device=dev)
    if op != "logprobs":
        state["dlogits"] = torch.empty(N, V, device=dev)
    if op in ("logprobs", "policy", "preference"):
        state["logp"] = torch.empty(N, device=dev)
    if op == "logprobs":
        state["entropy"] = torch.empty(N, device=dev)
    if op in ("logprobs", "preference"):
        state["stats"] = torch.empty(2 * N, device=dev)
    state["loss"] = torch.empty(1, device=dev)
    # scratch of the calls: (8 + top) floats a token and 2^20 more
    state["scratch"] = torch.empty((8 + case.get("top", 0)) * N + (1 << 20), device=dev)
    return state


# ── the plain forms ───────────────────────────────────────────────────────

def _softmax(x):
    """Shifted logits, exponentials, their sum (64 bits) and the maximum."""
    m = x.amax(1, keepdim=True)
    t = x - m
    e = torch.exp(t)
    return t, e, e.sum(1, dtype=torch.float64), m[:, 0]


def _label_logp(x, labels, s, m):
    """log softmax at the labels in 64 bits (ratios near a clipping border need it); which are scored."""
    scored = (labels >= 0) & (labels < x.shape[1])
    at = torch.where(scored, labels, 0).long()
    picked = x[torch.arange(x.shape[0], device=x.device), at]
    return torch.where(scored, picked.double() - m.double() - torch.log(s), 0.0), scored, at


def _plain_logprobs(st):
    x = st["logits"][:, :st["V"]]
    t, e, s, m = _softmax(x)
    logp, scored, _ = _label_logp(x, st["labels"], s, m)
    entropy = torch.log(s) - (e * t).sum(1, dtype=torch.float64) / s
    zero = torch.zeros((), device=x.device)
    return {"logp": logp.float(), "entropy": torch.where(scored, entropy.float(), zero)}


def _plain_logprobs_bwd(st):
    x, N = st["logits"][:, :st["V"]], st["N"]
    m, s = st["stats"][:N], st["stats"][N:]
    scored = (st["labels"] >= 0) & (st["labels"] < st["V"])
    up = torch.where(scored, st["dlogp"], 0.0)
    d = torch.exp(x - m[:, None]) * (-up / s)[:, None]
    d[torch.arange(N, device=x.device), torch.where(scored, st["labels"], 0).long()] += up
    return {"dlogits": d}


def _plain_policy(st):
    c = st["case"]
    x = st["logits"][:, :st["V"]]
    t, e, s, m = _softmax(x)
    logp, scored, at = _label_logp(x, st["labels"], s, m)
    w = torch.where(scored, st["weight"], 0.0).double()
    adv = st["advantage"].double()
    ratio = torch.exp(logp - st["old_logp"].double())
    free, held = ratio * adv, torch.clamp(ratio, 1.0 - CLIP[0], 1.0 + CLIP[1]) * adv
    open_ = free <= held
    gap = st["ref_logp"].double() - logp if c["kl"] else torch.zeros_like(logp)
    kl = torch.exp(gap) - gap - 1.0
    up = torch.where(open_, -free, 0.0) + c["kl"] * (1.0 - torch.exp(gap))
    loss = -torch.minimum(free, held) + c["kl"] * kl
    p = e * (1.0 / s).float()[:, None]
    up = (w * up).float()
    d = p * (-up)[:, None]
    entropy = torch.zeros_like(w)
    if c["entropy"]:
        logs = torch.log(s)
        entropy = logs - (e * t).sum(1, dtype=torch.float64) / s
        loss = loss - c["entropy"] * entropy
        d += p * (t + (entropy - logs).float()[:, None]) * (c["entropy"] * w).float()[:, None]
    d[torch.arange(st["N"], device=x.device), at] += up
    sums = torch.stack([(w * loss).sum(), (w * kl).sum(), (w * ~open_).sum(), (w * entropy).sum()])
    return {"sums": sums.float(), "logp": logp.float(), "dlogits": d}


def _plain_preference(st):
    c = st["case"]
    x, N, P = st["logits"][:, :st["V"]], st["N"], c["pairs"]
    t, e, s, m = _softmax(x)
    logp, scored, at = _label_logp(x, st["labels"], s, m)
    begin = torch.tensor(st["begin"], device=x.device)
    seq = torch.searchsorted(begin, torch.arange(N, device=x.device), right=True) - 1
    gain = torch.where(scored, logp - st["ref_logp"].double(), 0.0)
    total = torch.zeros(2 * P, device=x.device, dtype=torch.float64).index_add_(0, seq, gain)
    share = torch.ones_like(total)
    if c["average"]:
        count = torch.zeros_like(total).index_add_(0, seq, scored.double())
        share = torch.where(count > 0, 1.0 / torch.clamp(count, min=1.0), 0.0)
    rewards = BETA * total * share
    h = rewards[0::2] - rewards[1::2]
    if c["kind"] == "sigmoid":
        sm = c["smoothing"]
        each = (1.0 - sm) * _softplus(-h) + sm * _softplus(h)
        slope = -(1.0 - sm) / (1.0 + torch.exp(h)) + sm / (1.0 + torch.exp(-h))
    elif c["kind"] == "hinge":
        each = torch.clamp(1.0 - h, min=0.0)
        slope = torch.where(h < 1.0, -1.0, 0.0)
    else:
        off = h / BETA - 0.5 / BETA
        each, slope = off * off, 2.0 * off / BETA
    slope = torch.stack([slope, -slope], 1).reshape(-1) * share * BETA / P
    up = torch.where(scored, slope[seq], 0.0).float()
    d = e * (up.double() / -s).float()[:, None]
    d[torch.arange(N, device=x.device), at] += up
    return {"loss": (each.sum() / P).float().reshape(1), "rewards": rewards.float(), "logp": logp.float(),
            "dlogits": d}


def _softplus(h):
    return torch.clamp(h, min=0.0) + torch.log1p(torch.exp(-torch.abs(h)))


def _plain_distill(st):
    c = st["case"]
    x, V, T = st["logits"][:, :st["V"]], st["V"], c["temperature"]
    t, e, s, m = _softmax(x if T == 1.0 else x / T)
    ids = st["ids"].long()
    valid = (ids >= 0) & (ids < V)
    at = torch.where(valid, ids, 0)
    u = torch.where(valid, st["teacher"].double() / T, float("-inf"))
    if c["tail"]:
        q = torch.exp(u - st["teacher_lse"].double()[:, None])
        rest = torch.clamp(1.0 - q.sum(1), min=0.0)
    else:
        q = torch.exp(u - u.amax(1, keepdim=True))
        q = q / q.sum(1, keepdim=True)
        rest = torch.zeros_like(s)
    logp = x.gather(1, at).double() / T - m.double()[:, None] - torch.log(s)[:, None]
    each = torch.where(q > 0, q * (torch.log(q) - logp), 0.0).sum(1)
    w = st["weight"].double()
    known = torch.zeros(x.shape, dtype=torch.bool, device=x.device)
    mass = (q.sum(1) + rest) / s
    if c["tail"]:
        known.scatter_(1, torch.where(valid, ids, at[:, :1]), True)   # the first entry always is one
        left = torch.where(known, 0.0, e).sum(1, dtype=torch.float64)
        each = each + torch.where(rest > 0, rest * (torch.log(rest) - torch.log(left / s)), 0.0)
        mass_rest = mass - torch.where(left > 0, rest / left, mass)
        a = torch.where(known, (T * w * mass).float()[:, None], (T * w * mass_rest).float()[:, None])
    else:
        a = (T * w * mass).float()[:, None]
    d = e * a
    d.scatter_add_(1, at, torch.where(valid, -T * w[:, None] * q, 0.0).float())
    each = torch.where(w != 0, T * T * each, 0.0)
    return {"loss": (w * each).sum().float().reshape(1), "token_loss": each.float(), "dlogits": d}


_PLAIN = {"logprobs": _plain_logprobs, "logprobs_bwd": _plain_logprobs_bwd, "policy": _plain_policy,
          "preference": _plain_preference, "distill": _plain_distill}


# ── the framework's calls ─────────────────────────────────────────────────

def _own(st):
    import ctypes

    from juzhen_amd.capi import jz

    c, V, N, ld = st["case"], st["V"], st["N"], st["ld"]
    op = c["op"]

    def p(name):
        t = st.get(name)
        return None if t is None else t.data_ptr()

    if op == "logprobs":
        jz.token_logprobs(p("logp"), p("entropy"), p("stats"), p("scratch"), p("logits"), p("labels"), V, N, ld)
        return {"logp": st["logp"], "entropy": st["entropy"]}
    if op == "logprobs_bwd":
        jz.token_logprobs_bwd(p("dlogits"), p("dlogp"), p("logits"), p("labels"), p("stats"), V, N, ld, V)
        return {"dlogits": st["dlogits"]}
    if op == "policy":
        jz.policy_loss(p("sums"), p("logp"), p("dlogits"), p("scratch"), p("logits"), p("labels"), p("old_logp"),
                       p("ref_logp") if c["kl"] else None, p("advantage"), p("weight"), V, N, ld, V, CLIP[0], CLIP[1],
                       c["kl"], c["entropy"])
        return {"sums": st["sums"], "logp": st["logp"], "dlogits": st["dlogits"]}
    if op == "preference":
        P = c["pairs"]
        begin = (ctypes.c_int * (2 * P + 1))(*st["begin"])
        jz.preference_loss(p("loss"), p("rewards"), p("logp"), p("stats"), p("dlogits"), p("scratch"), p("logits"),
                           p("labels"), p("ref_logp"), begin, P, V, ld, V, KINDS.index(c["kind"]), BETA,
                           c["smoothing"], int(c["average"]), 1.0 / P)
        return {"loss": st["loss"], "rewards": st["rewards"], "logp": st["logp"], "dlogits": st["dlogits"]}
    jz.distill_topk(p("loss"), p("token_loss"), p("dlogits"), p("scratch"), p("logits"), p("teacher"), p("ids"),
                    p("teacher_lse"), p("weight"), V, c["top"], N, ld, V, c["top"], c["temperature"])
    return {"loss": st["loss"], "token_loss": st["token_loss"], "dlogits": st["dlogits"]}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# ── what a pass cannot do without ─────────────────────────────────────────

def work(case):
    V, N, op = case["vocab"], _tokens(case), case["op"]
    live = _scored(case)
    if op == "distill":
        live = N - len(range(3, N, 16))
    read, written = 4 * V * live, 4 * V * N
    # per logit: shift, exponential, sum, scaling; per token: labels, weights, results
    if op == "logprobs":
        return {"bytes": read + 20 * N, "flops": 5 * V * live}
    if op == "distill":
        return {"bytes": read + written + 8 * case["top"] * live + 12 * N, "flops": 5 * V * live}
    return {"bytes": read + written + 24 * N, "flops": (8 if case.get("entropy") else 5) * V * live}


# ── the definitions in 64 bits ────────────────────────────────────────────

def exact(case, seed):
    st = prepare(case, seed)
    V, N, op = st["V"], st["N"], case["op"]
    labels = st["labels"].long()
    keep = (labels >= 0) if op != "distill" else st["weight"] != 0
    rows = keep.nonzero()[:, 0]
    x = st["logits"][rows, :V].double()
    out = torch.zeros(N, V, dtype=torch.float64, device=x.device)

    def whole(values):
        return torch.zeros(N, dtype=torch.float64, device=x.device).index_copy_(0, rows, values)

    if op == "logprobs_bwd":
        up = st["dlogp"].double()[rows]
        x = torch.softmax(x, 1).mul_(-up[:, None])
        x.scatter_add_(1, labels[rows, None], up[:, None])
        return {"dlogits": out.index_copy_(0, rows, x)}
    if op == "distill":
        return _exact_distill(st, case, x, rows, out)
    x.requires_grad_(op != "logprobs")
    logq = torch.log_softmax(x, 1)
    logp = logq.gather(1, labels[rows, None])[:, 0]
    if op == "logprobs":
        return {"logp": whole(logp), "entropy": whole(-(logq.exp() * logq).sum(1))}
    if op == "policy":
        w, adv = st["weight"].double()[rows], st["advantage"].double()[rows]
        ratio = (logp - st["old_logp"].double()[rows]).exp()
        held = ratio.clamp(1.0 - CLIP[0], 1.0 + CLIP[1])
        obj = torch.minimum(ratio * adv, held * adv)
        cut = (ratio * adv > held * adv).double()
        gap = st["ref_logp"].double()[rows] - logp
        kl = torch.expm1(gap) - gap if case["kl"] else torch.zeros_like(gap)
        ent = -(logq.exp() * logq).sum(1) if case["entropy"] else torch.zeros_like(gap)
        loss = (w * (case["kl"] * kl - obj - case["entropy"] * ent)).sum()
        loss.backward()
        sums = torch.stack([loss.detach(), (w * kl).sum().detach(), (w * cut).sum(), (w * ent).sum().detach()])
        return {"sums": sums, "logp": whole(logp.detach()), "dlogits": out.index_copy_(0, rows, x.grad)}
    P, ref = case["pairs"], st["ref_logp"].double()
    every = torch.zeros(N, dtype=torch.float64, device=x.device).index_put((rows,), logp - ref[rows])
    rewards = []
    for a, b in zip(st["begin"], st["begin"][1:]):
        r = every[a:b].sum()
        if case["average"]:
            r = r / max(1, int(keep[a:b].sum()))
        rewards.append(BETA * r)
    rewards = torch.stack(rewards)
    h = rewards[0::2] - rewards[1::2]
    if case["kind"] == "sigmoid":
        like = torch.nn.functional.logsigmoid
        loss = -(1.0 - case["smoothing"]) * like(h) - case["smoothing"] * like(-h)
    elif case["kind"] == "hinge":
        loss = torch.relu(1.0 - h)
    else:
        loss = (h / BETA - 1.0 / (2.0 * BETA)) ** 2
    loss = loss.mean()
    loss.backward()
    return {"loss": loss.detach().reshape(1), "rewards": rewards.detach(), "logp": whole(logp.detach()),
            "dlogits": out.index_copy_(0, rows, x.grad)}


def _exact_distill(st, case, x, rows, out):
    """The divergence over the teacher's classes, its entries and (with the tail) the rest, and its gradient."""
    T, V, N = case["temperature"], st["V"], st["N"]
    w, ids, teacher = st["weight"].double()[rows], st["ids"].long()[rows], st["teacher"].double()[rows]
    gone = ids < 0
    lq = (teacher / T).masked_fill(gone, float("-inf"))
    lq = lq - (st["teacher_lse"].double()[rows, None] if case["tail"] else torch.logsumexp(lq, 1, keepdim=True))
    q = lq.exp()
    at = ids.masked_fill(gone, 0)
    lx = torch.log_softmax(x / T, 1)
    each = torch.where(gone, 0.0, q * (lq.masked_fill(gone, 0.0) - lx.gather(1, at))).sum(1)
    grad = lx.exp()
    if case["tail"]:
        rest = (1.0 - q.sum(1)).clamp(min=0.0)
        hit = torch.zeros(len(rows), V + 1, dtype=torch.bool, device=x.device)     # the last column takes what is no entry
        others = lx.masked_fill(hit.scatter_(1, ids.masked_fill(gone, V), True)[:, :V], float("-inf"))
        left = torch.logsumexp(others, 1)
        each = each + torch.where((rest > 0) & (left > float("-inf")), rest * (torch.log(rest) - left), 0.0)
        grad = grad * (q.sum(1) + rest)[:, None] - (rest[:, None] * (others - left[:, None]).exp()).nan_to_num(0.0)
    grad.scatter_add_(1, at, torch.where(gone, 0.0, -q))
    token = torch.zeros(N, dtype=torch.float64, device=x.device).index_copy_(0, rows, T * T * each)
    return {"loss": (w * T * T * each).sum().reshape(1), "token_loss": token,
            "dlogits": out.index_copy_(0, rows, grad * (T * w)[:, None])}
