"""What is measured of the operators on token probabilities: what follows the head's logits in scoring, policy-gradient training and
distillation.  ``x = softcap(logits) / temperature`` and ``p = softmax(x)``, a row for each token.

* ``scores``   log probability of the given token, entropy and the ``K`` most likely tokens (ties: the lowest id) with theirs
* ``grads``    the logits' gradient from the gradients of those: of the log probabilities, the entropy, the alternatives
* ``policy``   clipped policy gradient with a KL penalty to a reference and an entropy bonus; the loss and the logits' gradient
* ``distill``  KL from a teacher's ``K`` most likely tokens (renormalised over them, or with all others as one further outcome),
               mixed with cross entropy; the loss and the logits' gradient, or the loss alone

Where ``own`` is true ``run`` makes the framework's calls, elsewhere it computes the same from elementary torch operations.
"""
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CLIP_LOW, CLIP_HIGH, KL, BONUS = 0.2, 0.28, 0.04, 0.003       # of every policy case


def listed():
    return [
        # one sampled token with its alternatives, as a server returns them: latency
        {"name": "scores_token", "op": "scores", "T": 1, "V": 151936, "type": "bf16", "K": 20, "temperature": 0.7, "softcap": 0.0, "ignored": 0.0},
        # rollouts scored under the current weights, the prompts' positions left out: one piece of the head's rows
        {"name": "scores_rollout", "op": "scores", "T": 4096, "V": 151936, "type": "bf16", "K": 0, "temperature": 1.0, "softcap": 0.0, "ignored": 0.25},
        # a teacher's pass: its most likely tokens are kept for distillation
        {"name": "scores_teacher", "op": "scores", "T": 2048, "V": 128256, "type": "bf16", "K": 64, "temperature": 2.0, "softcap": 0.0, "ignored": 0.0},
        # a vocabulary that is not padded, in fp32: rows start off the 16-byte grid
        {"name": "scores_odd", "op": "scores", "T": 257, "V": 50257, "type": "fp32", "K": 5, "temperature": 1.0, "softcap": 0.0, "ignored": 0.1},
        # the backward pass of a loss of one's own on log probabilities and entropies
        {"name": "grads_entropy", "op": "grads", "T": 2048, "V": 128256, "type": "bf16", "K": 0, "temperature": 1.0, "softcap": 0.0, "ignored": 0.25},
        # the same through the alternatives' log probabilities, odd sizes
        {"name": "grads_odd", "op": "grads", "T": 333, "V": 50257, "type": "fp16", "K": 8, "temperature": 0.9, "softcap": 0.0, "ignored": 0.1},
        # a step's tokens of policy-gradient training: one piece of the head's rows
        {"name": "policy_step", "op": "policy", "T": 4096, "V": 151936, "type": "bf16", "temperature": 1.0, "softcap": 0.0, "ignored": 0.25},
        # a few short answers and a small vocabulary: launches
        {"name": "policy_short", "op": "policy", "T": 48, "V": 32000, "type": "bf16", "temperature": 1.0, "softcap": 0.0, "ignored": 0.1},
        # final logits that are capped, a large vocabulary, an odd number of tokens
        {"name": "policy_softcap", "op": "policy", "T": 1001, "V": 256000, "type": "bf16", "temperature": 1.0, "softcap": 30.0, "ignored": 0.25},
        # a student's step: softened probabilities mixed with the labels' cross entropy
        {"name": "distill_step", "op": "distill", "T": 4096, "V": 128256, "type": "bf16", "K": 64, "temperature": 2.0, "softcap": 0.0, "ignored": 0.25,
         "rest": "drop", "ce": 0.3, "grad": True},
        # all other tokens as one outcome; fp32, rows off the 16-byte grid
        {"name": "distill_rest_odd", "op": "distill", "T": 517, "V": 50257, "type": "fp32", "K": 20, "temperature": 1.0, "softcap": 0.0, "ignored": 0.1,
         "rest": "bucket", "ce": 0.0, "grad": True},
        # held-out tokens: the loss alone
        {"name": "distill_heldout", "op": "distill", "T": 2048, "V": 151936, "type": "bf16", "K": 128, "temperature": 1.0, "softcap": 0.0, "ignored": 0.1,
         "rest": "bucket", "ce": 0.0, "grad": False},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["scores", "scores", "grads", "policy", "distill", "distill"])
    T, V = _log(rng, 1, 4096), _log(rng, 1000, 262208)
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if T * V > 4096 * 151936 // (2 if kind == "fp32" else 1):
        T = max(1, 4096 * 151936 // 2 // V)
    c = {"op": op, "T": T, "V": V, "type": kind, "temperature": rng.choice([1.0, 1.0, 0.6, 1.3, 2.0]), "softcap": rng.choice([0.0, 0.0, 30.0]),
         "ignored": rng.choice([0.0, 0.1, 0.5])}
    if op == "scores":
        c["K"] = rng.choice([0, 1, _log(rng, 2, 128)])
    if op == "grads":
        c["K"] = rng.choice([0, 0, _log(rng, 1, 128)])
    if op == "distill":
        c.update(K=_log(rng, 1, 128), rest=rng.choice(["drop", "bucket"]), ce=rng.choice([0.0, 0.3]), grad=rng.random() < 0.7)
    return c


# ------------------------------------------------------------------------------------------- inputs
def _logits(g, T, V):
    """A broad bulk, one token well above it in most rows, as a trained model's logits are."""
    z = 2.2 * torch.randn(T, V, device="cuda", generator=g)
    peak = torch.randint(0, V, (T,), device="cuda", generator=g)
    z.scatter_add_(1, peak[:, None], 3 + 11 * torch.rand(T, 1, device="cuda", generator=g))
    return z, peak


def _logsoftmax(z, case, dtype):
    z = z.to(dtype)
    if case["softcap"]:
        z = case["softcap"] * torch.tanh(z / case["softcap"])
    return torch.log_softmax(z / case["temperature"], -1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, V, op = case["T"], case["V"], case["op"]
    z, peak = _logits(g, T, V)
    logits = z.to(TYPES[case["type"]])
    # the given token is the likeliest one in most rows; some rows (prompts, padding) carry none
    tokens = torch.where(torch.rand(T, device="cuda", generator=g) < 0.7, peak, torch.randint(0, V, (T,), device="cuda", generator=g))
    skip = torch.randperm(T, device="cuda", generator=g)[: int(T * case["ignored"])]
    tokens[skip] = -100
    st = {"case": case, "logits": logits, "targets": tokens}
    on = tokens >= 0
    if op != "scores" and case.get("grad", True):
        st["out"] = torch.empty_like(logits)
    if op == "grads":
        y = _logsoftmax(logits, case, torch.float32)
        p = y.exp()
        st["entropy"] = -(p * y).sum(-1) * on
        at = (logits.float() if not case["softcap"] else case["softcap"] * torch.tanh(logits.float() / case["softcap"])) / case["temperature"]
        st["lse"] = torch.logsumexp(at, -1) * on
        st["dlogprobs"] = torch.randn(T, device="cuda", generator=g) / T
        st["dentropy"] = -0.01 * torch.rand(T, device="cuda", generator=g) / T
        if case["K"]:
            st["top_ids"] = torch.topk(logits.float(), case["K"]).indices.masked_fill(~on[:, None], -1)
            st["dtop"] = torch.randn(T, case["K"], device="cuda", generator=g) / T
    if op == "policy":
        # the policy that sampled was another one by a few steps; ratios a hair off the clip's borders, whose side fp32 can tell
        lp = _logsoftmax(logits, case, torch.float32).gather(1, tokens.clamp(min=0)[:, None])[:, 0]
        step = 0.15 * torch.randn(T, device="cuda", generator=g)
        ratio = step.exp()
        near = ((ratio - (1 - CLIP_LOW)).abs() < 1e-4) | ((ratio - (1 + CLIP_HIGH)).abs() < 1e-4)
        st["old"] = lp - torch.where(near, step + 1e-3, step)
        st["ref"] = lp + 0.3 * torch.randn(T, device="cuda", generator=g)
        st["adv"] = torch.randn(T, device="cuda", generator=g)
    if op == "distill":
        # a teacher that agrees with the student on the whole
        y = _logsoftmax(z + 0.7 * torch.randn(T, V, device="cuda", generator=g), case, torch.float32)
        st["teacher"], st["ids"] = torch.topk(y, case["K"])
    return st


# ---------------------------------------------------------------------------------------- one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st):
    from flextrain_b200 import ops
    case, op = st["case"], st["case"]["op"]
    kw = dict(temperature=case["temperature"], softcap=case["softcap"])
    if op == "scores":
        s = ops.token_logprobs(st["logits"], st["targets"], top_k=case["K"], **kw)
        return (s.logprobs, s.entropy, s.lse) + ((s.top_ids, s.top_logprobs) if case["K"] else ())
    if op == "grads":
        s = ops.TokenLogprobs(None, st["entropy"], st["lse"], st.get("top_ids"), None)
        return ops.token_logprobs_bwd_(st["logits"], st["targets"], s, dlogprobs=st["dlogprobs"], dentropy=st["dentropy"], dtop_logprobs=st.get("dtop"),
                                       out=st["out"], **kw)
    scale = 1.0 / case["T"]
    if op == "policy":
        t = ops.policy_loss_(st["logits"], st["targets"], st["adv"], old_logprobs=st["old"], ref_logprobs=st["ref"], clip_low=CLIP_LOW,
                             clip_high=CLIP_HIGH, kl_beta=KL, entropy_coef=BONUS, grad_scale=scale, out=st["out"], **kw)
        return t.loss, t.logprobs, t.entropy, st["out"]
    kw.update(targets=st["targets"], rest=case["rest"], ce_weight=case["ce"])
    if not case["grad"]:
        return ops.distill_loss(st["logits"], st["ids"], st["teacher"], **kw)
    loss = ops.distill_loss_(st["logits"], st["ids"], st["teacher"], grad_scale=scale, out=st["out"], **kw)
    return loss, st["out"]


def _capped(st):
    """The logits in fp32 behind the cap, and the cap's slope."""
    cap = st["case"]["softcap"]
    z = st["logits"].to(torch.float32)
    if not cap:
        return z, 1.0
    t = torch.tanh(z / cap)
    return cap * t, 1.0 - t * t


def _normal(x):
    """``x - lse`` and ``lse``, by the largest of a row and the sum of what is left."""
    m = x.amax(-1, keepdim=True)
    d = x - m
    s = d.exp().sum(-1, keepdim=True).log()
    return d - s, (m + s)[:, 0]


def _run_plain(st):
    case, op = st["case"], st["case"]["op"]
    tau, tokens = case["temperature"], st["targets"]
    on = tokens >= 0
    at = tokens.clamp(min=0)[:, None]
    u, slope = _capped(st)
    if op == "grads":
        y = u / tau - st["lse"][:, None]
        p = y.exp()
        dl, dh = st["dlogprobs"][:, None], st["dentropy"][:, None]
        given = dl
        if case["K"]:
            given = given + st["dtop"].sum(-1, keepdim=True)
        d = -p * (given + dh * (y + st["entropy"][:, None]))
        d.scatter_add_(1, at, dl)
        if case["K"]:
            d.scatter_add_(1, st["top_ids"].clamp(min=0), st["dtop"])
        return (d * slope / tau * on[:, None]).to(st["logits"].dtype)
    y, lse = _normal(u / tau)
    if op == "distill":
        return _plain_distill(st, u, slope, y, on, at)
    p = y.exp()
    lp = y.gather(1, at)[:, 0]
    ent = -(p * y).sum(-1)
    if op == "scores":
        found = (lp * on, ent * on, lse * on)
        if case["K"]:
            ids = torch.sort(st["logits"].to(torch.float32), dim=-1, descending=True, stable=True).indices[:, : case["K"]]
            found += (torch.where(on[:, None], ids, -1), torch.where(on[:, None], y.gather(1, ids), float("-inf")))
        return found
    r, a = torch.exp(lp - st["old"]), st["adv"]
    inside = r * a <= r.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * a
    e = st["ref"] - lp
    loss = -torch.minimum(r * a, r.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * a) + KL * (e.exp() - e - 1) - BONUS * ent
    dlp = -r * a * inside + KL * (1 - e.exp())
    d = p * (BONUS * (y + ent[:, None]) - dlp[:, None])
    d.scatter_add_(1, at, dlp[:, None])
    d = d * slope * (on.to(torch.float32) / (case["T"] * tau))[:, None]
    return loss * on, lp * on, ent * on, d.to(st["logits"].dtype)


def _plain_distill(st, u, slope, y, on, at):
    case, ids, t = st["case"], st["ids"], st["teacher"]
    tau, ce, T = case["temperature"], case["ce"], case["T"]
    mine = y.gather(1, ids)
    if case["rest"] == "drop":
        lq = _normal(t)[0]
        q = lq.exp()
        kl = (q * (lq - mine)).sum(-1)
    else:
        q = t.exp()
        qr = (1 - q.double().sum(-1)).clamp(min=0).to(torch.float32)
        rest = y.scatter(1, ids, float("-inf"))
        lr = rest.amax(-1) + (rest - rest.amax(-1, keepdim=True)).exp().sum(-1).log()
        kl = (q * (t - mine)).sum(-1) + torch.where(qr > 0, qr * (qr.log() - lr), 0.0)
    loss = (1 - ce) * tau * tau * kl
    if ce:
        hard = _normal(u)[0]
        loss = loss - ce * hard.gather(1, at)[:, 0]
    if not case["grad"]:
        return loss * on
    if case["rest"] == "drop":
        d = y.exp()
    else:
        share = q.sum(-1) + qr                               # one, unless the teacher's sum is above it
        d = y.exp() * share[:, None] - (rest - lr[:, None]).exp() * qr[:, None]
    d.scatter_add_(1, ids, -q)
    d = d * ((1 - ce) * tau)
    if ce:
        h = hard.exp()
        h.scatter_add_(1, at, torch.full_like(h[:, :1], -1.0))
        d = d + ce * h
    d = d * slope * (on.to(torch.float32) / T)[:, None]
    return loss * on, d.to(st["logits"].dtype)


# ------------------------------------------------------------------------------ 64 bits, written apart
def _exact_top(logits, K):
    """Ids of the largest logits, the lowest id first among equals: one key for both, whose order is that of whole numbers."""
    bits = (logits.float() + 0.0).view(torch.int32).to(torch.int64)
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    key = order * (1 << 20) + ((1 << 20) - 1 - torch.arange(logits.shape[1], device=logits.device))
    return (1 << 20) - 1 - (torch.topk(key, K).values & ((1 << 20) - 1))


def exact(case, seed):
    st = prepare(case, seed)
    step = max(1, (1 << 27) // case["V"])                     # rows at a time, a GB of doubles
    pieces = [_exact_rows(st, slice(a, a + step)) for a in range(0, case["T"], step)]
    if not isinstance(pieces[0], tuple):
        return torch.cat(pieces)
    return tuple(torch.cat(p) for p in zip(*pieces))


def _exact_rows(st, rows):
    case, op, tau, cap = st["case"], st["case"]["op"], st["case"]["temperature"], st["case"]["softcap"]
    logits, tokens = st["logits"][rows], st["targets"][rows]
    n = torch.arange(len(tokens), device="cuda")
    z = logits.double()
    u = cap * torch.tanh(z / cap) if cap else z
    du = (1 - (u / cap) ** 2 if cap else torch.ones_like(z)) / tau
    x = u / tau
    off = (tokens == -100)
    t = tokens.masked_fill(off, 0)
    zero = lambda v: v.masked_fill(off if v.dim() == 1 else off[:, None], 0)                                          # noqa: E731
    if op == "grads":
        p = torch.exp(x - st["lse"][rows].double()[:, None])
        logp = x - st["lse"][rows].double()[:, None]
        dl, dh, h = (st[k][rows].double()[:, None] for k in ("dlogprobs", "dentropy", "entropy"))
        dx = -dl * p - dh * p * (logp + h)
        dx[n, t] += dl[:, 0]
        if case["K"]:
            for k in range(case["K"]):                        # one alternative after another
                g = st["dtop"][rows, k].double()
                dx -= g[:, None] * p
                dx[n, st["top_ids"][rows, k].clamp(min=0)] += g
        return zero(dx * du)
    lse = torch.logsumexp(x, 1)
    p = torch.exp(x - lse[:, None])
    lp = x[n, t] - lse
    if op == "scores" or op == "policy":
        h = lse - (p * x).sum(1)
    if op == "scores":
        found = (zero(lp), zero(h), zero(lse))
        if case["K"]:
            ids = _exact_top(logits, case["K"])
            top = torch.gather(x, 1, ids) - lse[:, None]
            found += (ids.masked_fill(off[:, None], -1), top.masked_fill(off[:, None], float("-inf")))
        return found
    scale = 1.0 / case["T"]
    if op == "policy":
        old, ref, a = (st[k][rows].double() for k in ("old", "ref", "adv"))
        r = torch.exp(lp - old)
        held = torch.where(a >= 0, torch.clamp(r, max=1 + CLIP_HIGH), torch.clamp(r, min=1 - CLIP_LOW))
        k3 = torch.exp(ref - lp) - (ref - lp) - 1
        loss = -a * held + KL * k3 - BONUS * h
        slope = torch.where(held == r, -a * r, torch.zeros_like(a)) + KL * (1 - torch.exp(ref - lp))
        onehot = torch.zeros_like(p)
        onehot[n, t] = 1
        dx = slope[:, None] * (onehot - p) + BONUS * p * (x - lse[:, None] + h[:, None])
        return zero(loss), zero(lp), zero(h), zero(dx * du * scale)
    ids, teacher = st["ids"][rows], st["teacher"][rows].double()
    known = torch.zeros_like(p, dtype=torch.bool).scatter_(1, ids, True)
    full = torch.zeros_like(p)
    if case["rest"] == "drop":
        w = torch.softmax(teacher, 1)
        full.scatter_(1, ids, w)
        kl = (w * (torch.log(w) - torch.gather(x, 1, ids) + lse[:, None])).sum(1)
    else:
        w = torch.exp(teacher)
        left = torch.clamp(1 - w.sum(1), min=0)
        others = torch.logsumexp(x.masked_fill(known, float("-inf")), 1)
        # what the teacher leaves goes to the other tokens as the student shares it among them
        full = torch.where(known, full, left[:, None] * torch.exp(x - others[:, None]))
        full.scatter_(1, ids, w)
        kl = (w * (teacher - torch.gather(x, 1, ids) + lse[:, None])).sum(1) + torch.special.xlogy(left, left) - left * (others - lse)
    ce, tau2 = case["ce"], tau * tau
    hard = torch.logsumexp(u, 1) - u[n, t]
    loss = zero((1 - ce) * tau2 * kl + ce * hard)
    if not case["grad"]:
        return loss
    dx = (1 - ce) * tau2 * (p * full.sum(1, keepdim=True) - full)
    if ce:
        soft = torch.softmax(u, 1)
        soft[n, t] -= 1
        dx += ce * tau * soft
    return loss, zero(dx * du * scale)


# --------------------------------------------------------------------------------------------- work
def work(case):
    T, V, op, size = case["T"], case["V"], case["op"], 4 if case["type"] == "fp32" else 2
    live, K = T - int(T * case["ignored"]), case.get("K", 0)
    each = 10 if case["softcap"] else 4                       # operations of an element: maximum, exponential, sums
    if op == "scores":
        return {"bytes": live * V * size + T * (8 + 12 + 12 * K), "flops": (each + 2) * live * V}
    if op == "grads":
        return {"bytes": (live + T) * V * size + T * (8 + 16 + 12 * K), "flops": (each + 4) * live * V}
    if op == "policy":
        return {"bytes": (live + T) * V * size + T * (8 + 12 + 12), "flops": (2 * each + 6) * live * V}
    write = T * V * size if case["grad"] else 0
    return {"bytes": live * V * size + write + T * (8 + 4 + 12 * K), "flops": each * (2 if case["grad"] else 1) * (2 if case["ce"] else 1) * live * V}
