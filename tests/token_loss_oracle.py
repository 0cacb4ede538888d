"""The operators on token probabilities from their definitions in 64 bits: losses as differentiable expressions, their gradients by
autograd, and for each gradient the size of the terms that it is the sum of (``size``), which errors are relative to.

An error of fp32 arithmetic in ``p`` is relative to it: the exponent's argument, up to 60 in base 2, is rounded to 2^-24 of it
(60 ln 2 2^-24 = 2.5e-6), the exponential is good to 2^-22 (2.4e-7), the sum of a row to some 1e-6; 1e-5 is above their sum.  A
soft-cap of 30 adds the tanh's two steps, 30 2^-23 = 3.6e-6 of u and twice that at a temperature of a half: 2e-5.  Its slope 1 - t^2
is off by two steps of one, 2.4e-7 of a term before the slope."""
import torch

from flextrain_b200 import ops

F64 = torch.float64


def u_of(z, cap):
    return torch.where(z == float("-inf"), z, cap * torch.tanh(z / cap)) if cap else z


def on_rows(T, V, targets, mask, ignore=-100, device="cpu"):
    on = torch.ones(T, dtype=torch.bool, device=device)
    if targets is not None:
        on &= (targets != ignore) & (targets >= 0) & (targets < V)
    return on if mask is None else on & (mask > 0)


def plogp(lp):
    """``p log p`` with nothing at ``p = 0``, differentiable."""
    safe = lp.masked_fill(lp == float("-inf"), 0.0)
    return torch.where(lp == float("-inf"), torch.zeros_like(lp), safe.exp() * safe)


def scores(logits, targets, on, tau, cap, K):
    """Differentiable ``(logprobs, entropy, lse, ids, top)`` of the rows that are on, in the order of the rows."""
    z = logits[on].to(F64).requires_grad_()
    x = u_of(z, cap) / tau
    lse = torch.logsumexp(x, -1)
    lp = x - lse[:, None]
    ent = -plogp(lp).sum(-1)
    given = None if targets is None else lp.gather(1, targets[on][:, None])[:, 0]
    ids = top = None
    if K:
        # value down, then index up, of each row by itself
        ids = torch.stack([torch.tensor(sorted(range(r.numel()), key=lambda i, r=r: (-r[i], i))[:K]) if r.numel() < 3000 else
                           torch.sort(r, descending=True, stable=True).indices[:K].cpu() for r in (logits[on].float().cpu() + 0.0)]) \
            if int(on.sum()) else torch.zeros(0, K, dtype=torch.int64)
        ids = ids.to(logits.device)
        top = lp.gather(1, ids)
    return z, lp, given, ent, lse, ids, top


def scatter_rows(on, part, like):
    full = torch.zeros(len(on), *part.shape[1:], dtype=F64, device=like.device)
    full[on] = part.detach()
    return full


def grad_of(total, z, on):
    g, = torch.autograd.grad(total, z)
    return scatter_rows(on, g, z)


def slope_of(logits, cap):
    return 1 - torch.tanh(logits.to(F64) / cap) ** 2 if cap else torch.ones_like(logits, dtype=F64)


def clean(v):
    return torch.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0)


def scores_grad(logits, targets, on, tau, cap, dl, dh, ids, dtop, scale):
    """Gradient by the logits and the size of its terms."""
    z, lp, given, ent, _, _, _ = scores(logits, targets, on, tau, cap, 0)
    total = z.sum() * 0
    V = logits.shape[1]
    size = torch.zeros_like(lp)
    G = torch.zeros(len(lp), dtype=F64, device=z.device)
    if dl is not None:
        total = total + (given * dl[on].to(F64)).sum()
        G += dl[on].abs()
        size.scatter_add_(1, targets[on][:, None], dl[on].abs().to(F64)[:, None])
    if dtop is not None:
        i, g = ids[on], dtop[on].to(F64)
        ok = (i >= 0) & (i < V)
        g = g * ok
        total = total + (lp.gather(1, i * ok) * g).sum()
        G += g.abs().sum(-1)
        size.scatter_add_(1, i * ok, g.abs())
    p = lp.detach().exp()
    if dh is not None:
        total = total + (ent * dh[on].to(F64)).sum()
        G = G[:, None] + dh[on].abs()[:, None] * (clean(lp.detach()).abs() + ent.detach()[:, None])
        size = size + p * G
    else:
        size = size + p * G[:, None]
    return grad_of(total * scale, z, on), scatter_rows(on, size.detach() * (scale / tau), z)


def policy(logits, targets, on, tau, cap, adv, old, kept, lo, hi, beta, bonus, scale):
    z, lp, given, ent, _, _, _ = scores(logits, targets, on, tau, cap, 0)
    a = torch.ones_like(given) if adv is None else adv[on].to(F64)
    if old is None:
        loss, g = -a * given, a.abs()
    else:
        r = torch.exp(given - old[on].to(F64))
        loss = -torch.minimum(r * a, r.clamp(1 - lo, 1 + hi) * a)
        g = (r * a).abs()
    if kept is not None and beta:
        d = kept[on].to(F64) - given
        loss = loss + beta * (d.exp() - d - 1)
        g = g + beta * (d.exp() + 1)
    if bonus:
        loss = loss - bonus * ent
    p = lp.detach().exp()
    size = p * (g[:, None] + bonus * (clean(lp.detach()).abs() + ent.detach()[:, None]))
    size = size.detach().scatter_add(1, targets[on][:, None], g.detach()[:, None])
    d = grad_of(loss.sum() * scale, z, on)
    return [scatter_rows(on, v, z) for v in (loss, given, ent)], d, scatter_rows(on, size * (scale / tau), z)


def distill(logits, ids, teacher, targets, on, rest, ce, tau, cap, scale):
    z, lp, given, ent, _, _, _ = scores(logits, targets, on, tau, cap, 0)
    V = logits.shape[1]
    i, t = ids[on], teacher[on].to(F64)
    ok = (i >= 0) & (i < V)
    t = t.masked_fill(~ok, float("-inf"))
    i = i * ok
    if rest == "drop":
        some = (t > float("-inf")).any(-1, keepdim=True)
        t = torch.where(some, t - torch.where(some, torch.logsumexp(t, -1, keepdim=True), 0.0), t)
    q = t.exp()
    held = lp.gather(1, i)
    # (entries without probability have no part, whatever the student has there)
    kl = torch.where(q > 0, q * (torch.where(q > 0, t, 0.0) - torch.where(q > 0, held, 0.0)), 0.0).sum(-1)
    p = lp.detach().exp()
    size = p * q.sum(-1, keepdim=True)
    size = size.scatter_add(1, i, q)
    if rest == "bucket":
        named = torch.zeros(len(i), V, dtype=torch.int32, device=z.device).scatter_add_(1, i, ok.to(torch.int32)) > 0
        others = lp.masked_fill(named, float("-inf"))
        left = others.detach().amax(-1) > float("-inf")
        qr = torch.where(left, (1 - q.sum(-1)).clamp(min=0), 0.0)
        lr = torch.logsumexp(torch.where(left[:, None], others, 0.0), -1)
        kl = kl + torch.where(qr > 0, qr * (torch.log(qr.clamp(min=1e-300)) - lr), 0.0)
        # 1 - sum q has the error of a sum near one, whatever is left: each q is off by 2^-22 of it (the exponential), so all by 2^-22,
        # and a sum by seven steps of pairs by 7 2^-24 of one: 6.6e-7, which is 0.066 in the terms' 1e-5
        size = size + p * qr[:, None] + torch.where(named, 0.0, (qr[:, None] + 0.066) * torch.exp(others.detach() - lr.detach()[:, None]))
    loss = (1 - ce) * tau * tau * kl
    size = size * (1 - ce) * tau
    if ce:
        hard = torch.log_softmax(u_of(z, cap), -1)
        at = targets[on][:, None]
        loss = loss - ce * hard.gather(1, at)[:, 0]
        size = size + ce * hard.detach().exp().scatter_add(1, at, torch.ones(len(at), 1, dtype=F64, device=z.device))
    d = grad_of(loss.sum() * scale, z, on)
    return scatter_rows(on, loss, z), d, scatter_rows(on, size.detach() * scale, z)


# ------------------------------------------------------------------------------------------- comparing
def value_error(V):
    """Of a log probability, lse or entropy relative to one and its own size: the rounded argument and logarithm, and a row's sum, whose
    terms a thread adds up one by one (some V / 256 of them: their roundings grow as the root)."""
    return 2.0 ** -24 * (40 + 4 * (V / 256) ** 0.5)


def near(got, want, V, cap=0.0, factor=1.0, size=1.0):
    """``size``: of the largest terms a value is the sum of."""
    tol = factor * (value_error(V) + (8e-6 if cap else 0.0)) * (size + want.abs())
    assert got.dtype == torch.float32 and got.shape == want.shape
    bad = ~((got.to(F64) - want).abs() <= tol) & ~((got == want) | (got.isnan() & want.isnan()))
    assert not bool(bad.any()), ((got.to(F64) - want).abs().max(), got[bad][:4], want[bad][:4])


def near_grad(got, want, size, logits, cap=0.0):
    """One rounding to the gradient's type, and what fp32 gives of each term."""
    slope = slope_of(logits, cap)
    half = torch.finfo(got.dtype).eps / 2
    tol = half * want.abs() * 1.01 + (2e-5 if cap else 1e-5) * size * slope + (5e-7 * size if cap else 0.0)
    tol = tol + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps       # steps of the smallest numbers
    bad = ~((got.to(F64) - want).abs() <= tol)
    assert got.shape == want.shape
    assert not bool(bad.any()), (int(bad.sum()), got[bad][:4], want[bad][:4], tol[bad][:4])


def wide(T, V, dtype, device, gap=0, shift=0, fill=7.0, seed=0):
    """Logits as columns of a wider buffer that begin ``shift`` elements in, rows ``gap`` further apart than they are long."""
    g = torch.Generator(device=device).manual_seed(seed)
    buf = torch.full((T, V + gap + shift), fill, dtype=dtype, device=device)
    z = buf[:, shift:shift + V]
    x = 2.5 * torch.randn(T, V, device=device, generator=g)
    x[torch.arange(T, device=device), torch.randint(0, V, (T,), device=device, generator=g)] += 8 * torch.rand(T, device=device, generator=g)
    z.copy_(x)
    return buf, z


def some_targets(T, V, device, seed=0):
    """The first, the last, random ones; one of the ignored kind, one outside."""
    g = torch.Generator(device=device).manual_seed(seed + 1)
    t = torch.randint(0, V, (T,), device=device, generator=g)
    for i, v in enumerate((0, V - 1, -100, V, V // 2)):
        if i < T:
            t[i] = v
    return t


def some_teacher(z, K, tau, cap, seed=0):
    """A teacher near the student: its K likeliest and their log probabilities over the whole vocabulary."""
    g = torch.Generator(device=z.device).manual_seed(seed + 2)
    y = torch.log_softmax(u_of(z.float(), cap) / tau + 0.5 * torch.randn(z.shape, device=z.device, generator=g), -1)
    t, i = torch.topk(y, K)
    return i, t


# --------------------------------------------------------------- the checks, on either kind of device
def check_scores(T, V, dtype, device, K=0, tau=1.0, cap=0.0, gap=0, shift=0, masked=False, given=True, z=None):
    if z is None:
        _, z = wide(T, V, dtype, device, gap, shift)
    t = some_targets(T, V, device) if given else None
    mask = (torch.arange(T, device=device) % 3 != 1).float() if masked else None
    before = z.clone()
    s = ops.token_logprobs(z, t, temperature=tau, softcap=cap, top_k=K, loss_mask=mask)
    assert torch.equal(z.view(torch.int32 if dtype == torch.float32 else torch.int16), before.view(torch.int32 if dtype == torch.float32 else torch.int16))
    on = on_rows(T, V, t, mask, device=device)
    _, _, lp, ent, lse, ids, top = scores(z, t, on, tau, cap, K)
    full = lambda v: scatter_rows(on, v, z)                                                                           # noqa: E731
    if given:
        near(s.logprobs, full(lp), V, cap / tau)
    else:
        assert s.logprobs is None
    near(s.entropy, full(ent), V, cap / tau, size=3.0)
    near(s.lse, full(lse), V, cap / tau)
    if K:
        assert s.top_ids.dtype == torch.int64 and torch.equal(s.top_ids[on], ids) and bool((s.top_ids[~on] == -1).all())
        near(s.top_logprobs[on], top.detach(), V, cap / tau)
        assert bool((s.top_logprobs[~on] == float("-inf")).all())
    else:
        assert s.top_ids is None and s.top_logprobs is None
    return s


def check_scores_grad(T, V, dtype, device, K=0, tau=1.0, cap=0.0, gap=0, shift=0, apart=True, which="lht", twice=False):
    buf, z = wide(T, V, dtype, device, gap, shift)
    t = some_targets(T, V, device)
    on = on_rows(T, V, t, None, device=device)
    s = ops.token_logprobs(z, t, temperature=tau, softcap=cap, top_k=K)
    g = torch.Generator(device=device).manual_seed(5)
    rand = lambda *shape: torch.randn(*shape, device=device, generator=g)                                             # noqa: E731
    dl, dh, dt = rand(T) if "l" in which else None, rand(T) if "h" in which else None, rand(T, K) if K and "t" in which else None
    if twice:
        ids = s.top_ids.clone()
        ids[:, 0], ids[:, 1], ids[:, 2] = ids[:, 3], torch.where(on, t, 0), -1
        s = s._replace(top_ids=ids)
    want, size = scores_grad(z, t, on, tau, cap, dl, dh, s.top_ids, dt, 0.25)
    logits = z.clone()
    out_buf, out = wide(T, V, dtype, device, gap + 3, shift + 1) if apart else (buf, z)
    got = ops.token_logprobs_bwd_(z, t, s, dlogprobs=dl, dentropy=dh, dtop_logprobs=dt, grad_scale=0.25, temperature=tau, softcap=cap,
                                  out=out if apart else None)
    assert got.data_ptr() == out.data_ptr()
    near_grad(got, want, size, logits, cap)
    untouched(out_buf, shift + (1 if apart else 0), V)
    if apart:
        assert torch.equal(z, logits)


def untouched(buf, shift, V):
    assert bool((buf[:, :shift] == 7).all()) and bool((buf[:, shift + V:] == 7).all())


def check_policy(T, V, dtype, device, tau=1.0, cap=0.0, gap=0, shift=0, apart=True, old=True, kept=True, adv=True, bonus=0.01, beta=0.05, masked=False):
    buf, z = wide(T, V, dtype, device, gap, shift)
    t = some_targets(T, V, device)
    mask = (torch.arange(T, device=device) % 3 != 1).float() if masked else None
    on = on_rows(T, V, t, mask, device=device)
    g = torch.Generator(device=device).manual_seed(9)
    lp = torch.zeros(T, device=device)
    lp[on] = scores(z, t, on, tau, cap, 0)[2].detach().float()
    # ratios on either side of the borders and well off them
    step = torch.tensor([0.0, 0.1, -0.1, 0.5, -0.5, 1.2, -1.2], device=device)[torch.randint(0, 7, (T,), device=device, generator=g)]
    kw = dict(old_logprobs=lp - step if old else None, ref_logprobs=lp + 0.5 * torch.randn(T, device=device, generator=g) if kept else None)
    a = torch.randn(T, device=device, generator=g) if adv else None
    (loss, given, ent), want, size = policy(z, t, on, tau, cap, a, kw["old_logprobs"], kw["ref_logprobs"], 0.2, 0.3, beta, bonus, 0.125)
    logits = z.clone()
    kw.update(clip_low=0.2, clip_high=0.3, kl_beta=beta, entropy_coef=bonus, temperature=tau, softcap=cap, loss_mask=mask)
    alone = ops.policy_loss(z, t, a, **kw)
    assert torch.equal(z, logits)
    out_buf, out = wide(T, V, dtype, device, gap + 3, shift + 1) if apart else (buf, z)
    got = ops.policy_loss_(z, t, a, grad_scale=0.125, out=out if apart else None, **kw)
    # (the two may sum a row's terms in other groups: each is held to the definition)
    for terms in (got, alone):
        # an advantage of up to 4 and a ratio of up to 4 multiply the log probability's error
        near(terms.loss, loss, V, cap / tau, factor=20.0)
        near(terms.logprobs, given, V, cap / tau)
        near(terms.entropy, ent, V, cap / tau, size=3.0)
    near_grad(out, want, size, logits, cap)
    untouched(out_buf, shift + (1 if apart else 0), V)


def check_distill(T, V, dtype, device, K=4, tau=1.0, cap=0.0, rest="drop", ce=0.0, gap=0, shift=0, apart=True, given=True, masked=False, change=None):
    buf, z = wide(T, V, dtype, device, gap, shift)
    t = some_targets(T, V, device) if given else None
    mask = (torch.arange(T, device=device) % 3 != 1).float() if masked else None
    on = on_rows(T, V, t, mask, device=device)
    ids, teacher = some_teacher(z, K, tau, cap)
    if change is not None:
        ids, teacher = change(z, ids.clone(), teacher.clone())
    loss, want, size = distill(z, ids, teacher, t, on, rest, ce, tau, cap, 0.125)
    logits = z.clone()
    kw = dict(targets=t, rest=rest, ce_weight=ce, temperature=tau, softcap=cap, loss_mask=mask)
    alone = ops.distill_loss(z, ids, teacher, **kw)
    assert torch.equal(z, logits)
    out_buf, out = wide(T, V, dtype, device, gap + 3, shift + 1) if apart else (buf, z)
    got = ops.distill_loss_(z, ids, teacher, grad_scale=0.125, out=out if apart else None, **kw)
    # sum q (log q - log p): terms of up to 12, times the temperature's square
    for value in (got, alone):
        near(value, loss, V, cap / tau, factor=max(1.0, tau * tau), size=12.0)
    near_grad(out, want, size, logits, cap)
    untouched(out_buf, shift + (1 if apart else 0), V)


def check_not_finite(device):
    """Logits of -inf and of the type's lowest value; rows of nothing else; NaN and infinities in rows that are left out, and in others."""
    inf = float("inf")
    # under a soft-cap -inf is no token, the lowest value is one at the cap
    z = torch.randn(3, 12, generator=torch.Generator().manual_seed(4)).to(device)
    z[0, 3:], z[1, 5:], z[2] = -inf, torch.finfo(torch.float32).min, -inf
    t = torch.tensor([1, 2, 0], device=device)
    s = ops.token_logprobs(z, t, softcap=3.0, top_k=4)
    want = torch.log_softmax(u_of(z.double(), 3.0), -1)
    assert bool(((s.logprobs[:2] - want[[0, 1], [1, 2]]).abs() < 64 * 2.0 ** -24).all()) and s.logprobs[2].isnan()
    assert s.top_ids[0, 3] == 3 and s.top_logprobs[0, 3] == -inf
    p = ops.policy_loss_(z, t, softcap=3.0, out=(out := torch.empty_like(z)))
    assert bool((out[0, 3:] == 0).all()) and bool(out[:2].isfinite().all()) and p.loss[2].isnan()
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        z = torch.randn(8, 12, generator=torch.Generator().manual_seed(3)).to(dtype).to(device)
        z[0, 3:] = -inf
        z[1, 5:] = torch.finfo(dtype).min
        z[2] = -inf
        z[3] = torch.finfo(dtype).min
        z[4, 2] = float("nan")
        z[5, 7] = inf
        z[6] = float("nan")
        t = torch.tensor([1, 2, 0, 4, 1, 1, -100, 3], device=device)
        s = ops.token_logprobs(z, t, top_k=6)
        assert s.top_ids[0].tolist()[3:] == [3, 4, 5] and bool((s.top_logprobs[0, 3:] == -inf).all())
        for r, n in ((0, 3), (1, 5), (3, 12), (7, 12)):           # what is left is a distribution over the first n
            want = torch.log_softmax(z[r, :n].double(), -1)
            tol = 16 * 2.0 ** -24
            assert abs(float(s.logprobs[r] - want[t[r]])) < tol * 4 and abs(float(s.entropy[r] + (want.exp() * want).sum())) < tol * 4
        for r in (2, 4, 5):
            assert s.logprobs[r].isnan() and s.entropy[r].isnan() and s.lse[r].isnan() and bool(s.top_logprobs[r].isnan().all())
        assert s.top_ids[2].tolist() == list(range(6)) and int(s.top_ids[4, 0]) == 2 and int(s.top_ids[5, 0]) == 7
        assert s.logprobs[6] == 0 and s.entropy[6] == 0 and s.lse[6] == 0 and s.top_ids[6].tolist() == [-1] * 6
        ids = torch.tensor([1, 2], device=device).repeat(8, 1)
        q = torch.tensor([-0.5, -1.5], device=device).repeat(8, 1)
        out = torch.empty_like(z)
        for rest in ("drop", "bucket", None, "scores"):
            if rest is None:
                loss = ops.policy_loss_(z, t, entropy_coef=0.1, out=out).loss
            elif rest == "scores":
                loss = s.logprobs
                ops.token_logprobs_bwd_(z, t, s, dlogprobs=torch.ones(8, device=device), dentropy=torch.ones(8, device=device), out=out)
            else:
                loss = ops.distill_loss_(z, ids, q, targets=t, rest=rest, ce_weight=0.25, temperature=2.0, out=out)
            assert loss[6] == 0 and bool((out[6] == 0).all())
            for r in (0, 1, 3, 7) if rest != "scores" else (0, 1, 7):          # (an lse near the lowest value has no digits left for p)
                assert loss[r].isfinite() and bool(out[r].isfinite().all()) and abs(float(out[r].double().sum())) < 0.02
            for r in (2, 4, 5):
                assert loss[r].isnan() and bool(out[r].isnan().any())
            assert bool((out[0, 3:] == 0).all()) and bool((out[1, 5:] == 0).all())
        # no other token has a finite logit: the rest is no outcome; the teacher's token has none: no agreement
        z[0, :3], z[1, 2] = torch.tensor([0.5, 1.0, -inf]).to(z), -inf
        ids[0] = torch.tensor([0, 1], device=device)
        loss = ops.distill_loss_(z, ids, q, rest="bucket", out=out)
        lp = torch.log_softmax(z[0, :2].double(), -1).cpu()
        want = sum(float(torch.tensor(a).exp()) * (a - float(b)) for a, b in zip((-0.5, -1.5), lp))
        assert abs(float(loss[0]) - want) < 16 * 2.0 ** -24 and bool(out[0].isfinite().all()) and loss[1] == inf
