"""Operators on token probabilities: scores of given tokens, policy gradients and distillation, from a head's logits.

A row of ``logits (T, V)`` (bf16, fp16 or fp32) is a token's: ``x = u / temperature``, ``u = softcap * tanh(logits / softcap)`` (the
logits themselves without a soft-cap), ``p = softmax(x)``.  ``x`` and all that follows from it are in fp32; losses and scores are
fp32, gradients have the logits' type and are by the logits as they were given.

Rows that are left out have a target outside ``[0, V)`` (``ignore_index`` among them) or a ``loss_mask`` that is not above zero: they
are not read, their scores, losses and gradients are zero, their alternatives ``-1`` with ``-inf``.  A logit of ``-inf`` is a token
without probability, under a soft-cap too; a row of nothing else, or with a NaN, reads as NaN, and so does one with ``+inf``, but under
a soft-cap that is a token at the cap.

The calls whose names end in ``_`` write the gradient over the logits, or into ``out`` (the same shape and type, beside the logits or
the logits themselves, not partly over them).  A call runs on the device of its tensors, on the stream that is current there; on a
GPU everything here runs on the package's own kernels or raises.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import reference as ref
from .fp8 import _launch, _partly_over

F32 = torch.float32
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MOST_TOP = 128                 # alternatives of a row, tokens of a teacher
MOST_TOKENS = 1600000          # of a vocabulary
TEMPERATURES = (1e-37, 1e18)   # whose reciprocals and squares fp32 has


class TokenLogprobs(NamedTuple):
    """What :func:`token_logprobs` finds of each row, fp32: ``logprobs`` of the given tokens (None without), ``entropy``, ``lse``
    (the logarithm of the sum of ``exp(x)``), and ``top_ids`` (int64) with ``top_logprobs``, both ``(T, top_k)`` (None without)."""
    logprobs: Optional[torch.Tensor]
    entropy: torch.Tensor
    lse: torch.Tensor
    top_ids: Optional[torch.Tensor]
    top_logprobs: Optional[torch.Tensor]


class PolicyTerms(NamedTuple):
    """Of each row, fp32: ``loss``, ``logprobs`` of the given tokens, ``entropy``."""
    loss: torch.Tensor
    logprobs: torch.Tensor
    entropy: torch.Tensor


# ------------------------------------------------------------------------------------------ arguments
def _of_rows(t, T: int, device, dtype, name: str, what: str, K: Optional[int] = None):
    """A value of each row (``K`` of them) as the kernels read it."""
    if t is None:
        return None
    shape = (T,) if K is None else (T, K)
    if t.shape != shape or t.device != device or t.is_complex() or (dtype is not F32 and t.is_floating_point()):
        raise ValueError(f"{what}: {name} {tuple(t.shape)} {t.dtype} on {t.device}, {shape} on {device} is read")
    return t if t.dtype is dtype and t.is_contiguous() else t.to(dtype).contiguous()


def _logits(logits, temperature, softcap, what: str):
    if logits.dim() != 2 or logits.dtype not in _TYPES:
        raise ValueError(f"{what}: logits {tuple(logits.shape)} {logits.dtype}, (T, V) in bf16, fp16 or fp32 are read")
    if not TEMPERATURES[0] <= temperature <= TEMPERATURES[1] or not (softcap == 0.0 or 1e-37 <= softcap <= 1e37):
        raise ValueError(f"{what}: temperature {temperature}, {TEMPERATURES[0]:g} to {TEMPERATURES[1]:g} are read; softcap {softcap}, zero (none) or "
                         "1e-37 to 1e37")
    T, V = logits.shape
    if V == 0 or V > MOST_TOKENS:
        raise ValueError(f"{what}: a vocabulary of {V} tokens, 1 to {MOST_TOKENS} are read")
    return T, V


def _target_rows(targets, loss_mask, T, device, what):
    return (_of_rows(targets, T, device, torch.int64, "targets", what), _of_rows(loss_mask, T, device, F32, "loss_mask", what))


def _along(t):
    """``t`` with the elements of a row next to one another."""
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _gradient(logits, out, what: str):
    """Where the gradient is written."""
    if out is None:
        out = logits
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device or (out.stride(1) != 1 and out.shape[1] > 1) or \
            (out.shape[0] > 1 and out.stride(0) < out.shape[1]):
        raise ValueError(f"{what}: the gradient is written to {tuple(out.shape)} {out.dtype} on {out.device}, strides {out.stride()}; "
                         f"{tuple(logits.shape)} {logits.dtype} on {logits.device} with contiguous rows, none over another, is needed")
    if out is not logits and logits.numel():
        if logits.stride(1) != 1 and logits.shape[1] > 1 or logits.shape[0] > 1 and logits.stride(0) < logits.shape[1]:
            # (rows over one another, or elements apart: no place of it may be written)
            first = logits.data_ptr()
            last = first + sum((n - 1) * s for n, s in zip(logits.shape, logits.stride())) * logits.element_size()
            begin = out.data_ptr()
            end = begin + ((out.shape[0] - 1) * out.stride(0) + out.shape[1]) * out.element_size()
            over = first < end and begin <= last
        else:
            over = _partly_over(logits, out)
        if over:
            raise ValueError(f"{what}: out (strides {out.stride()}) lies partly over the logits (strides {logits.stride()})")
    return out


def _on(logits, targets, loss_mask, ignore_index):
    """Which rows count."""
    on = torch.ones(logits.shape[0], dtype=torch.bool, device=logits.device)
    if targets is not None:
        on = (targets != ignore_index) & (targets >= 0) & (targets < logits.shape[1])
    return on if loss_mask is None else on & (loss_mask > 0)


def _at(t):
    return None if t is None else t.data_ptr()


def _rows_launch(family, entry, z, out, targets, mask, *, loss=None, logprob=None, entropy=None, lse=None, top_ids=None, top_logprob=None, adv=None,
                 old=None, ref_lp=None, ids=None, teacher=None, K=0, ignore=-100, bucket=False, tau=1.0, cap=0.0, scale=1.0, clip_low=0.0,
                 clip_high=0.0, kl=0.0, bonus=0.0, ce=0.0):
    T, V = z.shape
    _launch(family, z.get_device(), "token_loss", entry, z.data_ptr(), _at(out), _at(targets), _at(mask), _at(loss), _at(logprob), _at(entropy), _at(lse),
            _at(top_ids), _at(top_logprob), _at(adv), _at(old), _at(ref_lp), _at(ids), _at(teacher), _TYPES[z.dtype], z.stride(0),
            0 if out is None else out.stride(0), T, V, K, int(ignore), bucket, float(tau), float(cap), float(scale), float(clip_low), float(clip_high),
            float(kl), float(bonus), float(ce))


# --------------------------------------------------------------------------------------------- scores
def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, *, temperature: float = 1.0, softcap: float = 0.0, top_k: int = 0,
                   loss_mask: Optional[torch.Tensor] = None, ignore_index: int = -100) -> TokenLogprobs:
    """Log probability of each row's given token, its entropy, and the ``top_k`` tokens of the largest logits (largest first, the
    lowest id first among equal logits) with theirs; the logits are read once and stay as they are."""
    what = "token_logprobs"
    T, V = _logits(logits, temperature, softcap, what)
    if not 0 <= top_k <= min(MOST_TOP, V):
        raise ValueError(f"{what}: top_k {top_k}, 0 to {min(MOST_TOP, V)} of {V} tokens")
    targets, mask = _target_rows(targets, loss_mask, T, logits.device, what)
    if not logits.is_cuda:
        return TokenLogprobs(*ref.token_logprobs(logits, targets, _on(logits, targets, mask, ignore_index), temperature, softcap, top_k))
    z, device = _along(logits), logits.device
    lp, ent, lse = torch.empty(3, T, dtype=F32, device=device).unbind(0)
    if targets is None:
        lp = None
    ids = torch.empty(T, top_k, dtype=torch.int64, device=device) if top_k else None
    top = torch.empty(T, top_k, dtype=F32, device=device) if top_k else None
    if T:
        _rows_launch(what, "ftb_token_scores", z, None, targets, mask, logprob=lp, entropy=ent, lse=lse, top_ids=ids, top_logprob=top, K=top_k,
                     ignore=ignore_index, tau=temperature, cap=softcap)
    return TokenLogprobs(lp, ent, lse, ids, top)


def token_logprobs_bwd_(logits: torch.Tensor, targets: Optional[torch.Tensor], scores: TokenLogprobs, *, dlogprobs: Optional[torch.Tensor] = None,
                        dentropy: Optional[torch.Tensor] = None, dtop_logprobs: Optional[torch.Tensor] = None, grad_scale: float = 1.0,
                        temperature: float = 1.0, softcap: float = 0.0, loss_mask: Optional[torch.Tensor] = None, ignore_index: int = -100,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``grad_scale`` times the logits' gradient from those of :func:`token_logprobs`'s outputs (any of them None: zero), written over
    the logits or into ``out``, which is returned.  ``scores`` is what the forward call returned for the same arguments: its ``lse``
    is read, its ``entropy`` with ``dentropy`` and its ``top_ids`` with ``dtop_logprobs`` (ids outside the vocabulary have no part,
    an id twice has both).  Probabilities are taken from the fp32 ``lse``, whose rounding is some 2^-24 of it: at an lse of 1,000 they
    are off by 6e-5, and a row that a mask's lowest value leaves nothing else of has lost them."""
    what = "token_logprobs_bwd_"
    T, V = _logits(logits, temperature, softcap, what)
    device = logits.device
    targets, mask = _target_rows(targets, loss_mask, T, device, what)
    if dlogprobs is not None and targets is None:
        raise ValueError(f"{what}: dlogprobs without targets")
    lse = _of_rows(scores.lse, T, device, F32, "scores.lse", what)
    if lse is None or (dentropy is not None and scores.entropy is None) or (dtop_logprobs is not None and scores.top_ids is None):
        raise ValueError(f"{what}: a gradient of something that the scores do not hold")
    ent = _of_rows(scores.entropy, T, device, F32, "scores.entropy", what) if dentropy is not None else None
    dl, dh = _of_rows(dlogprobs, T, device, F32, "dlogprobs", what), _of_rows(dentropy, T, device, F32, "dentropy", what)
    ids, dt, K = None, None, 0
    if dtop_logprobs is not None:
        K = dtop_logprobs.shape[-1] if dtop_logprobs.dim() else 0
        if K > MOST_TOP:
            raise ValueError(f"{what}: {K} alternatives, {MOST_TOP} at most")
        ids, dt = _of_rows(scores.top_ids, T, device, torch.int64, "scores.top_ids", what, K), _of_rows(dtop_logprobs, T, device, F32, "dtop_logprobs", what, K)
    out = _gradient(logits, out, what)
    if not logits.is_cuda:
        return out.copy_(ref.token_logprobs_bwd(logits, targets, _on(logits, targets, mask, ignore_index), lse, ent, dl, dh, ids, dt, grad_scale,
                                                temperature, softcap))
    z = _along(logits)
    if T:
        _launch(what, z.get_device(), "token_loss", "ftb_token_scores_bwd", z.data_ptr(), out.data_ptr(), _at(targets), _at(mask), lse.data_ptr(), _at(ent),
                _at(dl), _at(dh), _at(dt), _at(ids), _TYPES[z.dtype], z.stride(0), out.stride(0), T, V, K, int(ignore_index), float(temperature),
                float(softcap), float(grad_scale))
    return out


# ------------------------------------------------------------------------------------- policy gradient
def _policy(what, logits, targets, advantages, old_logprobs, ref_logprobs, clip_low, clip_high, kl_beta, entropy_coef, temperature, softcap, grad_scale,
            loss_mask, ignore_index, grad, out):
    T, V = _logits(logits, temperature, softcap, what)
    device = logits.device
    if targets is None:
        raise ValueError(f"{what}: targets are needed")
    clip_high = clip_low if clip_high is None else clip_high
    if not (0.0 <= clip_low <= 1.0 and clip_high >= 0.0):
        raise ValueError(f"{what}: clip_low {clip_low} (0 to 1), clip_high {clip_high} (0 and above)")
    targets, mask = _target_rows(targets, loss_mask, T, device, what)
    adv, old, kept = (_of_rows(t, T, device, F32, n, what) for t, n in ((advantages, "advantages"), (old_logprobs, "old_logprobs"), (ref_logprobs, "ref_logprobs")))
    out = _gradient(logits, out, what) if grad else None
    if not logits.is_cuda:
        terms, d = ref.policy_loss(logits, targets, _on(logits, targets, mask, ignore_index), adv, old, kept, clip_low, clip_high, kl_beta, entropy_coef,
                                   temperature, softcap, grad_scale, grad)
        if grad:
            out.copy_(d)
        return PolicyTerms(*terms)
    z = _along(logits)
    loss, lp, ent = torch.empty(3, T, dtype=F32, device=device).unbind(0)
    if T:
        _rows_launch(what, "ftb_policy_loss", z, out, targets, mask, loss=loss, logprob=lp, entropy=ent, adv=adv, old=old, ref_lp=kept, ignore=ignore_index,
                     tau=temperature, cap=softcap, scale=grad_scale, clip_low=clip_low, clip_high=clip_high, kl=kl_beta, bonus=entropy_coef)
    return PolicyTerms(loss, lp, ent)


def policy_loss_(logits: torch.Tensor, targets: torch.Tensor, advantages: Optional[torch.Tensor] = None, *, old_logprobs: Optional[torch.Tensor] = None,
                 ref_logprobs: Optional[torch.Tensor] = None, clip_low: float = 0.2, clip_high: Optional[float] = None, kl_beta: float = 0.0,
                 entropy_coef: float = 0.0, temperature: float = 1.0, softcap: float = 0.0, grad_scale: float = 1.0,
                 loss_mask: Optional[torch.Tensor] = None, ignore_index: int = -100, out: Optional[torch.Tensor] = None) -> PolicyTerms:
    """Policy-gradient loss of the given tokens, in one pass with its gradient (times ``grad_scale``), which is written over the logits
    or into ``out``.  With ``old_logprobs``, those of the policy that sampled, ``r = exp(logp - old)``:

        ``L = -min(r * A, clip(r, 1 - clip_low, 1 + clip_high) * A) + kl_beta * (exp(d) - d - 1) - entropy_coef * H``

    ``d = ref_logprobs - logp`` (no penalty without them), ``clip_high`` is ``clip_low`` unless given; without ``old_logprobs`` the
    first term is ``-A * logp``.  ``advantages`` are one without any."""
    return _policy("policy_loss_", logits, targets, advantages, old_logprobs, ref_logprobs, clip_low, clip_high, kl_beta, entropy_coef, temperature, softcap,
                   grad_scale, loss_mask, ignore_index, True, out)


def policy_loss(logits: torch.Tensor, targets: torch.Tensor, advantages: Optional[torch.Tensor] = None, *, old_logprobs: Optional[torch.Tensor] = None,
                ref_logprobs: Optional[torch.Tensor] = None, clip_low: float = 0.2, clip_high: Optional[float] = None, kl_beta: float = 0.0,
                entropy_coef: float = 0.0, temperature: float = 1.0, softcap: float = 0.0, loss_mask: Optional[torch.Tensor] = None,
                ignore_index: int = -100) -> PolicyTerms:
    """:func:`policy_loss_` without the gradient (held-out data): the logits are read once and stay as they are."""
    return _policy("policy_loss", logits, targets, advantages, old_logprobs, ref_logprobs, clip_low, clip_high, kl_beta, entropy_coef, temperature, softcap,
                   1.0, loss_mask, ignore_index, False, None)


# ---------------------------------------------------------------------------------------- distillation
def _distill(what, logits, teacher_ids, teacher_logprobs, targets, rest, ce_weight, temperature, softcap, grad_scale, loss_mask, ignore_index, grad, out):
    T, V = _logits(logits, temperature, softcap, what)
    device = logits.device
    if rest not in ("drop", "bucket"):
        raise ValueError(f"{what}: rest {rest!r}, 'drop' or 'bucket'")
    if not 0.0 <= ce_weight <= 1.0 or (ce_weight > 0.0 and targets is None):
        raise ValueError(f"{what}: ce_weight {ce_weight} (0 to 1; targets are needed above zero)")
    K = teacher_ids.shape[-1] if teacher_ids.dim() == 2 else 0
    if not 1 <= K <= MOST_TOP:
        raise ValueError(f"{what}: teacher_ids {tuple(teacher_ids.shape)}, (T, K) with K of 1 to {MOST_TOP}")
    ids = _of_rows(teacher_ids, T, device, torch.int64, "teacher_ids", what, K)
    teacher = _of_rows(teacher_logprobs, T, device, F32, "teacher_logprobs", what, K)
    if teacher is None:
        raise ValueError(f"{what}: teacher_logprobs are needed")
    targets, mask = _target_rows(targets, loss_mask, T, device, what)
    out = _gradient(logits, out, what) if grad else None
    if not logits.is_cuda:
        loss, d = ref.distill_loss(logits, ids, teacher, targets, _on(logits, targets, mask, ignore_index), rest == "bucket", ce_weight, temperature,
                                   softcap, grad_scale, grad)
        if grad:
            out.copy_(d)
        return loss
    z = _along(logits)
    loss = torch.empty(T, dtype=F32, device=device)
    if T:
        _rows_launch(what, "ftb_distill_loss", z, out, targets, mask, loss=loss, ids=ids, teacher=teacher, K=K, ignore=ignore_index, bucket=rest == "bucket",
                     tau=temperature, cap=softcap, scale=grad_scale, ce=ce_weight)
    return loss


def distill_loss_(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logprobs: torch.Tensor, *, targets: Optional[torch.Tensor] = None,
                  rest: str = "drop", ce_weight: float = 0.0, temperature: float = 1.0, softcap: float = 0.0, grad_scale: float = 1.0,
                  loss_mask: Optional[torch.Tensor] = None, ignore_index: int = -100, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Distillation from a teacher's ``K`` most likely tokens of each row, ``teacher_ids`` and ``teacher_logprobs (T, K)`` as
    ``token_logprobs(..., temperature=temperature, top_k=K)`` of the teacher's logits gives them; the gradient (times ``grad_scale``)
    is written over the logits or into ``out``.  Returns the loss of each row:

        ``(1 - ce_weight) * temperature ** 2 * KL + ce_weight * CE``,   ``KL = sum_k q_k * (log q_k - log p_k)``

    ``rest="drop"``: ``q`` is renormalised over the K tokens.  ``rest="bucket"``: ``q = exp(teacher_logprobs)``, and all other tokens
    are one further outcome, ``q_r = max(1 - sum(q), 0)`` (left out where no other token has a finite logit).  ``CE`` is the cross
    entropy with ``targets`` at temperature 1; a ``ce_weight`` of one is the cross entropy alone, whatever KL is.  Ids outside the
    vocabulary (padding: ``-1``) have no part; an id twice has both."""
    return _distill("distill_loss_", logits, teacher_ids, teacher_logprobs, targets, rest, ce_weight, temperature, softcap, grad_scale, loss_mask,
                    ignore_index, True, out)


def distill_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logprobs: torch.Tensor, *, targets: Optional[torch.Tensor] = None,
                 rest: str = "drop", ce_weight: float = 0.0, temperature: float = 1.0, softcap: float = 0.0, loss_mask: Optional[torch.Tensor] = None,
                 ignore_index: int = -100) -> torch.Tensor:
    """:func:`distill_loss_` without the gradient (held-out data): the logits are read once and stay as they are."""
    return _distill("distill_loss", logits, teacher_ids, teacher_logprobs, targets, rest, ce_weight, temperature, softcap, 1.0, loss_mask, ignore_index,
                    False, None)
