"""Loss functions plugged into the LM head (flextrain/nn/loss.py:68-442).

A loss receives the logits of one micro-chunk and turns them *in place* into ``dZ`` scaled by
``grad_scale`` (the per-step ``1 / active_tokens`` factor), returning per-token losses; the
``(T, V)`` logits never exist for more than one micro-chunk.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Dict, Optional, Protocol

import torch

from .. import ops
from ..ops.token_loss import MOST_TOKENS


@dataclass
class TokenSlice:
    """What a loss needs for the rows of one micro-chunk (flextrain/nn/loss.py:66-106); ``labels`` is the
    reference's name for ``targets``."""
    targets: Optional[torch.Tensor] = None
    loss_mask: Optional[torch.Tensor] = None
    advantages: Optional[torch.Tensor] = None
    ref_logprobs: Optional[torch.Tensor] = None
    offset: int = 0
    size: Optional[int] = None
    extra: Dict[str, torch.Tensor] = field(default_factory=dict)
    labels: Optional[torch.Tensor] = field(default=None, repr=False)

    def __post_init__(self):
        if self.targets is None:
            self.targets = self.labels
        self.labels = self.targets
        if self.size is None and self.targets is not None:
            self.size = int(self.targets.shape[0])


@dataclass
class TokenContext:
    """The same fields for a whole training chunk; :meth:`slice_for` narrows them to a micro-chunk
    (flextrain/nn/loss.py:108-166)."""
    labels: Optional[torch.Tensor] = None
    loss_mask: Optional[torch.Tensor] = None
    advantages: Optional[torch.Tensor] = None
    ref_logprobs: Optional[torch.Tensor] = None
    extra: Dict[str, torch.Tensor] = field(default_factory=dict)

    def slice_for(self, offset: int, size: int) -> TokenSlice:
        cut = lambda t: None if t is None else t[offset:offset + size]
        return TokenSlice(cut(self.labels), cut(self.loss_mask), cut(self.advantages), cut(self.ref_logprobs),
                          offset=offset, size=size, extra={k: v[offset:offset + size] for k, v in self.extra.items()})

    @property
    def total_tokens(self) -> int:
        for t in (self.labels, self.loss_mask, self.advantages, self.ref_logprobs, *self.extra.values()):
            if t is not None:
                return int(t.shape[0])
        raise ValueError("TokenContext is empty; cannot infer total_tokens")


class LossFn(Protocol):
    """``loss(logits, token_slice, grad_scale, softcap) -> per-token losses``, with the logits overwritten by
    ``dZ * grad_scale``.  A loss written for the reference, an object with
    ``compute(logits, token_slice, *, loss_scale, per_token_loss_out) -> (dZ, aux)`` and UNscaled ``dZ``
    (flextrain/nn/loss.py:174-213), is accepted too: :func:`apply_loss` adapts it."""

    def __call__(self, logits: torch.Tensor, sl: TokenSlice, grad_scale: float, softcap: float) -> torch.Tensor: ...


def apply_loss(loss_fn, logits: torch.Tensor, sl: TokenSlice, grad_scale: float, softcap: float = 0.0) -> torch.Tensor:
    """Run either kind of loss on one micro-chunk: ``logits`` becomes ``dZ * grad_scale``, the per-token losses come
    back.  For a ``compute``-style loss the final soft-cap, which the built-in kernels fuse, is applied here: the loss
    sees the capped logits and its gradient is carried back through the cap."""
    if callable(loss_fn) and (getattr(loss_fn, "_native", False) or not hasattr(loss_fn, "compute")):
        return loss_fn(logits, sl, grad_scale, softcap)
    out = torch.empty(logits.shape[0], dtype=torch.float32, device=logits.device)
    slope = None
    if softcap and softcap > 0:
        capped = torch.tanh(logits.to(torch.float32) / softcap)
        slope = 1.0 - capped * capped
        logits.copy_((capped * softcap).to(logits.dtype))
    ret = loss_fn.compute(logits, sl, loss_scale=grad_scale, per_token_loss_out=out)
    dz = ret[0] if isinstance(ret, tuple) else ret
    if dz is not logits:
        logits.copy_(dz.to(logits.dtype))
    if slope is not None:
        logits.copy_((logits.to(torch.float32) * slope * grad_scale).to(logits.dtype))
    else:
        logits.mul_(grad_scale)
    return out


class _NativeLoss:
    """Built-in losses answer to both call styles."""
    _native = True

    def compute(self, logits, token_slice, *, loss_scale: float = 1.0, per_token_loss_out=None):
        """The reference's entry point: UNscaled ``dZ`` written over the logits; returns ``(dZ, {})``."""
        per_tok = self(logits, token_slice, 1.0, 0.0)
        if per_token_loss_out is not None:
            per_token_loss_out.copy_(per_tok)
        return logits, {}


class CrossEntropyLoss(_NativeLoss):
    """Softmax cross-entropy; ``-100`` targets and ``loss_mask <= 0`` rows contribute neither loss nor gradient."""

    def __init__(self, ignore_index: int = -100):
        self.ignore_index = int(ignore_index)

    def __call__(self, logits, sl: TokenSlice, grad_scale: float, softcap: float = 0.0) -> torch.Tensor:
        return ops.softmax_ce_(logits, sl.targets, grad_scale=grad_scale, softcap=softcap, loss_mask=sl.loss_mask,
                               ignore_index=self.ignore_index)

    def loss_only(self, logits, sl: TokenSlice, softcap: float = 0.0) -> torch.Tensor:
        """The losses without the gradient: the logits are read once and not written."""
        return ops.softmax_ce_loss(logits, sl.targets, softcap=softcap, loss_mask=sl.loss_mask,
                                   ignore_index=self.ignore_index)


class MSELoss(_NativeLoss):
    """Mean-squared error between logits and one-hot targets (regression / debugging head)."""

    def __call__(self, logits, sl: TokenSlice, grad_scale: float, softcap: float = 0.0) -> torch.Tensor:
        z = logits.to(torch.float32)
        valid = (sl.targets != -100)
        onehot = torch.zeros_like(z).scatter_(1, sl.targets.clamp(min=0).long().unsqueeze(1), 1.0)
        diff = (z - onehot) * valid.unsqueeze(1)
        logits.copy_((2.0 * diff * grad_scale / z.shape[1]).to(logits.dtype))
        return diff.pow(2).mean(-1)


class GRPOLoss(_NativeLoss):
    """Policy-gradient loss with per-token advantages and an optional KL penalty to reference log-probs:
    ``L = -A * logp(target) + beta * KL(pi || ref)`` using the k3 estimator on the taken token
    (``kl_coef`` is the reference's name for ``kl_beta``)."""

    def __init__(self, kl_beta: float = 0.0, *, kl_coef: Optional[float] = None):
        self.kl_beta = float(kl_coef if kl_coef is not None else kl_beta)

    def __call__(self, logits, sl: TokenSlice, grad_scale: float, softcap: float = 0.0) -> torch.Tensor:
        if logits.is_cuda and logits.dtype in (torch.bfloat16, torch.float16, torch.float32) and logits.shape[1] <= MOST_TOKENS:
            # (as below: no mask but -100, other negative targets are token 0, one advantage may stand for all, and the logits as they are)
            t, rows = sl.targets.long(), logits if logits.stride(1) == 1 else logits.contiguous()
            all_rows = lambda v: None if v is None else v.to(logits.device, torch.float32).expand(t.shape)                 # noqa: E731
            loss = ops.policy_loss_(rows, torch.where(t == -100, t, t.clamp(min=0)), all_rows(sl.advantages),
                                    ref_logprobs=all_rows(sl.ref_logprobs) if self.kl_beta > 0 else None, kl_beta=max(self.kl_beta, 0.0),
                                    grad_scale=grad_scale).loss
            return loss if rows is logits else (logits.copy_(rows), loss)[1]
        z = logits.to(torch.float32)
        valid = (sl.targets != -100).to(torch.float32)
        tgt = sl.targets.clamp(min=0).long()
        logp = torch.log_softmax(z, -1)
        lp = logp.gather(1, tgt.unsqueeze(1)).squeeze(1)
        adv = sl.advantages.to(torch.float32) if sl.advantages is not None else torch.ones_like(lp)
        coef = -adv
        loss = -adv * lp
        if self.kl_beta > 0 and sl.ref_logprobs is not None:
            d = sl.ref_logprobs.to(torch.float32) - lp
            loss = loss + self.kl_beta * (torch.exp(d) - d - 1)
            coef = coef + self.kl_beta * (1 - torch.exp(d))
        p = torch.exp(logp)
        onehot = torch.zeros_like(p).scatter_(1, tgt.unsqueeze(1), 1.0)
        dz = (onehot - p) * (coef * valid * grad_scale).unsqueeze(1)
        logits.copy_(dz.to(logits.dtype))
        return loss * valid


class PolicyLoss(_NativeLoss):
    """Clipped policy gradient (``ops.policy_loss_``): the ratio to ``Sequence.old_logprobs`` (without them ``-A * logp``), per-token
    ``advantages``, a k3 KL penalty to ``ref_logprobs`` and an entropy bonus, under the head's soft-cap and at a temperature.  Rows
    whose target is ``-100`` or whose ``loss_mask`` is not above zero contribute nothing.  All of a call's sequences carry
    ``old_logprobs`` or none; with a penalty the same holds for ``ref_logprobs``."""

    def __init__(self, clip_low: float = 0.2, clip_high: Optional[float] = None, *, kl_coef: float = 0.0, entropy_coef: float = 0.0,
                 temperature: float = 1.0, ignore_index: int = -100):
        self.options = dict(clip_low=float(clip_low), clip_high=None if clip_high is None else float(clip_high), kl_beta=float(kl_coef),
                            entropy_coef=float(entropy_coef), temperature=float(temperature), ignore_index=int(ignore_index))

    def check_sequences(self, seqs) -> None:
        """What only some of a call's sequences carry would be zeros for the others."""
        if len({s.old_logprobs is None for s in seqs}) > 1:
            raise ValueError("PolicyLoss: some sequences of the step carry old_logprobs and some do not")
        if self.options["kl_beta"] != 0.0 and len({s.ref_logprobs is None for s in seqs}) > 1:
            raise ValueError("PolicyLoss: some sequences of the step carry ref_logprobs and some do not")

    def _given(self, sl: TokenSlice, softcap: float):
        ref = sl.ref_logprobs if sl.ref_logprobs is not None else sl.extra.get("ref_logprobs")
        return dict(old_logprobs=sl.extra.get("old_logprobs"), ref_logprobs=ref, softcap=softcap, loss_mask=sl.loss_mask, **self.options)

    def __call__(self, logits, sl: TokenSlice, grad_scale: float, softcap: float = 0.0) -> torch.Tensor:
        return ops.policy_loss_(logits, sl.targets, sl.advantages, grad_scale=grad_scale, **self._given(sl, softcap)).loss

    def loss_only(self, logits, sl: TokenSlice, softcap: float = 0.0) -> torch.Tensor:
        """The losses without the gradient: the logits are read once and not written."""
        return ops.policy_loss(logits, sl.targets, sl.advantages, **self._given(sl, softcap)).loss


class DistillationLoss(_NativeLoss):
    """Distillation from a teacher's most likely tokens (``ops.distill_loss_``), ``Sequence.teacher_ids`` and ``teacher_logprobs`` as
    ``ActiveModel.score(..., top_k=K, temperature=temperature)`` of the teacher gives them, mixed with ``ce_weight`` of the targets'
    cross entropy.  Rows of a step without a teacher's tokens have the cross entropy's part alone."""

    def __init__(self, *, rest: str = "drop", ce_weight: float = 0.0, temperature: float = 1.0, ignore_index: int = -100):
        self.options = dict(rest=rest, ce_weight=float(ce_weight), temperature=float(temperature), ignore_index=int(ignore_index))

    def check_sequences(self, seqs) -> None:
        """Without a teacher's tokens anywhere there is nothing but cross entropy.  (A rank among others takes part all the same: the
        teacher's sequences may be theirs, and they would wait for it.)"""
        alone = not (torch.distributed.is_available() and torch.distributed.is_initialized() and torch.distributed.get_world_size() > 1)
        if self.options["ce_weight"] == 0.0 and seqs and alone and not any(s.teacher_ids is not None for s in seqs):
            raise ValueError("DistillationLoss: no sequence carries teacher_ids and teacher_logprobs")

    def _given(self, logits, sl: TokenSlice, softcap: float):
        ids, lps = sl.extra.get("teacher_ids"), sl.extra.get("teacher_logprobs")
        if ids is None:
            ids = torch.full((logits.shape[0], 1), -1, dtype=torch.int64, device=logits.device)
            lps = torch.zeros(logits.shape[0], 1, dtype=torch.float32, device=logits.device)
        return (logits, ids, lps), dict(targets=sl.targets, softcap=softcap, loss_mask=sl.loss_mask, **self.options)

    def __call__(self, logits, sl: TokenSlice, grad_scale: float, softcap: float = 0.0) -> torch.Tensor:
        args, kw = self._given(logits, sl, softcap)
        return ops.distill_loss_(*args, grad_scale=grad_scale, **kw)

    def loss_only(self, logits, sl: TokenSlice, softcap: float = 0.0) -> torch.Tensor:
        """The losses without the gradient: the logits are read once and not written."""
        args, kw = self._given(logits, sl, softcap)
        return ops.distill_loss(*args, **kw)


class TokenScorer(_NativeLoss):
    """What ``ActiveModel.score`` runs in a loss's place: keeps the scores of each micro-chunk; the losses are the negative log
    probabilities."""

    def __init__(self, top_k: int = 0, temperature: float = 1.0):
        self.top_k, self.temperature = int(top_k), float(temperature)
        self._pieces: list = []

    def __call__(self, logits, sl: TokenSlice, grad_scale: float, softcap: float = 0.0) -> torch.Tensor:
        raise RuntimeError("scores have no gradient here; ops.token_logprobs_bwd_ takes theirs")

    def loss_only(self, logits, sl: TokenSlice, softcap: float = 0.0) -> torch.Tensor:
        s = ops.token_logprobs(logits, sl.targets, temperature=self.temperature, softcap=softcap, top_k=self.top_k, loss_mask=sl.loss_mask)
        self._pieces.append(s)
        return -s.logprobs

    def take(self) -> "ops.TokenLogprobs":
        """The scores since the last call, row after row."""
        got, self._pieces = self._pieces, []
        return ops.TokenLogprobs(*(None if p[0] is None else torch.cat(p) for p in zip(*got)))


def has_loss_only(loss_fn) -> bool:
    """Whether held-out data may take the loss's own form without a gradient: the class that defines the one has to define the other."""
    owner = lambda name: next((c for c in type(loss_fn).__mro__ if name in vars(c)), None)
    return (getattr(loss_fn, "_native", False) and isinstance(loss_fn, (PolicyLoss, DistillationLoss, TokenScorer))
            and owner("__call__") is owner("loss_only"))
