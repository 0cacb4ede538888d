"""Linear layers in 8 bits: e4m3 operands with an fp32 scale for each block of 128, their quantisers and products.

A matrix in 8 bits is a :class:`Fp8Matrix`: its e4m3 ``data``, and one fp32 ``scale`` for each group of elements:

=========  ===========  ======================================  ==================================================
group      elements     scale of ``(M, N)`` data                read by
=========  ===========  ======================================  ==================================================
``row``    1 x 128      ``(M, ceil(N / 128))``                  products that reduce over ``N`` (activations, ``dy``)
``col``    128 x 1      ``(ceil(M / 128), N)``                  products that reduce over ``M`` (weight gradients)
``block``  128 x 128    ``(ceil(M / 128), ceil(N / 128))``      either (weights, read along and across)
=========  ===========  ======================================  ==================================================

An element's value is ``data * scale``, ``scale = max(largest magnitude / 448, 2^-126)``.  A group with an infinity or a NaN has a
scale that is one, and reads as NaN.  On a GPU everything here runs on the package's own kernels or raises; there is no library
path.  The scales of two operands are multiplied in fp32, so the product of a pair of scales has to be finite and not below
2^-126 to count, and sums below that are zero.
"""
from __future__ import annotations

import ctypes
import functools
import struct
import sys
from typing import NamedTuple, Optional

import torch

from . import reference as ref

_ops = sys.modules[__package__]

FP8, F32, BF16 = torch.float8_e4m3fn, torch.float32, torch.bfloat16
_GROUPS = ("row", "col", "block")
_entries: dict = {}
TILE = 0       # of the products: 0 by size, 1 128 x 128, 2 128 x 256, 3 256 x 256 on two SMs (tests and timings)


class Fp8Matrix(NamedTuple):
    """``data`` ``(M, N)`` e4m3 (``(E, M, N)`` for stacked weights in ``block`` groups), ``scale`` fp32, ``group``."""
    data: torch.Tensor
    scale: torch.Tensor
    group: str

    @property
    def device(self):
        return self.data.device


def _entry(lib: str, name: str):
    """A library's entry point that takes its arguments in 8 bytes each, as a function of them."""
    from . import cuda
    address = ctypes.cast(getattr(cuda.load(lib), name), ctypes.c_void_p).value
    fast = cuda.fastcall()
    if fast is not None:
        return functools.partial(fast.call, address)
    entry, bits = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p)(address), struct.Struct("d")
    word = lambda a: 0 if a is None else int.from_bytes(bits.pack(a), "little", signed=True) if isinstance(a, float) else a

    def call(*args):
        words = (ctypes.c_int64 * len(args))(*map(word, args))       # (held until the entry point has returned)
        return entry(ctypes.addressof(words))
    return call


def _launch(family: str, index: int, lib: str, name: str, *args) -> None:
    """One call of a library's entry point on the device of its tensors, on the stream that is current there."""
    entry = _entries.get(name)
    if entry is None:
        entry = _entries[name] = _entry(lib, name)
    before = torch._C._cuda_getDevice()
    if before == index:
        rc = entry(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        torch._C._cuda_setDevice(index)
        try:
            rc = entry(*args, torch._C._cuda_getCurrentRawStream(index))
        finally:
            torch._C._cuda_setDevice(before)
    if rc != 0:
        raise RuntimeError(f"{name} failed with code {rc}")
    _ops._count()
    _ops._used(family, "ftb")


def _rows(t):
    """``t`` with elements of a row next to one another."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _empty_q(shape, device):
    """e4m3 room for ``shape`` with rows on 16 bytes, as the products read them; the pieces behind a row's end hold nothing."""
    n = shape[-1]
    ld = (n + 15) // 16 * 16
    if len(shape) != 2:
        return torch.empty(*shape[:-1], ld, dtype=FP8, device=device)[..., :n]
    q = torch.empty_strided((shape[0], ld), (ld, 1), dtype=FP8, device=device)      # (1.5 us on the host for 2.4 of torch.empty; a view
    return q if n == ld else q.as_strided((shape[0], n), (ld, 1))                     # of it 0.9 for 2.2 of a slice)


# --------------------------------------------------------------------------------------- quantisers
def quant_fp8(x: torch.Tensor, group: str = "row") -> Fp8Matrix:
    """``x (M, N)`` (bf16 or fp32; also ``(E, M, N)`` for ``block``) in 8 bits."""
    if group not in _GROUPS:
        raise ValueError(f"quant_fp8: group {group!r}, one of {_GROUPS}")
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"quant_fp8: bf16 or fp32, not {x.dtype}")
    if x.dim() != 2 and not (x.dim() == 3 and group == "block"):
        raise ValueError(f"quant_fp8: {tuple(x.shape)} in groups {group!r} (matrices; stacks of them in 'block' groups)")
    if not x.is_cuda:
        return Fp8Matrix(*ref.quant_fp8(x, group), group)
    x = _rows(x)
    M, N = x.shape[-2:]
    q = _empty_q(x.shape, x.device)
    m, n = (M + 127) // 128, (N + 127) // 128
    if group == "row":
        scale = torch.empty_strided((M, n), (1, M), dtype=F32, device=x.device)   # a group's scales of neighbouring rows together
    else:
        scale = torch.empty(*x.shape[:-2], m, N if group == "col" else n, dtype=torch.float32, device=x.device)
    if x.numel() == 0:
        return Fp8Matrix(q, scale.fill_(ref.FP8_FLOOR), group)
    E = x.shape[0] if x.dim() == 3 else 1
    batch = (lambda t: t.stride(0) if x.dim() == 3 else 0)
    _launch("quant_fp8", x.get_device(), "fp8", "ftb_quant_fp8", x.data_ptr(), q.data_ptr(), scale.data_ptr(), x.dtype == F32, x.stride(-2),
            batch(x), q.stride(-2), batch(q), scale.stride(-2), scale.stride(-1), batch(scale), E, M, N, _GROUPS.index(group))
    return Fp8Matrix(q, scale, group)


def dequant_fp8(m: Fp8Matrix, dtype=torch.bfloat16) -> torch.Tensor:
    """The values that ``m`` holds, rounded to ``dtype`` (plain torch operations, for looking at them)."""
    _check(m, "dequant_fp8", stacked=m.data.dim() == 3)
    return ref.dequant_fp8(m.data, m.scale, m.group, dtype)


def rmsnorm_fp8_fwd(x: torch.Tensor, w: Optional[torch.Tensor], eps: float, *, residual: Optional[torch.Tensor] = None):
    """RMSNorm of ``h = x + residual`` (rounded to ``x``'s type), its output in 8 bits: ``(Fp8Matrix in row groups, rstd, h)``.
    Without a residual ``h`` is ``x`` itself.  The backward pass is :func:`rmsnorm_bwd` of ``h`` and ``rstd``, with the residual
    stream's gradient as its ``dx_add``; it re-emits the output in bf16 for a weight gradient (``emit_y``)."""
    if x.dim() != 2 or (residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device)):
        raise ValueError(f"rmsnorm_fp8_fwd: x {tuple(x.shape)} {x.dtype}, residual "
                         f"{None if residual is None else (tuple(residual.shape), residual.dtype, residual.device)}")
    if w is not None and (w.shape != x.shape[1:] or w.device != x.device):
        raise ValueError(f"rmsnorm_fp8_fwd: gain {tuple(w.shape)} on {w.device} for rows of {x.shape[1]} on {x.device}")
    if x.dtype not in ((torch.bfloat16,) if x.is_cuda else (torch.bfloat16, torch.float32)):
        raise ValueError(f"rmsnorm_fp8_fwd: {x.dtype} on {x.device.type} (bf16; fp32 on the CPU only)")
    if not x.is_cuda:
        q, scale, rstd, h = ref.rmsnorm_fp8_fwd(x, w, eps, residual)
        return Fp8Matrix(q, scale, "row"), rstd, h
    T, D = x.shape
    device, h = x.device, x
    x = _rows(x)
    if w is not None and (w.dtype is not F32 or not w.is_contiguous()):
        w = w.to(F32).contiguous()
    q = _empty_q((T, D), device)
    scale = torch.empty_strided((T, (D + 127) // 128), (1, T), dtype=F32, device=device)
    rstd = torch.empty(T, dtype=F32, device=device)
    if residual is not None:
        residual = _rows(residual)
        h = torch.empty(T, D, dtype=x.dtype, device=device)
    if D == 0:
        return Fp8Matrix(q, scale, "row"), rstd.fill_(eps ** -0.5), h
    if T:
        r = (None, None, 0) if residual is None else (residual.data_ptr(), h.data_ptr(), residual.stride(0))
        _launch("rmsnorm_fp8_fwd", x.get_device(), "fp8", "ftb_rmsnorm_fp8_fwd", x.data_ptr(), r[0], None if w is None else w.data_ptr(),
                q.data_ptr(), scale.data_ptr(), rstd.data_ptr(), r[1], x.stride(0), r[2], q.stride(0), T, T, D, float(eps))
    return Fp8Matrix(q, scale, "row"), rstd, h


# ----------------------------------------------------------------------------------------- products
def _check(m, what: str, stacked: bool = False) -> None:
    """That ``m`` is a matrix in 8 bits whose parts fit together."""
    q, s, group = m
    if q.dtype is FP8 and s.dtype is F32 and group in _GROUPS and q.get_device() == s.get_device():
        a, b = q.shape, s.shape
        if len(a) == len(b) == (3 if stacked else 2):
            rows, cols = a[-2], a[-1]
            if b[-2] == (rows if group == "row" else (rows + 127) >> 7) and b[-1] == (cols if group == "col" else (cols + 127) >> 7) and \
                    (not stacked or a[0] == b[0]):
                return
    raise ValueError(f"{what}: {'a stack of matrices' if stacked else 'a matrix'} in 8 bits is read here; data {tuple(q.shape)} {q.dtype} on "
                     f"{q.device}, scale {tuple(s.shape)} {s.dtype} on {s.device}, group {group!r}")


def _along(m, trans: bool, what: str):
    """``(step of a row or column of the product, step of a block of the reduction, shift)`` of an operand's scale.  ``trans``: the
    reduction runs down the data's columns."""
    if m[2] != "block" and m[2] != ("col" if trans else "row"):
        raise ValueError(f"{what}: groups {m.group!r}, and the reduction runs {'down the columns' if trans else 'along the rows'}")
    st = m[1].stride()
    return (st[-1], st[-2], 7 if m[2] == "block" else 0) if trans else (st[-2], st[-1], 7 if m[2] == "block" else 0)


def _on_grid(q):
    """Data as the tensor maps describe it (rows contiguous, everything on 16 bytes; copied where it lies otherwise), its address and
    what is between its rows and matrices."""
    st, at = q.stride(), q.data_ptr()
    if at & 15 or st[-2] & 15 or st[-2] < q.shape[-1] or (st[-1] != 1 and q.shape[-1] != 1) or (len(st) == 3 and (st[0] <= 0 or st[0] & 15)):
        buf = _empty_q(q.shape, q.device)
        buf.view(torch.uint8).copy_(q.view(torch.uint8))
        q, st, at = buf, buf.stride(), buf.data_ptr()
    return q, at, st[-2], st[0]


def _result(out, M: int, N: int, dtype, like, what: str):
    if out is None:
        return torch.empty_strided((M, N), (N, 1), dtype=dtype, device=like.device)
    if out.shape != (M, N) or (out.dtype is not BF16 and out.dtype is not F32) or out.get_device() != like.get_device() or \
            (out.stride(-1) != 1 and N > 1) or (M > 1 and out.stride(0) < N):
        raise ValueError(f"{what}: out {tuple(out.shape)} {out.dtype} on {out.device}, strides {out.stride()}; "
                         f"{(M, N)} in bf16 or fp32 with contiguous rows, none over another, on {like.device}")
    return out


def _partly_over(c, d) -> bool:
    """Whether ``c`` shares elements with ``d`` other than as the same matrix in the same place (both with contiguous rows)."""
    (M, N), (lc, _), (ld, _), es = d.shape, c.stride(), d.stride(), d.element_size()
    at = c.data_ptr() - d.data_ptr()
    if at == 0 and (M == 1 or lc == ld):
        return False
    if at >= ((M - 1) * ld + N) * es or -at >= ((M - 1) * lc + N) * es:
        return False
    return M == 1 or lc != ld or not N * es <= at % (ld * es) <= (ld - N) * es


def gemm_fp8(a: Fp8Matrix, b: Fp8Matrix, *, trans_a: bool = False, trans_b: bool = False, alpha: float = 1.0, beta: float = 0.0, c=None,
             bias=None, out=None, out_dtype=None):
    """``alpha * op(a) @ op(b) + beta * c (+ bias)`` as :func:`gemm` has it, of operands in 8 bits; ``c`` is ``out`` where only that is
    given, and may be ``out`` itself, but not lie partly over it.  The result is bf16 or fp32, rounded once from fp32 sums."""
    _check(a, "gemm_fp8 (a)")
    _check(b, "gemm_fp8 (b)")
    sa_m, sa_k, sa_shift = _along(a, trans_a, "gemm_fp8 (a)")
    sb_n, sb_k, sb_shift = _along(b, not trans_b, "gemm_fp8 (b)")
    qa, qb = a.data, b.data
    K, M = qa.shape if trans_a else qa.shape[::-1]
    N, kb = qb.shape if trans_b else qb.shape[::-1]
    if K != kb or qa.get_device() != qb.get_device():
        raise ValueError(f"gemm_fp8: {tuple(qa.shape)} trans_a={trans_a} on {qa.device} by {tuple(qb.shape)} trans_b={trans_b} on {qb.device}")
    dtype = out_dtype or (out.dtype if out is not None else torch.bfloat16)
    if (dtype is not BF16 and dtype is not F32) or (out is not None and out.dtype != dtype):
        raise ValueError(f"gemm_fp8: a result in {dtype}, out in {None if out is None else out.dtype}")
    if beta != 0.0 and c is None and out is None:
        raise ValueError("gemm_fp8: beta without c or out")
    D = _result(out, M, N, dtype, qa, "gemm_fp8")
    if beta == 0.0:
        c = None
    elif c is None:
        c = D
    elif c.shape != D.shape or c.dtype != dtype or c.device != D.device:
        raise ValueError(f"gemm_fp8: c {tuple(c.shape)} {c.dtype} on {c.device} for a result {tuple(D.shape)} {dtype}")
    else:
        c = _rows(c)
        if out is not None and M and N and _partly_over(c, D):
            raise ValueError(f"gemm_fp8: c (strides {c.stride()}) lies partly over the result (strides {D.stride()})")
    if bias is not None and (bias.shape != (N,) or bias.dtype != torch.float32 or bias.device != D.device):
        raise ValueError(f"gemm_fp8: bias {tuple(bias.shape)} {bias.dtype} on {bias.device}, fp32 of {N} is read")
    if M == 0 or N == 0:
        return D
    if not qa.is_cuda or K == 0:
        return ref.gemm(ref.dequant_fp8(*a), ref.dequant_fp8(*b), trans_a=trans_a, trans_b=trans_b, alpha=alpha, beta=beta, c=c, bias=bias, out=D)
    (qa, at, lda, _), (qb, bt, ldb, _) = _on_grid(qa), _on_grid(qb)
    if bias is not None:
        bias = bias.contiguous()
    _launch("gemm_fp8", qa.get_device(), "gemm_fp8", "ftb_gemm_fp8", at, bt, D.data_ptr(),
            None if c is None else c.data_ptr(), None if bias is None else bias.data_ptr(), a.scale.data_ptr(), b.scale.data_ptr(), None, M, N, K,
            trans_a, not trans_b, lda, ldb, D.stride(0), 0 if c is None else c.stride(0), sa_m, sa_k, sa_shift, sb_n, sb_k,
            sb_shift, 0, float(alpha), float(beta), dtype is F32, 0, 0, 0, 0, TILE, 0)
    return D


def linear_fp8_fwd(x: Fp8Matrix, w: Fp8Matrix, *, bias=None, residual=None, out=None, out_dtype=None):
    """``y = x @ w.T (+ bias) (+ residual)``, ``x`` in row groups, ``w (out, in)`` in blocks (or row groups)."""
    return _ops.gemm_fp8(x, w, trans_b=True, beta=0.0 if residual is None else 1.0, c=residual, bias=bias, out=out, out_dtype=out_dtype)


def linear_fp8_dgrad(dy: Fp8Matrix, w: Fp8Matrix, *, out=None, accumulate=False, out_dtype=None):
    """``dx = dy @ w``, ``dy`` in row groups, the same ``w (out, in)`` in blocks read across; optionally accumulated into ``out``."""
    return _ops.gemm_fp8(dy, w, beta=1.0 if accumulate else 0.0, out=out, out_dtype=out_dtype)


def linear_fp8_wgrad(dy: Fp8Matrix, x: Fp8Matrix, gw, *, alpha=1.0, accumulate=True):
    """``gw (out, in) (+)= alpha * dy.T @ x`` of operands in column groups or blocks (the reduction runs over the tokens); ``x`` in
    blocks is the fast form: a scale for each column of the result costs as much again as its sums."""
    return _ops.gemm_fp8(dy, x, trans_a=True, alpha=alpha, beta=1.0 if accumulate else 0.0, out=gw)


def _offsets(offsets, E: int, like, what: str):
    if offsets.shape != (E + 1,) or offsets.dtype not in (torch.int32, torch.int64) or offsets.device != like.device:
        raise ValueError(f"{what}: offsets {tuple(offsets.shape)} {offsets.dtype} on {offsets.device} for {E} experts on {like.device}")
    if offsets.dtype is torch.int64:                     # (what lies outside of 32 bits stays outside of the rows)
        offsets = offsets.clamp(-(1 << 31), (1 << 31) - 1)
    return offsets.to(torch.int32).contiguous()


def grouped_gemm_fp8(x: Fp8Matrix, w: Fp8Matrix, offsets, *, trans_w: bool = True, out=None, alpha: float = 1.0, beta: float = 0.0):
    """``out[rows_e] = alpha * x[rows_e] @ op(w[e]) + beta * out[rows_e]`` for every expert in one launch: ``x (R, K)`` in row groups,
    ``w (E, N, K)`` (``trans_w``) or ``(E, K, N)`` in blocks, ``rows_e = offsets[e]:offsets[e + 1]`` of any number.  Rows behind the last
    segment are left as they are.  The offsets are read on the device; they ascend, and what they name outside of the rows is left out."""
    _check(x, "grouped_gemm_fp8 (x)")
    _check(w, "grouped_gemm_fp8 (w)", stacked=True)
    sa_m, sa_k, sa_shift = _along(x, False, "grouped_gemm_fp8 (x)")
    sb_n, sb_k, _ = _along(w, not trans_w, "grouped_gemm_fp8 (w)")
    if x.group != "row" or w.group != "block":
        raise ValueError(f"grouped_gemm_fp8: x in groups {x.group!r}, w in {w.group!r}; 'row' and 'block' are read")
    E = w.data.shape[0]
    N, kw = w.data.shape[1:] if trans_w else w.data.shape[:0:-1]
    R, K = x.data.shape
    if K != kw or x.data.device != w.data.device:
        raise ValueError(f"grouped_gemm_fp8: {tuple(x.data.shape)} on {x.data.device} by {tuple(w.data.shape)} trans_w={trans_w} on {w.data.device}")
    off = _offsets(offsets, E, x.data, "grouped_gemm_fp8")
    if beta != 0.0 and out is None:
        raise ValueError("grouped_gemm_fp8: beta without out")
    D = _result(out, R, N, BF16, x.data, "grouped_gemm_fp8")
    if R == 0 or N == 0 or E == 0:
        return D
    if not x.data.is_cuda or K == 0:
        xf, wf, o = ref.dequant_fp8(*x), ref.dequant_fp8(*w), off.tolist()
        for e in range(E):
            i, j = min(max(o[e], 0), R), min(o[e + 1], R)
            if j > i:
                ref.gemm(xf[i:j], wf[e], trans_b=trans_w, alpha=alpha, beta=beta, out=D[i:j])
        return D
    (qx, xt, ldx, _), (qw, wt, ldw, stack) = _on_grid(x.data), _on_grid(w.data)
    _launch("grouped_gemm_fp8", qx.get_device(), "gemm_fp8", "ftb_gemm_fp8", xt, wt, D.data_ptr(), None, None,
            x.scale.data_ptr(), w.scale.data_ptr(), off.data_ptr(), R, N, K, 0, not trans_w, ldx, ldw, D.stride(0), 0, sa_m,
            sa_k, sa_shift, sb_n, sb_k, 7, w.scale.stride(0), float(alpha), float(beta), D.dtype is F32, 1, E, stack, 0, TILE, 0)
    return D


def grouped_wgrad_fp8(dy: Fp8Matrix, x: Fp8Matrix, offsets, gw, *, alpha: float = 1.0, pad: int = 1):
    """``gw[e] += alpha * dy[rows_e].T @ x[rows_e]``, ``dy`` in column groups and ``x`` in those or blocks, ``gw (E, N, K)`` bf16 or
    fp32.  Every expert's segment is padded to a multiple of 128 rows with zero rows (``pad``, as the routing plan lays them out), so
    that no group of 128 tokens lies in two segments.  A segment that starts or ends inside a group is not read, and its expert keeps
    its ``gw``: on a GPU the library's error word reports it (``device_error_words``), on the CPU it is a ``ValueError``.  An expert
    without rows keeps its ``gw``."""
    _check(dy, "grouped_wgrad_fp8 (dy)")
    _check(x, "grouped_wgrad_fp8 (x)")
    if dy.group != "col" or x.group not in ("col", "block"):
        raise ValueError(f"grouped_wgrad_fp8: dy in groups {dy.group!r}, x in {x.group!r}; 'col', and 'col' or 'block', are read")
    if pad < 1 or pad % 128:
        raise ValueError(f"grouped_wgrad_fp8: segments padded to {pad} rows; a multiple of 128 is read")
    (R, N), (Rx, K) = dy.data.shape, x.data.shape
    E = gw.shape[0] if gw.dim() == 3 else -1
    if R != Rx or gw.shape != (E, N, K) or gw.dtype not in (torch.bfloat16, torch.float32) or not gw.is_contiguous() or \
            not dy.data.device == x.data.device == gw.device:
        raise ValueError(f"grouped_wgrad_fp8: dy {tuple(dy.data.shape)} on {dy.data.device}, x {tuple(x.data.shape)} on {x.data.device}, gw "
                         f"{tuple(gw.shape)} {gw.dtype} on {gw.device}, strides {gw.stride()}")
    off = _offsets(offsets, E, gw, "grouped_wgrad_fp8")
    if R == 0 or gw.numel() == 0:
        return gw
    if not gw.is_cuda:
        df, xf, o = ref.dequant_fp8(*dy), ref.dequant_fp8(*x), off.tolist()
        segments = [(min(max(i, 0), R), min(j, R)) for i, j in zip(o, o[1:])]
        for e, (i, j) in enumerate(segments):
            if j > i and (o[e] % 128 or (o[e + 1] % 128 and j < R)):
                raise ValueError(f"grouped_wgrad_fp8: rows {o[e]}:{o[e + 1]} of {R} start or end inside a group of 128")
        for e, (i, j) in enumerate(segments):
            if j > i:
                ref.gemm(df[i:j], xf[i:j], trans_a=True, alpha=alpha, beta=1.0, out=gw[e])
        return gw
    sa_m, sa_k, _ = _along(dy, True, "grouped_wgrad_fp8 (dy)")
    sb_n, sb_k, sb_shift = _along(x, True, "grouped_wgrad_fp8 (x)")
    (qd, dt, ldd, _), (qx, xt, ldx, _) = _on_grid(dy.data), _on_grid(x.data)
    _launch("grouped_wgrad_fp8", gw.get_device(), "gemm_fp8", "ftb_gemm_fp8", dt, xt, gw.data_ptr(), None, None,
            dy.scale.data_ptr(), x.scale.data_ptr(), off.data_ptr(), N, K, R, 1, 1, ldd, ldx, gw.stride(1), 0, sa_m, sa_k, 0,
            sb_n, sb_k, sb_shift, 0, float(alpha), 1.0, gw.dtype is F32, 2, E, 0, gw.stride(0), TILE, 0)
    return gw
