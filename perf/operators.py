"""What is measured of the linear layers in 8 bits: e4m3 values with an fp32 scale for each block of 128.

* ``quant``    an activation, gradient or weight turned into e4m3 with scales of 128 along a row (``row``), down a column
               (``col``: the weight gradient reduces over tokens) or of squares of 128 x 128 (``block``: weights)
* ``norm``     the RMSNorm in front of a projection, with the residual's addition where it has one, written in 8 bits
* ``gemm``     ``fwd`` x W^T (optionally added to a residual), ``dgrad`` dy W, ``wgrad`` dy^T x added to fp32 sums
* ``grouped``  the same three for the experts of a layer, whose rows follow one another in ragged segments

Where ``own`` is true ``run`` makes the framework's calls, elsewhere it computes the same from elementary torch operations.
"""
import torch

own = False

FP8 = torch.float8_e4m3fn
TOP, FLOOR = 448.0, 2.0 ** -126


def listed():
    return [
        # the output gradient of a projection before its input gradient: one step's tokens at a width of 4096
        {"name": "quant_rows", "op": "quant", "group": "row", "T": 16384, "D": 4096, "type": "bf16"},
        # what a weight gradient reads: groups run over the tokens, whose number is odd after packing
        {"name": "quant_cols_odd", "op": "quant", "group": "col", "T": 9377, "D": 2048, "type": "bf16"},
        # a few tokens in front of the first projection: latency
        {"name": "norm_few", "op": "norm", "T": 8, "D": 2048, "residual": False},
        # a training step's tokens, the block's branch added to the residual stream on the way
        {"name": "norm_step", "op": "norm", "T": 16384, "D": 4096, "residual": True},
        # a short prompt through a square projection: the weight's bytes and the launch
        {"name": "gemm_few", "op": "gemm", "form": "fwd", "T": 16, "N": 4096, "K": 4096, "add": False},
        # gate and up projections of a training step in one product
        {"name": "gemm_up", "op": "gemm", "form": "fwd", "T": 16384, "N": 28672, "K": 4096, "add": False},
        # a down projection added to the residual stream, an odd number of tokens
        {"name": "gemm_down_odd", "op": "gemm", "form": "fwd", "T": 3001, "N": 4096, "K": 14336, "add": True},
        # the input gradient of an up projection: the weight is read across its rows
        {"name": "gemm_dgrad", "op": "gemm", "form": "dgrad", "T": 8192, "N": 14336, "K": 4096, "add": False},
        # a weight gradient added to fp32 sums, the last block of tokens cut off
        {"name": "gemm_wgrad_odd", "op": "gemm", "form": "wgrad", "T": 9377, "N": 4096, "K": 2048, "add": True},
        # 64 experts' up projections, about 512 rows each, some none
        {"name": "grouped_up", "op": "grouped", "form": "fwd", "R": 32768, "E": 64, "N": 2048, "K": 2048},
        # their input gradients with 128 narrower experts
        {"name": "grouped_dgrad", "op": "grouped", "form": "dgrad", "R": 16384, "E": 128, "N": 768, "K": 2048},
        # their weight gradients; segments padded to 128 rows as the routing plan lays them out
        {"name": "grouped_wgrad", "op": "grouped", "form": "wgrad", "R": 32768, "E": 64, "N": 1024, "K": 2048},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["quant", "norm", "gemm", "gemm", "grouped"])
    if op == "quant":
        return {"op": op, "group": rng.choice(["row", "col", "block"]), "T": _log(rng, 1, 16384), "D": _log(rng, 40, 16384),
                "type": rng.choice(["bf16", "fp32"])}
    if op == "norm":
        return {"op": op, "T": _log(rng, 1, 32768), "D": _log(rng, 128, 8192), "residual": rng.random() < 0.5}
    if op == "gemm":
        form = rng.choice(["fwd", "fwd", "dgrad", "wgrad"])
        return {"op": op, "form": form, "T": _log(rng, 1, 16384), "N": _log(rng, 64, 14336), "K": _log(rng, 64, 14336),
                "add": form == "wgrad" or rng.random() < 0.3}
    return {"op": op, "form": rng.choice(["fwd", "dgrad", "wgrad"]), "R": _log(rng, 64, 32768), "E": _log(rng, 2, 128),
            "N": _log(rng, 128, 2048), "K": _log(rng, 128, 4096)}


# ------------------------------------------------------------------------------------------- inputs
def _ceil(a, b):
    return -(-a // b)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(g, T, D):
    """Normal, with a few channels ten to thirty times as large as the others, as hidden states have them."""
    x = torch.randn(T, D, device="cuda", generator=g)
    loud = torch.rand(D, device="cuda", generator=g) < 0.004
    return x * torch.where(loud, 10 + 20 * torch.rand(D, device="cuda", generator=g), 1.0)


def _gradients(g, T, D):
    """Small, of sizes that differ from token to token, none at all for an eighth of them (prompts that carry no loss)."""
    size = 1e-5 * torch.exp(1.5 * torch.randn(T, 1, device="cuda", generator=g))
    return torch.randn(T, D, device="cuda", generator=g) * size * (torch.rand(T, 1, device="cuda", generator=g) >= 0.125)


def _grid(q):
    """``q`` with rows that start on 16 bytes, as the operands of the products are kept."""
    *b, m, n = q.shape
    buf = torch.zeros(*b, m, _ceil(n, 16) * 16, dtype=torch.uint8, device="cuda")
    buf[..., :n] = q.view(torch.uint8)
    return buf.view(FP8)[..., :n]


def _groups(x, down, along):
    """Largest magnitude of each ``down x along`` group of the last two axes."""
    *b, m, n = x.shape
    M, N = _ceil(m, down), _ceil(n, along)
    x = torch.nn.functional.pad(x.abs(), (0, N * along - n, 0, M * down - m))
    return x.reshape(*b, M, down, N, along).amax((-3, -1))


SHAPES = {"row": (1, 128), "col": (128, 1), "block": (128, 128)}


def _spread(s, group, m, n):
    """Scales brought to the elements' shape."""
    down, along = SHAPES[group]
    if down > 1:
        s = s.repeat_interleave(down, -2)
    if along > 1:
        s = s.repeat_interleave(along, -1)
    return s[..., :m, :n]


def _quant(x, group):
    x = x.to(torch.float32)
    s = (_groups(x, *SHAPES[group]) / TOP).clamp(min=FLOOR)
    return (x * _spread(1.0 / s, group, x.shape[-2], x.shape[-1])).clamp(-TOP, TOP).to(FP8), s


def _operand(x, group):
    q, s = _quant(x, group)
    return _grid(q), s.mT.contiguous().mT if group == "row" else s    # a row's scales lie a row apart, as the quantiser leaves them


def _segments(case, g):
    """Row offsets of the experts: uneven, some empty; padded to 128 rows where the gradient's reduction runs over them."""
    E, R = case["E"], case["R"]
    p = torch.rand(E, device="cuda", generator=g) + 0.25
    p[torch.rand(E, device="cuda", generator=g) < 0.1] = 0
    p[0] = 1
    ends = torch.floor(torch.cumsum(p, 0).double() / p.sum().double() * R)
    ends[-1] = R
    counts = torch.diff(ends, prepend=ends.new_zeros(1))
    pad = 128 if case["form"] == "wgrad" else 1
    off = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    off[1:] = torch.cumsum((counts + pad - 1) // pad * pad, 0)
    return off, counts.to(torch.int64)


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    if op == "quant":
        make = {"row": _gradients, "col": _activations, "block": lambda g, m, n: 0.02 * torch.randn(m, n, device="cuda", generator=g)}
        x = make[case["group"]](g, case["T"], case["D"])
        return {"case": case, "x": x.to(torch.bfloat16) if case["type"] == "bf16" else x}
    if op == "norm":
        T, D = case["T"], case["D"]
        return {"case": case, "x": _activations(g, T, D).to(torch.bfloat16), "w": 1 + 0.2 * torch.randn(D, device="cuda", generator=g), "eps": 1e-5,
                "residual": 3 * torch.randn(T, D, device="cuda", generator=g).to(torch.bfloat16) if case["residual"] else None}
    form, N, K = case["form"], case["N"], case["K"]
    st = {"case": case}
    if op == "gemm":
        T = case["T"]
        if form == "wgrad":
            st["a"], st["sa"] = _operand(_gradients(g, T, N), "col")
            st["b"], st["sb"] = _operand(_activations(g, T, K), "col")
            shape = (N, K)
        else:
            st["a"], st["sa"] = _operand(_activations(g, T, K) if form == "fwd" else _gradients(g, T, N), "row")
            st["b"], st["sb"] = _operand(0.02 * torch.randn(N, K, device="cuda", generator=g), "block")
            shape = (T, N) if form == "fwd" else (T, K)
        st["c"] = None
        if case["add"]:
            c = torch.randn(*shape, device="cuda", generator=g)
            st["c"] = 1e-4 * c if form == "wgrad" else 1e-4 * c.to(torch.bfloat16) if form == "dgrad" else c.to(torch.bfloat16)
        return st
    st["off"], st["counts"] = _segments(case, g)
    R = int(st["off"][-1])
    st["most"] = int(torch.diff(st["off"]).max())
    if form == "wgrad":
        # rows that pad a segment are zero
        seg = torch.searchsorted(st["off"][1:].contiguous(), torch.arange(R, device="cuda", dtype=torch.int32), right=True)
        real = (torch.arange(R, device="cuda") - st["off"][seg] < st["counts"][seg]).unsqueeze(1)
        st["a"], st["sa"] = _operand(_gradients(g, R, N) * real, "col")
        st["b"], st["sb"] = _operand(_activations(g, R, K) * real, "col")
        st["c"] = 1e-4 * torch.randn(case["E"], N, K, device="cuda", generator=g)
    else:
        st["a"], st["sa"] = _operand(_activations(g, R, K) if form == "fwd" else _gradients(g, R, N), "row")
        st["b"], st["sb"] = _operand(0.02 * torch.randn(case["E"], N, K, device="cuda", generator=g), "block")
    return st


# ---------------------------------------------------------------------------------------- one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st):
    from flextrain_b200 import ops
    case = st["case"]
    op = case["op"]
    if op == "quant":
        m = ops.quant_fp8(st["x"], case["group"])
        return m.data, m.scale
    if op == "norm":
        m, rstd, h = ops.rmsnorm_fp8_fwd(st["x"], st["w"], st["eps"], residual=st["residual"])
        return (m.data, m.scale, rstd, h) if case["residual"] else (m.data, m.scale, rstd)
    form = case["form"]
    if op == "gemm":
        if form == "wgrad":
            a, b = ops.Fp8Matrix(st["a"], st["sa"], "col"), ops.Fp8Matrix(st["b"], st["sb"], "col")
            return ops.gemm_fp8(a, b, trans_a=True, beta=1.0 if case["add"] else 0.0, c=st["c"], out_dtype=torch.float32)
        a, b = ops.Fp8Matrix(st["a"], st["sa"], "row"), ops.Fp8Matrix(st["b"], st["sb"], "block")
        return ops.gemm_fp8(a, b, trans_b=form == "fwd", beta=1.0 if case["add"] else 0.0, c=st["c"])
    if form == "wgrad":
        a, b = ops.Fp8Matrix(st["a"], st["sa"], "col"), ops.Fp8Matrix(st["b"], st["sb"], "col")
        return ops.grouped_wgrad_fp8(a, b, st["off"], st["c"].clone(), pad=128)
    a, b = ops.Fp8Matrix(st["a"], st["sa"], "row"), ops.Fp8Matrix(st["b"], st["sb"], "block")
    return ops.grouped_gemm_fp8(a, b, st["off"], trans_w=form == "fwd")


def _value(q, s, group, dtype=torch.float32):
    return q.to(dtype) * _spread(s.to(dtype), group, q.shape[-2], q.shape[-1])


def _padded(x, off, most):
    """Rows of ragged segments as ``(E, most, n)``, zeros behind each segment, and the places they came from."""
    E, R = off.numel() - 1, x.shape[0]
    row = torch.arange(R, device=x.device)
    seg = torch.searchsorted(off[1:].contiguous(), row.to(off.dtype), right=True)
    at = seg * most + row - off[seg]
    return torch.zeros(E * most, x.shape[1], dtype=x.dtype, device=x.device).index_copy_(0, at, x).view(E, most, -1), at


def _run_plain(st):
    case = st["case"]
    op = case["op"]
    if op == "quant":
        return _quant(st["x"], case["group"])
    if op == "norm":
        h = st["x"]
        if case["residual"]:
            h = (h.to(torch.float32) + st["residual"].to(torch.float32)).to(torch.bfloat16)
        f = h.to(torch.float32)
        rstd = torch.rsqrt(f.square().mean(-1) + st["eps"])
        q, s = _quant(f * rstd.unsqueeze(-1) * st["w"], "row")
        return (q, s, rstd, h) if case["residual"] else (q, s, rstd)
    return _products(st, torch.float32)


def _products(st, dtype):
    case, form = st["case"], st["case"]["form"]
    group = ("col", "col") if form == "wgrad" else ("row", "block")
    a, b = _value(st["a"], st["sa"], group[0], dtype), _value(st["b"], st["sb"], group[1], dtype)
    if case["op"] == "gemm":
        y = a.mT @ b if form == "wgrad" else a @ b.mT if form == "fwd" else a @ b
        if case["add"]:
            y = y + st["c"].to(dtype)
        return y if dtype == torch.float64 else y.to(torch.float32 if form == "wgrad" else torch.bfloat16)
    pa, at = _padded(a, st["off"], st["most"])
    if form == "wgrad":
        return torch.bmm(pa.mT, _padded(b, st["off"], st["most"])[0]) + st["c"].to(dtype)
    y = torch.bmm(pa, b.mT if form == "fwd" else b).view(-1, b.shape[1] if form == "fwd" else b.shape[2])[at]
    return y if dtype == torch.float64 else y.to(torch.bfloat16)


# ------------------------------------------------------------------------------ 64 bits, written apart
def _e4m3_64(v):
    """Nearest e4m3 value (ties to the even one) of a double: steps of 2^(e-3), of 2^-9 below 2^-6."""
    _, e = torch.frexp(v)
    step = torch.exp2((e - 1).clamp(min=-6).to(torch.float64) - 3)
    return (torch.round(v / step) * step).clamp(-TOP, TOP)


def _quant_64(x, group):
    """Group by group in place of the padded view of the plain form: running maxima through an index of groups."""
    m, n = x.shape
    down, along = SHAPES[group]
    ri = torch.arange(m, device=x.device) // down
    ci = torch.arange(n, device=x.device) // along
    by_row = torch.zeros(_ceil(m, down), n, dtype=x.dtype, device=x.device).index_reduce_(0, ri, x.abs(), "amax")
    top = torch.zeros(by_row.shape[0], _ceil(n, along), dtype=x.dtype, device=x.device).index_reduce_(1, ci, by_row, "amax")
    s = torch.maximum(top / TOP, torch.full_like(top, FLOOR))
    return _e4m3_64(x / s[ri][:, ci]), s


def exact(case, seed):
    st, op = prepare(case, seed), case["op"]
    if op == "quant":
        return _quant_64(st["x"].double(), case["group"])
    if op == "norm":
        h = st["x"].double()
        if case["residual"]:
            # h is kept in 16 bits, and the norm is of what is kept
            h = (h + st["residual"].double()).to(torch.bfloat16).double()
        rstd = 1.0 / torch.sqrt((h * h).sum(-1) / case["D"] + st["eps"])
        q, s = _quant_64(h * rstd[:, None] * st["w"].double(), "row")
        return (q, s, rstd, h) if case["residual"] else (q, s, rstd)
    form = case["form"]
    a, b = st["a"].double(), st["b"].double()
    # the scales by the index of each element's group, the product by blocks of its output's columns
    rows = lambda s: s.double()[..., torch.arange(a.shape[1], device="cuda") // 128]                                    # noqa: E731
    cols = lambda s, t: s.double()[torch.arange(t.shape[0], device="cuda") // 128]                                      # noqa: E731
    if form == "wgrad":
        a, b = a * cols(st["sa"], a), b * cols(st["sb"], b)
        if op == "gemm":
            return torch.einsum("tn,tk->nk", a, b) + (st["c"].double() if case["add"] else 0)
        off = st["off"].tolist()
        return torch.stack([a[i:j].t() @ b[i:j] for i, j in zip(off, off[1:])]) + st["c"].double()
    a = a * rows(st["sa"])
    iN = torch.arange(b.shape[-2], device="cuda") // 128
    iK = torch.arange(b.shape[-1], device="cuda") // 128
    b = b * st["sb"].double()[..., iN, :][..., iK]
    if op == "gemm":
        y = torch.einsum("tk,nk->tn" if form == "fwd" else "tn,nk->tk", a, b)
        return y + st["c"].double() if case["add"] else y
    off = st["off"].tolist()
    return torch.cat([a[i:j] @ (w.t() if form == "fwd" else w) for i, j, w in zip(off, off[1:], b)])


# --------------------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "quant":
        n = case["T"] * case["D"]
        down, along = SHAPES[case["group"]]
        return {"bytes": n * (2 if case["type"] == "bf16" else 4) + n + 4 * _ceil(case["T"], down) * _ceil(case["D"], along), "flops": 3 * n}
    if op == "norm":
        n, T = case["T"] * case["D"], case["T"]
        return {"bytes": n * (7 if case["residual"] else 3) + 4 * T * (_ceil(case["D"], 128) + 1) + 4 * case["D"], "flops": 8 * n}
    form, N, K = case["form"], case["N"], case["K"]
    T, E = (case["T"], 1) if op == "gemm" else (case["R"], case["E"])
    if form == "wgrad":
        read = T * (N + K) + 4 * _ceil(T, 128) * (N + K)
        out = E * N * K * (8 if op == "grouped" or case["add"] else 4)
    else:
        red, wide = (K, N) if form == "fwd" else (N, K)
        read = T * red + 4 * T * _ceil(red, 128) + E * (N * K + 4 * _ceil(N, 128) * _ceil(K, 128))
        out = T * wide * (4 if op == "gemm" and case["add"] else 2)
    return {"bytes": read + out, "flops": 2 * T * N * K}
