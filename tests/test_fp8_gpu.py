"""Linear layers in 8 bits on the GPU against plain implementations in 64 bits.

Roundings counted in the tolerances: e4m3 half a step, 2^-4 of the value, or 2^-10 of the scale below the smallest normal value;
bf16 2^-8; an fp32 operation 2^-24.  A product of a block of 128 may be off by 128 * 2^-23 of the sum of its terms' magnitudes,
whatever the order of its additions, and the blocks' sums by another 2^-24 for each block, scale and epilogue operation."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _ops():
    from flextrain_b200 import ops
    return ops


def _no_errors():
    from flextrain_b200.ops import cuda as k
    torch.cuda.synchronize()
    assert k.device_error_words().get("gemm_fp8", 0) == 0


def _spread(m, dtype=torch.float64):
    down, along = {"row": (1, 128), "col": (128, 1), "block": (128, 128)}[m.group]
    i = torch.arange(m.data.shape[-2], device=m.data.device) // down
    j = torch.arange(m.data.shape[-1], device=m.data.device) // along
    return m.scale.to(dtype)[..., i, :][..., j]


def _value(m):
    return m.data.double() * _spread(m)


def _bits(q):
    return q.contiguous().view(torch.uint8)


# --------------------------------------------------------------------------------------- quantisers
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group", ["row", "col", "block"])
@pytest.mark.parametrize("M,N", [(1, 1), (1, 128), (3, 127), (128, 128), (129, 130), (257, 1000), (640, 264), (1000, 40)])
def test_quant(dtype, group, M, N):
    ops = _ops()
    torch.manual_seed(M * 1000 + N)
    x = (torch.randn(M, N, device=DEV) * torch.exp(2 * torch.randn(M, 1, device=DEV))).to(dtype)
    x[torch.rand(M, device=DEV) < 0.2] = 0                       # whole rows of zeros: groups whose scale is the floor
    m = ops.quant_fp8(x, group)
    q, s = ops.ref.quant_fp8(x.cpu(), group)                     # the same fp32 operations
    assert m.data.shape == x.shape and m.group == group
    assert torch.equal(m.scale.cpu(), s) and torch.equal(_bits(m.data).cpu(), _bits(q))
    step = torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * _spread(m))
    assert torch.all((_value(m) - x.double()).abs() <= step * (1 + 2.0 ** -20))


@pytest.mark.parametrize("group", ["row", "col", "block"])
def test_quant_views_and_far_offsets(group):
    """Rows that lie apart, that start off 16 bytes, columns that lie apart, and elements behind 2^31."""
    ops = _ops()
    torch.manual_seed(0)
    base = torch.randn(300, 700, device=DEV).bfloat16()
    for x in (base[:, 8:520], base[5:, 3:400], base[::2, 1:301], base.t(), base[:, ::3]):
        m = ops.quant_fp8(x, group)
        q, s = ops.ref.quant_fp8(x.cpu(), group)
        assert torch.equal(m.scale.cpu(), s) and torch.equal(_bits(m.data).cpu(), _bits(q))
    wide = torch.zeros(3, 1 << 30, dtype=torch.bfloat16, device=DEV)[:, :200]
    wide.normal_()
    m = ops.quant_fp8(wide, group)
    q, s = ops.ref.quant_fp8(wide.cpu(), group)
    assert torch.equal(m.scale.cpu(), s) and torch.equal(_bits(m.data).cpu(), _bits(q))


def test_quant_stack():
    ops = _ops()
    torch.manual_seed(0)
    w = torch.randn(5, 200, 300, device=DEV).bfloat16()
    for x in (w, w[1::2], w[:, :130, 8:]):
        m = ops.quant_fp8(x, "block")
        for e in range(x.shape[0]):
            q, s = ops.ref.quant_fp8(x[e].cpu(), "block")
            assert torch.equal(m.scale[e].cpu(), s) and torch.equal(_bits(m.data[e]).cpu(), _bits(q))


@pytest.mark.parametrize("group", ["row", "col", "block"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quant_values_at_the_edges(group, dtype):
    """NaN and infinities stay in their groups, denormals count, the largest and smallest numbers come back."""
    ops = _ops()
    fi = torch.finfo(dtype)
    x = torch.ones(256, 256, device=DEV, dtype=dtype)
    x[3, 7], x[130, 200], x[5, 140] = float("nan"), float("inf"), float("-inf")
    x[200:, :100] = fi.tiny / 4                                  # denormal
    x[129, 3], x[140, 5] = fi.max, -fi.max
    m = ops.quant_fp8(x, group)
    q, s = ops.ref.quant_fp8(x.cpu(), group)
    assert torch.equal(torch.isnan(m.scale.cpu()), torch.isnan(s))
    assert torch.equal(m.scale.cpu().nan_to_num(7), s.nan_to_num(7))
    got, want = ops.dequant_fp8(m, torch.float32).cpu(), ops.ref.dequant_fp8(q, s, group)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(7), want.nan_to_num(7))
    bad = ~torch.isfinite(x.cpu())
    down, along = {"row": (1, 128), "col": (128, 1), "block": (128, 128)}[group]
    hit = bad.view(256 // down, down, 256 // along, along).any(3).any(1)
    assert torch.equal(torch.isnan(got), hit.repeat_interleave(down, 0).repeat_interleave(along, 1))


# --------------------------------------------------------------------------------------------- norm
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("gain", [True, False])
@pytest.mark.parametrize("T,D", [(1, 128), (1, 2048), (5, 1), (7, 130), (33, 1000), (3, 1024), (9, 2056), (20, 4096), (6, 5120), (4, 8192),
                                 (3, 8200), (2, 20001)])
def test_rmsnorm(residual, gain, T, D):
    ops = _ops()
    torch.manual_seed(T * 100000 + D)
    x = torch.randn(T, D, device=DEV).bfloat16()
    r = 3 * torch.randn(T, D, device=DEV).bfloat16() if residual else None
    w = 1 + 0.3 * torch.randn(D, device=DEV) if gain else None
    m, rstd, h = ops.rmsnorm_fp8_fwd(x, w, 1e-5, residual=r)
    want_h = x if r is None else (x.float() + r.float()).bfloat16()
    assert torch.equal(h, want_h) and (residual or h is x)
    hd = want_h.double()
    r64 = 1 / torch.sqrt((hd * hd).mean(-1) + 1e-5)
    # a thread adds D / 128 squares at most, then 8 + 8 partial sums, all positive; half of that in the root, and its own 2^-22
    off = (D / 128 + 20) * 2.0 ** -25 + 2.0 ** -22
    assert torch.all((rstd.double() - r64).abs() <= off * r64)
    y = hd * r64[:, None] * (1 if w is None else w.double())
    assert m.scale.shape == (T, -(-D // 128))
    top = torch.nn.functional.pad(y.abs(), (0, -D % 128)).view(T, -1, 128).amax(-1)
    s64 = (top / 448).clamp(min=2.0 ** -126)
    assert torch.all((m.scale.double() - s64).abs() <= (off + 2.0 ** -21) * s64)
    step = torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * _spread(m)) + 2 * (off + 2.0 ** -21) * y.abs()
    assert torch.all((_value(m) - y).abs() <= step)


def test_rmsnorm_views_and_rows_of_nothing():
    ops = _ops()
    torch.manual_seed(0)
    wide, res = torch.randn(40, 700, device=DEV).bfloat16(), torch.randn(40, 512, device=DEV).bfloat16()
    wide[3] = 0
    wide[5, 60] = float("nan")
    res[3] = 0
    w = torch.rand(512, device=DEV) + 0.5
    for x, r in ((wide[:, 8:520], res), (wide[:, 3:515], res), (wide[:, 100:612], None)):
        m, rstd, h = ops.rmsnorm_fp8_fwd(x, w, 1e-6, residual=r)
        m2, rstd2, h2 = ops.rmsnorm_fp8_fwd(x.contiguous(), w, 1e-6, residual=r)
        assert torch.equal(_bits(m.data), _bits(m2.data)) and torch.equal(m.scale.nan_to_num(7), m2.scale.nan_to_num(7))
        nan = torch.isnan(ops.dequant_fp8(m, torch.float32)).all(1)
        assert nan.sum() == int(torch.isnan(x[5]).any()) and torch.isfinite(rstd[torch.arange(40, device=DEV) != 5]).all()
        if r is not None:
            assert torch.all(m.data[3].float() == 0) and torch.all(m.scale[3] == 2.0 ** -126)


# ----------------------------------------------------------------------------------------- products
def _room(want, mag, K, dtype, extra=0):
    return ((2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24) * want.abs()
            + ((128 * 2 + (K + 127) // 128 + 6) * 2.0 ** -24) * mag + extra)


def _operands(form, M, N, K, scale_a=1.0):
    ops = _ops()
    a = scale_a * torch.randn(M, K, device=DEV) * torch.exp(torch.randn(M, 1, device=DEV))
    b = 0.1 * torch.randn(N, K, device=DEV)
    if form == "fwd":
        A, B = ops.quant_fp8(a, "row"), ops.quant_fp8(b, "block")
    elif form == "rows":
        A, B = ops.quant_fp8(a, "row"), ops.quant_fp8(b, "row")
    elif form == "blocks":
        A, B = ops.quant_fp8(a, "block"), ops.quant_fp8(b, "block")
    elif form == "dgrad":
        A, B = ops.quant_fp8(a, "row"), ops.quant_fp8(b.t().contiguous(), "block")
    elif form == "wgrad_block":
        A, B = ops.quant_fp8(a.t().contiguous(), "col"), ops.quant_fp8(b.t().contiguous(), "block")
    elif form == "wgrad":
        A, B = ops.quant_fp8(a.t().contiguous(), "col"), ops.quant_fp8(b.t().contiguous(), "col")
    else:                                                        # a read across, b along
        A, B = ops.quant_fp8(a.t().contiguous(), "col"), ops.quant_fp8(b, "row")
    ta, tb = form in ("wgrad", "wgrad_block", "across"), form not in ("dgrad", "wgrad", "wgrad_block")
    va, vb = _value(A), _value(B)
    va, vb = va.t() if ta else va, vb.t() if tb else vb
    return A, B, ta, tb, va @ vb, va.abs() @ vb.abs()


SIZES = [(1, 128, 128), (16, 256, 512), (128, 128, 128), (130, 257, 100), (3, 40, 1000), (300, 520, 129), (1, 1, 1), (513, 600, 16),
         (640, 512, 640), (1025, 776, 200), (200, 4096, 384), (777, 1031, 2049), (5, 300, 5000), (100, 133, 2100), (128, 1000, 1500)]


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("form", ["fwd", "rows", "blocks", "dgrad", "wgrad", "wgrad_block", "across"])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_gemm(out_dtype, form, M, N, K):
    """Plain, with bias and alpha, with a C of other strides, into a strided result whose neighbours stay as they are."""
    ops = _ops()
    torch.manual_seed(M + N + K)
    A, B, ta, tb, want, mag = _operands(form, M, N, K)
    kw = dict(trans_a=ta, trans_b=tb)
    got = ops.gemm_fp8(A, B, out_dtype=out_dtype, **kw)
    assert got.dtype == out_dtype and torch.all((got.double() - want).abs() <= _room(want, mag, K, out_dtype))
    assert torch.equal(got, ops.gemm_fp8(A, B, out_dtype=out_dtype, **kw))
    bias = torch.randn(N, device=DEV)
    got = ops.gemm_fp8(A, B, out_dtype=out_dtype, alpha=0.5, bias=bias, **kw)
    w2 = 0.5 * want + bias.double()
    assert torch.all((got.double() - w2).abs() <= _room(w2, 0.5 * mag + bias.abs().double(), K, out_dtype))
    wide = torch.randn(M, N + 24, device=DEV).to(out_dtype)
    keep = wide.clone()
    ops.gemm_fp8(A, B, out=wide[:, 8:8 + N], beta=1.0, **kw)
    w3 = want + keep[:, 8:8 + N].double()
    assert torch.all((wide[:, 8:8 + N].double() - w3).abs() <= _room(w3, mag + keep[:, 8:8 + N].abs().double(), K, out_dtype))
    assert torch.equal(wide[:, :8], keep[:, :8]) and torch.equal(wide[:, 8 + N:], keep[:, 8 + N:])
    c = torch.randn(M, N + 3, device=DEV).to(out_dtype)[:, 3:]
    got = ops.gemm_fp8(A, B, c=c, beta=-2.0, out_dtype=out_dtype, **kw)
    w4 = want - 2.0 * c.double()
    assert torch.all((got.double() - w4).abs() <= _room(w4, mag + 2 * c.abs().double(), K, out_dtype))
    _no_errors()


@pytest.fixture(params=[0, 1, 2, 3])
def tile(request, monkeypatch):
    """The products' tile: by size, 128 x 128, 128 x 256, 256 x 256 on two SMs."""
    from flextrain_b200.ops import fp8
    monkeypatch.setattr(fp8, "TILE", request.param)
    return request.param


@pytest.mark.parametrize("form", ["fwd", "rows", "dgrad", "wgrad", "across"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (130, 257, 300), (257, 129, 640), (300, 520, 130), (600, 1100, 1000)])
def test_gemm_tiles(tile, form, M, N, K):
    """Every tile at sizes that end inside it, into both types, with C in place, elsewhere and not at all."""
    ops = _ops()
    torch.manual_seed(M + N + K)
    A, B, ta, tb, want, mag = _operands(form, M, N, K)
    for dtype in (torch.bfloat16, torch.float32):
        got = ops.gemm_fp8(A, B, trans_a=ta, trans_b=tb, out_dtype=dtype)
        assert torch.all((got.double() - want).abs() <= _room(want, mag, K, dtype))
        Np = (N + 7) // 8 * 8                                    # rows on 16 bytes, and rows that are not
        for c in (torch.randn(M, Np, device=DEV).to(dtype)[:, :N], torch.randn(M, N, device=DEV).to(dtype)):
            w2, m2 = want + c.double(), mag + c.abs().double()
            got = ops.gemm_fp8(A, B, trans_a=ta, trans_b=tb, beta=1.0, c=c, out_dtype=dtype)
            assert torch.all((got.double() - w2).abs() <= _room(w2, m2, K, dtype))
            ops.gemm_fp8(A, B, trans_a=ta, trans_b=tb, beta=1.0, out=c)
            assert torch.all((c.double() - w2).abs() <= _room(w2, m2, K, dtype))
    _no_errors()


@pytest.mark.parametrize("N,K", [(520, 136), (129, 1030)])
def test_grouped_tiles(tile, N, K):
    ops = _ops()
    torch.manual_seed(0)
    cnt = [3, 0, 129, 1, 300, 0, 255, 128]
    off = torch.tensor([0] + torch.tensor(cnt).cumsum(0).tolist(), device=DEV, dtype=torch.int32)
    used, E = sum(cnt), len(cnt)
    X, W = ops.quant_fp8(torch.randn(used, K, device=DEV), "row"), ops.quant_fp8(torch.randn(E, N, K, device=DEV), "block")
    vx, vw, o = _value(X), _value(W), off.tolist()
    for dtype in (torch.bfloat16, torch.float32):
        out = torch.full((used + 5, N), 7.0, device=DEV, dtype=dtype)
        ops.grouped_gemm_fp8(X, W, off, out=out[:used])
        for e in range(E):
            want, mag = vx[o[e]:o[e + 1]] @ vw[e].t(), vx[o[e]:o[e + 1]].abs() @ vw[e].abs().t()
            assert torch.all((out[o[e]:o[e + 1]].double() - want).abs() <= _room(want, mag, K, dtype))
        assert torch.all(out[used:] == 7)
    cnt = [128, 0, 384, 256]
    off = torch.tensor([0] + torch.tensor(cnt).cumsum(0).tolist(), device=DEV, dtype=torch.int32)
    D, X = ops.quant_fp8(torch.randn(768, N, device=DEV), "col"), ops.quant_fp8(torch.randn(768, K, device=DEV), "col")
    vd, vx, o = _value(D), _value(X), off.tolist()
    for dtype in (torch.bfloat16, torch.float32):
        gw = torch.randn(4, N, K, device=DEV).to(dtype)
        keep = gw.clone()
        ops.grouped_wgrad_fp8(D, X, off, gw, pad=128)
        for e in range(4):
            want = keep[e].double() + vd[o[e]:o[e + 1]].t() @ vx[o[e]:o[e + 1]]
            mag = keep[e].abs().double() + vd[o[e]:o[e + 1]].abs().t() @ vx[o[e]:o[e + 1]].abs()
            assert torch.all((gw[e].double() - want).abs() <= _room(want, mag, 768, dtype))
    _no_errors()


@pytest.mark.parametrize("form", ["fwd", "dgrad", "wgrad"])
def test_gemm_infinities_stay_in_their_rows(tile, form):
    """A row or column of NaN reaches the results that it is part of and no others; C is not read without beta."""
    ops = _ops()
    torch.manual_seed(0)
    M, N, K = 260, 700, 300
    a, b = torch.randn(M, K, device=DEV), torch.randn(N, K, device=DEV)
    a[M // 2, K - 1] = float("inf")
    a[0, 0] = float("nan")
    if form == "wgrad":
        b[N - 1, 3] = float("nan")
    ga, gb = ("col", "col") if form == "wgrad" else ("row", "block")
    A = ops.quant_fp8(a.t().contiguous() if form == "wgrad" else a, ga)
    B = ops.quant_fp8(b if form == "fwd" else b.t().contiguous(), gb)
    out = torch.full((M, N), float("nan"), device=DEV)
    y = ops.gemm_fp8(A, B, trans_a=form == "wgrad", trans_b=form == "fwd", out=out)
    bad = torch.zeros(M, N, dtype=torch.bool, device=DEV)
    bad[0], bad[M // 2] = True, True
    if form == "wgrad":
        bad[:, N - 1] = True
    assert torch.equal(~torch.isfinite(y), bad)
    _no_errors()


def test_gemm_operands_off_the_grid():
    """Data whose rows or base lie off 16 bytes is copied; scales of any strides are read where they lie."""
    ops = _ops()
    torch.manual_seed(0)
    A, B = ops.quant_fp8(torch.randn(70, 300, device=DEV), "row"), ops.quant_fp8(torch.randn(200, 300, device=DEV), "block")
    want = ops.linear_fp8_fwd(A, B)
    u = lambda q: q.view(torch.uint8)
    odd = torch.zeros(70, 333, dtype=torch.uint8, device=DEV)
    odd[:, 5:305] = u(A.data)
    shifted = torch.zeros(200 * 301 + 1, dtype=torch.uint8, device=DEV)[1:].view(200, 301)
    shifted[:, :300] = u(B.data)
    sa = torch.zeros(70, 9, device=DEV)[:, 1:9:3]
    sa.copy_(A.scale)
    sb = torch.zeros(3, 5, device=DEV)[:, 1:3].t()
    sb.copy_(B.scale)
    f8 = torch.float8_e4m3fn
    got = ops.linear_fp8_fwd(ops.Fp8Matrix(odd.view(f8)[:, 5:305], sa, "row"), ops.Fp8Matrix(shifted.view(f8)[:, :300], sb, "block"))
    assert torch.equal(got, want)
    turned = ops.Fp8Matrix(u(A.data).t().contiguous().t().view(f8), A.scale, "row")
    assert torch.equal(ops.linear_fp8_fwd(turned, B), want)


# ------------------------------------------------------------------------------------------ experts
COUNTS = {"even": [256] * 4, "ragged": [3, 0, 129, 1, 700, 0, 255], "one": [0, 0, 513, 0], "none": [0, 0], "single": [1]}


@pytest.mark.parametrize("counts", list(COUNTS))
@pytest.mark.parametrize("trans_w", [True, False])
@pytest.mark.parametrize("N,K", [(128, 128), (520, 136), (300, 1030), (768, 256)])
def test_grouped_gemm(counts, trans_w, N, K):
    ops = _ops()
    torch.manual_seed(N + K)
    cnt = COUNTS[counts]
    E, used = len(cnt), sum(cnt)
    off = torch.tensor([0] + torch.tensor(cnt).cumsum(0).tolist(), device=DEV, dtype=torch.int32)
    x = torch.randn(used + 130, K, device=DEV)
    x[used:] = float("nan")
    X = ops.quant_fp8(x, "row")
    w = 0.1 * torch.randn(E, N, K, device=DEV)
    W = ops.quant_fp8(w if trans_w else w.mT.contiguous(), "block")
    vx, vw = _value(X), _value(W)
    vw = vw if trans_w else vw.mT
    seg = torch.cat([torch.full((c,), e) for e, c in enumerate(cnt)] + [torch.zeros(0)]).long().to(DEV)
    want = torch.cat([vx[o:o + c] @ vw[e].t() for e, (o, c) in enumerate(zip(off.tolist(), cnt))])
    mag = torch.cat([vx[o:o + c].abs() @ vw[e].abs().t() for e, (o, c) in enumerate(zip(off.tolist(), cnt))])
    assert seg.numel() == used
    for dtype in (torch.bfloat16, torch.float32):
        wide = torch.randn(used + 130, N + 10, device=DEV).to(dtype)
        for out in (wide[:, :N], torch.randn(used + 130, N, device=DEV).to(dtype)):
            keep = out.clone()
            ops.grouped_gemm_fp8(X, W, off, trans_w=trans_w, out=out, alpha=2.0)
            assert torch.all((out[:used].double() - 2 * want).abs() <= _room(2 * want, 2 * mag, K, dtype))
            assert torch.equal(out[used:], keep[used:])
            before = out.clone()
            ops.grouped_gemm_fp8(X, W, off.long(), trans_w=trans_w, out=out, beta=1.0)
            w2 = want + before[:used].double()
            assert torch.all((out[:used].double() - w2).abs() <= _room(w2, mag + before[:used].abs().double(), K, dtype))
            assert torch.equal(out[used:], keep[used:])
    y = ops.grouped_gemm_fp8(X, W, off, trans_w=trans_w)
    assert y.shape == (used + 130, N) and torch.all((y[:used].double() - want).abs() <= _room(want, mag, K, torch.bfloat16))
    _no_errors()


@pytest.mark.parametrize("group", ["col", "block"])
@pytest.mark.parametrize("counts", [[128, 256, 0, 384], [0, 128, 0], [1280, 128], [128] * 9])
@pytest.mark.parametrize("N,K", [(128, 128), (520, 136), (300, 1030), (768, 512)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_grouped_wgrad(counts, N, K, dtype, group):
    ops = _ops()
    torch.manual_seed(N + K)
    E, used = len(counts), sum(counts)
    off = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), device=DEV, dtype=torch.int32)
    dy, x = torch.randn(used + 128, N, device=DEV), torch.randn(used + 128, K, device=DEV)
    dy[used:] = float("nan")
    x[5] = 0
    DY, X = ops.quant_fp8(dy, "col"), ops.quant_fp8(x, group)
    vd, vx = _value(DY), _value(X)
    gw = torch.randn(E, N, K, device=DEV).to(dtype)
    keep = gw.clone()
    assert ops.grouped_wgrad_fp8(DY, X, off, gw, alpha=0.5, pad=128) is gw
    for e in range(E):
        i, j = int(off[e]), int(off[e + 1])
        if i == j:
            assert torch.equal(gw[e], keep[e])
            continue
        want = 0.5 * vd[i:j].t() @ vx[i:j] + keep[e].double()
        mag = 0.5 * vd[i:j].abs().t() @ vx[i:j].abs() + keep[e].abs().double()
        assert torch.all((gw[e].double() - want).abs() <= _room(want, mag, j - i, dtype))
    _no_errors()


def test_offsets_that_are_none():
    """Offsets that descend, that lie outside of the rows or inside a group of 128: nothing outside is read or written, and the last
    are reported."""
    ops = _ops()
    from flextrain_b200.ops import cuda as k
    torch.manual_seed(0)
    X, W = ops.quant_fp8(torch.randn(300, 256, device=DEV), "row"), ops.quant_fp8(torch.randn(3, 200, 256, device=DEV), "block")
    room = torch.full((900, 200), 7.0, device=DEV, dtype=torch.bfloat16)
    for off in ([-50, 100, 90, 5000], [0, 1 << 30, 0, -1], [300, 300, 300, 300], [400, 500, 600, 700]):
        ops.grouped_gemm_fp8(X, W, torch.tensor(off, device=DEV, dtype=torch.int32), out=room[300:600])
        torch.cuda.synchronize()
        assert torch.all(room[:300] == 7) and torch.all(room[600:] == 7)
    assert k.device_error_words().get("gemm_fp8", 0) == 0
    D, X = ops.quant_fp8(torch.randn(300, 200, device=DEV), "col"), ops.quant_fp8(torch.randn(300, 256, device=DEV), "col")
    gw = torch.zeros(5, 200, 256, device=DEV)
    ops.grouped_wgrad_fp8(D, X, torch.tensor([-3, 128, 1000], device=DEV, dtype=torch.int32), gw[1:3], pad=128)
    torch.cuda.synchronize()
    assert torch.all(gw[0] == 0) and torch.all(gw[3:] == 0)
    k.device_error_words()
    for off in ([0, 100, 300], [0, 128, 200], [0, 200, 200]):
        ops.grouped_wgrad_fp8(D, X, torch.tensor(off, device=DEV, dtype=torch.int32), gw[1:3], pad=128)
        torch.cuda.synchronize()
        assert k.device_error_words()["gemm_fp8"] == 3040 and k.device_error_words()["gemm_fp8"] == 0
    for off in ([0, 128, 300], [0, 300, 300], [0, 0, 256]):            # (the rows end where the data does, or on a multiple)
        ops.grouped_wgrad_fp8(D, X, torch.tensor(off, device=DEV, dtype=torch.int32), gw[1:3], pad=128)
        torch.cuda.synchronize()
        assert k.device_error_words()["gemm_fp8"] == 0


def test_gemm_in_place_and_expanded():
    """C that is the result itself or one row for all, results of a single row with any stride, NaN in what is not read."""
    ops = _ops()
    torch.manual_seed(0)
    A, B = ops.quant_fp8(torch.randn(300, 200, device=DEV), "row"), ops.quant_fp8(torch.randn(264, 200, device=DEV), "block")
    want = ops.linear_fp8_fwd(A, B, out_dtype=torch.float32)
    row = torch.randn(1, 264, device=DEV)
    assert torch.equal(ops.gemm_fp8(A, B, trans_b=True, beta=1.0, c=row.expand(300, 264), out_dtype=torch.float32), want + row)
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.randn(300, 264, device=DEV).to(dtype)
        keep = out.clone()
        ops.gemm_fp8(A, B, trans_b=True, beta=1.0, c=out, out=out)
        assert torch.equal(out, (want + keep.float()).to(dtype))
    one = ops.Fp8Matrix(A.data[:1], A.scale[:1], "row")
    for out in (torch.empty(264, 1, device=DEV).t(), torch.empty(1, 264, device=DEV).expand(1, 264), torch.empty(1, 270, device=DEV)[:, 3:267]):
        assert torch.equal(ops.linear_fp8_fwd(one, B, out=out), want[:1])
    none = torch.full((300, 264), float("nan"), device=DEV)
    assert torch.equal(ops.gemm_fp8(A, B, trans_b=True, c=none, out=none), want)


def _far(t, ld):
    """``t`` with its rows ``ld`` elements apart."""
    out = torch.empty_strided(t.shape, (ld, 1), dtype=t.dtype, device=DEV)
    out.copy_(t) if t.dtype != torch.float8_e4m3fn else out.view(torch.uint8).copy_(t.view(torch.uint8))
    return out


@pytest.mark.parametrize("tile", [0, 1, 2, 3])
@pytest.mark.parametrize("dtype,N", [(torch.bfloat16, 264), (torch.float32, 264), (torch.float32, 261)])
def test_gemm_rows_far_apart(monkeypatch, tile, dtype, N):
    """Operands and results whose rows begin beyond 2^31 elements: the same bits as where they lie together."""
    from flextrain_b200.ops import fp8
    ops = _ops()
    monkeypatch.setattr(fp8, "TILE", tile)
    torch.manual_seed(N)
    A, B = ops.quant_fp8(torch.randn(300, 200, device=DEV), "row"), ops.quant_fp8(torch.randn(N, 200, device=DEV), "block")
    at, bt = ops.quant_fp8(torch.randn(200, 300, device=DEV), "col"), ops.quant_fp8(torch.randn(200, N, device=DEV), "block")
    c = torch.randn(300, N, device=DEV).to(dtype)
    for a, b, ta, tb in ((A, B, False, True), (at, bt, True, False)):
        want = ops.gemm_fp8(a, b, trans_a=ta, trans_b=tb, beta=1.0, c=c, out_dtype=dtype)
        far_a, far_b = (m._replace(data=_far(m.data, 1 << 24)) for m in (a, b))
        for out in (_far(c, (1 << 23) + 8), c.clone()):
            got = ops.gemm_fp8(far_a, far_b, trans_a=ta, trans_b=tb, beta=1.0, out=out)
            assert torch.equal(got, want)
        assert torch.equal(ops.gemm_fp8(a, b, trans_a=ta, trans_b=tb, beta=1.0, c=_far(c, (1 << 23) + 8), out_dtype=dtype), want)
    _no_errors()


# --------------------------------------------------------------------------------- together, as used
def _layer(ops, x, res, gain, w, dy):
    """Norm, projection and their backward pass as a training step runs them: everything that it hands on."""
    h8, rstd, h = ops.rmsnorm_fp8_fwd(x, gain, 1e-5, residual=res)
    w8 = ops.quant_fp8(w, "block")
    y = ops.linear_fp8_fwd(h8, w8)
    dh = ops.linear_fp8_dgrad(ops.quant_fp8(dy, "row"), w8)
    dgain = torch.zeros_like(gain)
    dx, n = ops.rmsnorm_bwd(dh, h, gain, rstd, dx_add=res, emit_y=True, dw_out=dgain)
    dw = torch.zeros(w.shape, device=w.device)
    ops.linear_fp8_wgrad(ops.quant_fp8(dy, "col"), ops.quant_fp8(n, "col"), dw)
    return y, dx, dw, dgain


def _layer_inputs(T, D, N):
    torch.manual_seed(T + D + N)
    x, res = torch.randn(T, D, device=DEV).bfloat16(), torch.randn(T, D, device=DEV).bfloat16()
    return x, res, 1 + 0.2 * torch.randn(D, device=DEV), 0.05 * torch.randn(N, D, device=DEV).bfloat16(), torch.randn(T, N, device=DEV).bfloat16()


@pytest.mark.parametrize("T,D,N", [(1, 256, 512), (130, 384, 640), (1000, 1024, 768)])
def test_layer(T, D, N):
    """A run of them together against the formulas in 64 bits: each output's error, in the 2-norm, is that of its operands' 8 bits.
    A rounding to e4m3 is off by at most 2^-4 of its value (2^-10 of the scale, below 2^-17 of the group's largest, adds under 2^-10
    of a group's norm), so a product of two such operands by at most (2 * 2^-4 + 2^-8 + 2^-7) of |A| |B|, in norm."""
    ops = _ops()
    x, res, gain, w, dy = _layer_inputs(T, D, N)
    got = _layer(ops, x, res, gain, w, dy)
    h = (x.float() + res.float()).bfloat16().double()
    r = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-5)
    n, W, g = h * r * gain.double(), w.double(), dy.double()
    dh = g @ W
    dn = dh * gain.double()
    dx = r * dn - h * r ** 3 * (dn * h).mean(-1, keepdim=True) + res.double()
    want = (n @ W.t(), dx, g.t() @ n, (dh * h * r).sum(0))
    # the sizes that the errors go by: |A| |B| row by row, carried through the norm's backward pass by its largest factor
    dh_mag = g.abs() @ W.abs()
    mags = (n.abs() @ W.abs().t(),
            r * (dh_mag * gain.double().abs() + (h * r).abs() * ((dh_mag * gain.double().abs()) * (h * r).abs()).mean(-1, keepdim=True))
            + res.double().abs(), g.abs().t() @ n.abs(), (dh_mag * (h * r).abs()).sum(0))
    for a, b, mag in zip(got, want, mags):
        assert a.shape == b.shape and torch.all((a.double() - b).abs() <= (2 * 2.0 ** -4 + 2.0 ** -8 + 2.0 ** -7 + 2.0 ** -8) * mag + 1e-6)


def test_layer_captured_and_on_another_stream():
    """Captured into a graph and replayed on other inputs, and run on a stream of its own beside another: the same bits."""
    ops = _ops()
    ins = [_layer_inputs(257, 512, 640), _layer_inputs(257, 512, 640)]
    ins[1] = tuple(t.flip(0).contiguous() for t in ins[1])
    want = [[t.clone() for t in _layer(ops, *i)] for i in ins]
    static = [t.clone() for t in ins[0]]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _layer(ops, *static)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _layer(ops, *static)
    for k in (1, 0, 1):
        for a, b in zip(static, ins[k]):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[k]))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for st, i in zip(streams, ins):
        with torch.cuda.stream(st):
            got.append(_layer(ops, *i))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
    _no_errors()


def test_experts_with_the_routing_plan():
    """Router's plan, rows gathered by expert, both products of the experts and all three gradients, in 8 bits."""
    ops = _ops()
    torch.manual_seed(0)
    T, D, F, E, K = 300, 256, 384, 8, 2
    x, dy = torch.randn(T, D, device=DEV).bfloat16(), torch.randn(T, F, device=DEV).bfloat16()
    experts = torch.stack([torch.randperm(E - 1, device=DEV)[:K] for _ in range(T)]).to(torch.int32)      # the last expert gets none
    plan = ops.moe_plan(experts, E, pad=128)
    rows = ops.gather_rows(x, plan.row_src, idx_div=K)
    drows = ops.gather_rows(dy, plan.row_src, idx_div=K)
    w8 = ops.quant_fp8(0.1 * torch.randn(E, F, D, device=DEV).bfloat16(), "block")
    used = int(plan.offsets[-1])
    y = ops.grouped_gemm_fp8(ops.quant_fp8(rows, "row"), w8, plan.offsets)
    dx = ops.grouped_gemm_fp8(ops.quant_fp8(drows, "row"), w8, plan.offsets, trans_w=False)
    gw = torch.zeros(E, F, D, device=DEV)
    d8, x8 = ops.quant_fp8(drows, "col"), ops.quant_fp8(rows, "col")
    ops.grouped_wgrad_fp8(d8, x8, plan.offsets, gw, pad=128)
    X, DY, W = _value(ops.quant_fp8(rows, "row")), _value(ops.quant_fp8(drows, "row")), _value(w8)
    off = plan.offsets.tolist()
    for e in range(E):
        i, j = off[e], off[e + 1]
        for got, a, b, k in ((y, X, W[e].t(), D), (dx, DY, W[e], F)):
            want = a[i:j] @ b
            assert torch.all((got[i:j].double() - want).abs() <= _room(want, a[i:j].abs() @ b.abs(), k, torch.bfloat16))
        want = _value(d8)[i:j].t() @ _value(x8)[i:j]
        assert torch.all((gw[e].double() - want).abs() <= _room(want, _value(d8)[i:j].abs().t() @ _value(x8)[i:j].abs(), j - i + 1, torch.float32))
    assert used % 128 == 0 and off[-1] == off[-2]
    _no_errors()


def test_without_the_fast_call_extension(monkeypatch):
    """Every operator through ctypes, the path without the extension: the same bits."""
    from flextrain_b200.ops import cuda, fp8
    ops = _ops()
    ins = _layer_inputs(300, 256, 384)
    W = ops.quant_fp8(torch.randn(3, 200, 256, device=DEV), "block")
    off = torch.tensor([0, 128, 128, 256], device=DEV, dtype=torch.int32)
    gw = torch.randn(3, 384, 256, device=DEV)

    def everything():
        y = ops.grouped_gemm_fp8(ops.quant_fp8(ins[0]), W, off)[:256]
        g = ops.grouped_wgrad_fp8(ops.quant_fp8(ins[4], "col"), ops.quant_fp8(ins[0], "block"), off, gw.clone(), pad=128)
        return (*_layer(ops, *ins), y, g)

    want = everything()
    monkeypatch.setattr(cuda, "fastcall", lambda: None)
    monkeypatch.setattr(fp8, "_entries", {})
    got = everything()
    assert len(fp8._entries) == 3 and not any(hasattr(e, "func") for e in fp8._entries.values())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    _no_errors()


@pytest.mark.parametrize("form", ["fwd", "wgrad"])
def test_gemm_long_reductions_beside_another_stream(tile, form):
    """Hundreds of blocks whose values come early for some and late for others, memory and tensor cores busy with something else:
    right, and the same bits each time."""
    ops = _ops()
    torch.manual_seed(tile)
    M, N, K = 300, 520, 40001
    A, B, ta, tb, want, mag = _operands(form, M, N, K)
    busy = torch.randn(4096, 4096, device=DEV).bfloat16()
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(8):
        with torch.cuda.stream(other):
            busy.copy_(busy.flip(0))
            ops.linear_fp8_fwd(ops.quant_fp8(busy[:512]), ops.quant_fp8(busy, "block"))
        got.append(ops.gemm_fp8(A, B, trans_a=ta, trans_b=tb, out_dtype=torch.float32))
    torch.cuda.synchronize()
    assert torch.all((got[0].double() - want).abs() <= _room(want, mag, K, torch.float32))
    assert all(torch.equal(g, got[0]) for g in got[1:])
    _no_errors()


@pytest.mark.parametrize("group", ["col", "block"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_experts_gradients_of_part_of_a_group(tile, group, dtype):
    """A segment that starts or ends inside a group of 128 tokens: reported, its expert's sums as they were, the others' right."""
    ops = _ops()
    from flextrain_b200.ops import cuda as k
    torch.manual_seed(0)
    R, N, K = 700, 520, 136
    D, X = ops.quant_fp8(torch.randn(R, N, device=DEV), "col"), ops.quant_fp8(torch.randn(R, K, device=DEV), group)
    vd, vx = _value(D), _value(X)
    keep = torch.randn(4, N, K, device=DEV).to(dtype)
    k.device_error_words()
    for off, good in (([0, 128, 200, 384, R], [0, 3]), ([0, 256, 256, 300, 300], [0]), ([3, 128, 256, 384, 640], [1, 2, 3]), ([0, 100, 228, 356, R], [])):
        gw = keep.clone()
        ops.grouped_wgrad_fp8(D, X, torch.tensor(off, device=DEV, dtype=torch.int32), gw, pad=128)
        torch.cuda.synchronize()
        assert k.device_error_words()["gemm_fp8"] == 3040
        for e in range(4):
            i, j = off[e], off[e + 1]
            if e not in good:
                assert torch.equal(gw[e], keep[e])
                continue
            want = keep[e].double() + vd[i:j].t() @ vx[i:j]
            mag = keep[e].abs().double() + vd[i:j].abs().t() @ vx[i:j].abs()
            assert torch.all((gw[e].double() - want).abs() <= _room(want, mag, j - i, dtype))
    _no_errors()


def _within(got, want, room):
    return bool(torch.all((got.double().cpu() - want.cpu()).abs() <= room.cpu()))


@pytest.mark.parametrize("group", ["block", "col"])
@pytest.mark.parametrize("T,D,N", [(1, 256, 512), (130, 384, 640), (1000, 1024, 768)])
def test_layer_terms(T, D, N, group):
    """The run of a layer, each step against 64 bits of the operands that it reads (``group``: of a weight gradient's input; models have
    squares).  What a step hands on is 8 bits or bf16, and the next step's oracle starts from that, so that the room is a step's own
    roundings: a product's as everywhere here; of the norm's backward pass bf16's 2^-8 of each result, and 2^-24 for each of the D
    terms of a row's sum, the T terms of a gain's, and 16 more operations.  An oracle that misses a term is off by more."""
    ops = _ops()
    x, res, gain, w, dy = _layer_inputs(T, D, N)
    h8, rstd, h = ops.rmsnorm_fp8_fwd(x, gain, 1e-5, residual=res)
    w8, dy8, dyc = ops.quant_fp8(w, "block"), ops.quant_fp8(dy, "row"), ops.quant_fp8(dy, "col")
    y = ops.linear_fp8_fwd(h8, w8)
    dh = ops.linear_fp8_dgrad(dy8, w8)
    dgain = torch.zeros_like(gain)
    dx, n = ops.rmsnorm_bwd(dh, h, gain, rstd, dx_add=res, emit_y=True, dw_out=dgain)
    n8 = ops.quant_fp8(n, group)
    dw = torch.zeros(w.shape, device=DEV)
    ops.linear_fp8_wgrad(dyc, n8, dw)
    if group == "col":                                           # (as the other tests run it)
        assert all(torch.equal(a, b) for a, b in zip((y, dx, dw, dgain), _layer(ops, x, res, gain, w, dy)))

    # the operands in 8 bits: half a step of e4m3, the norm's scale and root
    hd, g = h.double(), gain.double()
    r = rstd.double()[:, None]
    xh = hd * r
    assert torch.equal(h, (x.float() + res.float()).bfloat16())
    assert torch.all((r - 1 / torch.sqrt((hd * hd).mean(-1, keepdim=True) + 1e-5)).abs() <= ((D / 128 + 20) * 2.0 ** -25 + 2.0 ** -22) * r)
    for m, v in ((h8, xh * g), (w8, w.double()), (dy8, dy.double()), (dyc, dy.double()), (n8, n.double())):
        step = torch.maximum(2.0 ** -4 * v.abs(), 2.0 ** -10 * _spread(m)) + 2.0 ** -20 * v.abs()
        assert torch.all((_value(m) - v).abs() <= step)

    vh, vw, vr, vc, vn = (_value(m) for m in (h8, w8, dy8, dyc, n8))
    for got, a, b, dtype in ((y, vh, vw.t(), torch.bfloat16), (dh, vr, vw, torch.bfloat16), (dw, vc.t(), vn, torch.float32)):
        want, mag = a @ b, a.abs() @ b.abs()
        assert _within(got, want, _room(want, mag, a.shape[1], dtype))
        for some in (a[:, :-1] @ b[:-1], torch.zeros_like(want)):          # a term too few in the reduction, nothing at all
            assert not _within(got, some, _room(some, mag, a.shape[1], dtype))

    assert _within(n, xh * g, (2.0 ** -8 + 8 * 2.0 ** -24) * (xh * g).abs())
    dn = dh.double() * g
    mean = (dn * xh).mean(-1, keepdim=True)
    mag = r * (dn.abs() + xh.abs() * (dn * xh).abs().mean(-1, keepdim=True)) + res.double().abs()
    room = lambda v: 2.0 ** -8 * v.abs() + (D + 16) * 2.0 ** -24 * mag
    want = r * (dn - xh * mean) + res.double()
    assert _within(dx, want, room(want))
    for wrong in (want - res.double(), r * dn + res.double(), r * (dh.double() - xh * mean) + res.double()):
        assert not _within(dx, wrong, room(wrong))
    terms = dh.double() * xh
    room = (T + 16) * 2.0 ** -24 * terms.abs().sum(0)
    assert _within(dgain, terms.sum(0), room)
    assert not _within(dgain, terms[:-1].sum(0), room) and not _within(dgain, torch.zeros_like(g), room)
    _no_errors()


def test_experts_with_squares():
    """What the layers run for experts: products by the routing plan, gradients of columns by squares; padded rows add nothing."""
    ops = _ops()
    torch.manual_seed(1)
    T, D, F, E, K = 300, 256, 384, 8, 2
    x, dy = torch.randn(T, D, device=DEV).bfloat16(), torch.randn(T, F, device=DEV).bfloat16()
    experts = torch.stack([torch.randperm(E - 1, device=DEV)[:K] for _ in range(T)]).to(torch.int32)
    plan = ops.moe_plan(experts, E, pad=128)
    off = plan.offsets.tolist()
    rows, drows = (ops.gather_rows(t, plan.row_src, idx_div=K) for t in (x, dy))
    d8, x8 = ops.quant_fp8(drows, "col"), ops.quant_fp8(rows, "block")
    for dtype in (torch.bfloat16, torch.float32):
        gw = torch.randn(E, F, D, device=DEV).to(dtype)
        keep = gw.clone()
        ops.grouped_wgrad_fp8(d8, x8, plan.offsets, gw, pad=128)
        vd, vx = _value(d8), _value(x8)
        for e in range(E):
            i, j = off[e], off[e + 1]
            want = keep[e].double() + vd[i:j].t() @ vx[i:j]
            mag = keep[e].double().abs() + vd[i:j].abs().t() @ vx[i:j].abs()
            room = _room(want, mag, j - i, dtype)
            assert _within(gw[e], want, room)
            tokens = (experts == e).any(1)
            # the tokens that the plan sends there, in 2-norm: two operands' roundings of 2^-4 / sqrt(6) each, four times that
            a, b = dy[tokens].double(), x[tokens].double()
            noise = 4 * 2.0 ** -4 / 3 ** 0.5 * ((a * a).t() @ (b * b)).sum().sqrt() + 2.0 ** -8 * want.norm()
            assert (gw[e].double() - keep[e].double() - a.t() @ b).norm() <= noise
            if j > i:
                assert not _within(keep[e], want, room) and (a.t() @ b).norm() > noise
    assert off[-1] == off[-2]
    _no_errors()


@pytest.mark.parametrize("M,N,K", [(1, 128, 128), (130, 257, 300), (300, 129, 130), (600, 520, 1000)])
def test_gemm_squares_read_down_their_columns(tile, M, N, K):
    """A in squares read across (a weight gradient of it), beside each kind of B."""
    ops = _ops()
    torch.manual_seed(M + N + K)
    a, b = torch.randn(K, M, device=DEV) * torch.exp(torch.randn(K, 1, device=DEV)), 0.1 * torch.randn(K, N, device=DEV)
    A = ops.quant_fp8(a, "block")
    for B, tb in ((ops.quant_fp8(b, "block"), False), (ops.quant_fp8(b, "col"), False), (ops.quant_fp8(b.t().contiguous(), "row"), True),
                  (ops.quant_fp8(b.t().contiguous(), "block"), True)):
        va, vb = _value(A).t(), _value(B).t() if tb else _value(B)
        want, mag = va @ vb, va.abs() @ vb.abs()
        for dtype in (torch.bfloat16, torch.float32):
            got = ops.gemm_fp8(A, B, trans_a=True, trans_b=tb, out_dtype=dtype)
            assert _within(got, want, _room(want, mag, K, dtype))
            c = torch.randn(M, N, device=DEV).to(dtype)
            w2, keep = want + c.double(), mag + c.abs().double()
            ops.gemm_fp8(A, B, trans_a=True, trans_b=tb, beta=1.0, out=c)
            assert _within(c, w2, _room(w2, keep, K, dtype))
    _no_errors()
