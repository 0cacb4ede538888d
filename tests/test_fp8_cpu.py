"""Linear layers in 8 bits on the CPU: the quantisers against their definition, the products against the values, refusals."""
import pytest
import torch

from flextrain_b200 import ops

FP8 = torch.float8_e4m3fn


@pytest.mark.parametrize("group,down,along", [("row", 1, 128), ("col", 128, 1), ("block", 128, 128)])
@pytest.mark.parametrize("M,N", [(1, 1), (130, 257), (128, 128), (0, 5), (5, 0)])
def test_quant_is_its_definition(group, down, along, M, N):
    torch.manual_seed(0)
    x = torch.randn(M, N) * torch.exp(torch.randn(M, 1))
    m = ops.quant_fp8(x, group)
    assert m.data.shape == (M, N) and m.scale.shape == (-(-M // down), -(-N // along))
    for i in range(m.scale.shape[0]):
        for j in range(m.scale.shape[1]):
            part = x[i * down:(i + 1) * down, j * along:(j + 1) * along].double()
            s = max(float(part.abs().max()) / 448 if part.numel() else 0, 2.0 ** -126)
            assert abs(float(m.scale[i, j]) - s) <= 2.0 ** -24 * s
            q = m.data[i * down:(i + 1) * down, j * along:(j + 1) * along].double()
            # half a step of e4m3, 2^-4 of the value or 2^-10 of the scale; the scale and its reciprocal are rounded once each
            assert torch.all((q * s - part).abs() <= torch.clamp(2.0 ** -4 * part.abs(), min=2.0 ** -10 * s) * (1 + 2.0 ** -20))
            assert not part.numel() or float(q.abs().max()) == (448 if part.abs().max() > 0 else 0)


def test_zeros_and_what_is_not_a_number():
    x = torch.zeros(2, 300)
    x[1, 5], x[1, 200] = float("nan"), float("inf")
    m = ops.quant_fp8(x)
    assert torch.all(m.scale[0] == 2.0 ** -126) and torch.all(m.data[0].float() == 0)
    v = ops.dequant_fp8(m, torch.float32)
    assert torch.isnan(v[1, :256]).all() and torch.all(v[1, 256:] == 0) and torch.all(v[0] == 0)


def test_norm_is_the_norm_of_the_rounded_sum():
    torch.manual_seed(0)
    x, r = torch.randn(5, 200).bfloat16(), torch.randn(5, 200).bfloat16()
    w = torch.rand(200) + 0.5
    m, rstd, h = ops.rmsnorm_fp8_fwd(x, w, 1e-5, residual=r)
    assert torch.equal(h, (x.float() + r.float()).bfloat16())
    y, rstd2 = ops.rmsnorm_fwd(h.float(), w, 1e-5)
    q, s = ops.ref.quant_fp8(y, "row")
    assert torch.equal(rstd, rstd2) and torch.equal(m.scale, s) and torch.equal(m.data.view(torch.uint8), q.view(torch.uint8))


@pytest.mark.parametrize("M,N,K", [(3, 5, 7), (130, 140, 260), (1, 1, 1), (0, 4, 4), (4, 4, 0)])
def test_products_of_the_values(M, N, K):
    torch.manual_seed(0)
    a, b = torch.randn(M, K), torch.randn(N, K)
    c, bias = torch.randn(M, N), torch.randn(N)
    for trans_a in (False, True):
        for trans_b in (False, True):
            A = ops.quant_fp8(a.t().contiguous(), "col") if trans_a else ops.quant_fp8(a, "row")
            for groups in ("block", "vector"):
                B = ops.quant_fp8(b if trans_b else b.t().contiguous(), "block" if groups == "block" else "row" if trans_b else "col")
                va, vb = ops.dequant_fp8(A, torch.float64), ops.dequant_fp8(B, torch.float64)
                want = 0.5 * (va.t() if trans_a else va) @ (vb.t() if trans_b else vb) + 2 * c.double() + bias.double()
                got = ops.gemm_fp8(A, B, trans_a=trans_a, trans_b=trans_b, alpha=0.5, beta=2.0, c=c, bias=bias, out_dtype=torch.float32)
                torch.testing.assert_close(got.double(), want, rtol=1e-5, atol=1e-4)


def test_grouped_products_of_the_values():
    torch.manual_seed(0)
    off = torch.tensor([0, 3, 3, 140])
    X, W = ops.quant_fp8(torch.randn(150, 70), "row"), ops.quant_fp8(torch.randn(3, 40, 70), "block")
    vx, vw = ops.dequant_fp8(X, torch.float64), ops.dequant_fp8(W, torch.float64)
    out = torch.full((150, 40), 7.0)
    ops.grouped_gemm_fp8(X, W, off, out=out)
    for e in range(3):
        torch.testing.assert_close(out[off[e]:off[e + 1]].double(), vx[off[e]:off[e + 1]] @ vw[e].t(), rtol=1e-5, atol=1e-4)
    assert torch.all(out[140:] == 7)
    off = torch.tensor([0, 128, 128, 256])
    D, X = ops.quant_fp8(torch.randn(256, 40), "col"), ops.quant_fp8(torch.randn(256, 70), "col")
    gw = torch.ones(3, 40, 70)
    ops.grouped_wgrad_fp8(D, X, off, gw, pad=128)
    for e in range(3):
        want = 1 + ops.dequant_fp8(D, torch.float64)[off[e]:off[e + 1]].t() @ ops.dequant_fp8(X, torch.float64)[off[e]:off[e + 1]]
        torch.testing.assert_close(gw[e].double(), want, rtol=1e-5, atol=1e-4)


def test_gradients_against_differences():
    """The products' gradients against differences of the loss, with values that 8 bits hold exactly."""
    torch.manual_seed(0)
    pick = lambda *s: torch.randint(-8, 9, s).float()
    x, w, dy = pick(4, 130), pick(6, 130), pick(4, 6)
    for t in (x, w, dy):                                         # largest magnitudes of 448 / 32: scales of 2^-5, nothing rounded
        t[:, 0], t[:, -1] = 14, 14
        t[0], t[-1] = 14, 14
    exact = lambda t, g: ops.quant_fp8(t, g)
    for t, g in ((x, "row"), (x, "col"), (w, "block"), (dy, "row"), (dy, "col")):
        assert torch.equal(ops.dequant_fp8(exact(t, g), torch.float32), t)
    loss = lambda x, w: float(((x.double() @ w.double().t()) * dy.double()).sum())
    assert torch.equal(ops.linear_fp8_fwd(exact(x, "row"), exact(w, "block"), out=torch.empty(4, 6)).double(), x.double() @ w.double().t())
    dx = ops.linear_fp8_dgrad(exact(dy, "row"), exact(w, "block"), out=torch.empty(4, 130))
    dw = ops.linear_fp8_wgrad(exact(dy, "col"), exact(x, "col"), torch.empty(6, 130), accumulate=False)
    for i, j in ((0, 0), (1, 64), (3, 129), (2, 100)):
        e = torch.zeros_like(x)
        e[i, j] = 0.5
        assert float(dx[i, j]) == loss(x + e, w) - loss(x - e, w)
        e = torch.zeros_like(w)
        e[i, j] = 0.5
        assert float(dw[i, j]) == loss(x, w + e) - loss(x, w - e)


def _m(groups, M, N, **over):
    m = ops.quant_fp8(torch.ones(M, N), groups)
    return m._replace(**over)


@pytest.mark.parametrize("call", [
    lambda: ops.quant_fp8(torch.ones(2, 2), "rows"),
    lambda: ops.quant_fp8(torch.ones(2, 2, dtype=torch.float16)),
    lambda: ops.quant_fp8(torch.ones(2)),
    lambda: ops.quant_fp8(torch.ones(2, 2, 2), "row"),
    lambda: ops.rmsnorm_fp8_fwd(torch.ones(2, 4), torch.ones(5), 1e-5),
    lambda: ops.rmsnorm_fp8_fwd(torch.ones(2, 4), None, 1e-5, residual=torch.ones(1, 4)),
    lambda: ops.rmsnorm_fp8_fwd(torch.ones(2, 4), None, 1e-5, residual=torch.ones(2, 4).bfloat16()),
    lambda: ops.rmsnorm_fp8_fwd(torch.ones(4), None, 1e-5),
    lambda: ops.rmsnorm_fp8_fwd(torch.ones(2, 4, dtype=torch.float16), None, 1e-5),
    lambda: ops.gemm_fp8(_m("row", 4, 8), _m("row", 8, 4)),                         # groups that do not run along the reduction
    lambda: ops.gemm_fp8(_m("col", 4, 8), _m("block", 8, 4)),
    lambda: ops.gemm_fp8(_m("row", 4, 8), _m("block", 9, 4)),                       # inner sizes
    lambda: ops.gemm_fp8(_m("row", 4, 8, scale=torch.ones(4, 2)), _m("block", 8, 4)),
    lambda: ops.gemm_fp8(_m("row", 4, 8, scale=torch.ones(4, 1, dtype=torch.float64)), _m("block", 8, 4)),
    lambda: ops.gemm_fp8(_m("row", 4, 8, data=torch.ones(4, 8)), _m("block", 8, 4)),
    lambda: ops.gemm_fp8(_m("row", 4, 8, group="rows"), _m("block", 8, 4)),
    lambda: ops.gemm_fp8(_m("row", 4, 8), ops.quant_fp8(torch.ones(2, 8, 4), "block")),
    lambda: ops.gemm_fp8(_m("row", 4, 8), _m("block", 8, 4), out_dtype=torch.float16),
    lambda: ops.gemm_fp8(_m("row", 4, 8), _m("block", 8, 4), out=torch.ones(4, 4), out_dtype=torch.bfloat16),
    lambda: ops.gemm_fp8(_m("row", 4, 8), _m("block", 8, 4), out=torch.ones(4, 5)),
    lambda: ops.gemm_fp8(_m("row", 4, 8), _m("block", 8, 4), out=torch.ones(4, 4).t()),
    lambda: ops.gemm_fp8(_m("row", 4, 8), _m("block", 8, 4), out=torch.ones(1, 4).expand(4, 4)),     # rows over one another
    lambda: ops.gemm_fp8(_m("row", 4, 8), _m("block", 8, 4), out=torch.ones(16).as_strided((4, 4), (2, 1))),
    lambda: ops.gemm_fp8(_m("row", 4, 8), _m("block", 8, 4), beta=1.0),
    lambda: ops.gemm_fp8(_m("row", 4, 8), _m("block", 8, 4), beta=1.0, c=torch.ones(4, 4)),          # c in fp32, result in bf16
    lambda: ops.gemm_fp8(_m("row", 4, 8), _m("block", 8, 4), bias=torch.ones(5)),
    lambda: ops.gemm_fp8(_m("row", 4, 8), _m("block", 8, 4), bias=torch.ones(4).bfloat16()),
    lambda: ops.grouped_gemm_fp8(_m("row", 4, 8), _m("block", 8, 4), torch.tensor([0, 4])),
    lambda: ops.grouped_gemm_fp8(_m("block", 4, 8), ops.quant_fp8(torch.ones(1, 4, 8), "block"), torch.tensor([0, 4])),
    lambda: ops.grouped_gemm_fp8(_m("row", 4, 8), ops.quant_fp8(torch.ones(1, 4, 8), "block"), torch.tensor([0, 2, 4])),
    lambda: ops.grouped_gemm_fp8(_m("row", 4, 8), ops.quant_fp8(torch.ones(1, 4, 8), "block"), torch.tensor([0.0, 4.0])),
    lambda: ops.grouped_gemm_fp8(_m("row", 4, 8), ops.quant_fp8(torch.ones(1, 4, 9), "block"), torch.tensor([0, 4])),
    lambda: ops.grouped_gemm_fp8(_m("row", 4, 8), ops.quant_fp8(torch.ones(1, 4, 8), "block"), torch.tensor([0, 4]), beta=1.0),
    lambda: ops.grouped_wgrad_fp8(_m("col", 128, 8), _m("col", 128, 4), torch.tensor([0, 128]), torch.ones(1, 8, 4)),
    lambda: ops.grouped_wgrad_fp8(_m("col", 128, 8), _m("col", 128, 4), torch.tensor([0, 128]), torch.ones(1, 8, 4), pad=64),
    lambda: ops.grouped_wgrad_fp8(_m("row", 128, 8), _m("col", 128, 4), torch.tensor([0, 128]), torch.ones(1, 8, 4), pad=128),
    lambda: ops.grouped_wgrad_fp8(_m("col", 128, 8), _m("col", 256, 4), torch.tensor([0, 128]), torch.ones(1, 8, 4), pad=128),
    lambda: ops.grouped_wgrad_fp8(_m("col", 128, 8), _m("col", 128, 4), torch.tensor([0, 128]), torch.ones(1, 4, 8).mT, pad=128),
])
def test_refusals(call):
    with pytest.raises(ValueError):
        call()


@pytest.mark.parametrize("extension", [True, False])
def test_an_entry_point_gets_its_arguments(monkeypatch, extension):
    """All words of a call (integers, addresses, None as 0, floats as the bits of a double) are there while the library reads them,
    through the extension and through ctypes."""
    import ctypes
    import struct
    from types import SimpleNamespace

    from flextrain_b200.ops import cuda, fp8
    args = [*range(1000, 1033), (1 << 62) + 5, -7, 0.5, -3e-40, None, True, False]
    got = []

    @ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p)
    def library(at):
        [bytearray(8 * len(args)) for _ in range(64)]              # (whatever a callee allocates)
        got.append(list((ctypes.c_int64 * len(args)).from_address(at)))
        return 17

    if extension:
        assert cuda.fastcall() is not None, "fastcall extension was not built"
    else:
        monkeypatch.setattr(cuda, "fastcall", lambda: None)
    monkeypatch.setattr(cuda, "load", lambda name: SimpleNamespace(entry=library))
    entry = fp8._entry("lib", "entry")
    want = [struct.unpack("q", struct.pack("d", a))[0] if isinstance(a, float) else int(a or 0) for a in args]
    for _ in range(3):
        assert entry(*args) == 17
    assert got == [want] * 3


@pytest.mark.parametrize("off", [[0, 100, 256], [0, 128, 200], [-3, 128, 256], [0, 130, 130], [64, 64, 128]])
def test_experts_gradients_of_part_of_a_group(off):
    """A segment that starts or ends inside a group of 128 tokens: refused before anything is written."""
    D, X = ops.quant_fp8(torch.randn(256, 40), "col"), ops.quant_fp8(torch.randn(256, 70), "block")
    gw = torch.ones(2, 40, 70)
    with pytest.raises(ValueError, match="inside a group of 128"):
        ops.grouped_wgrad_fp8(D, X, torch.tensor(off), gw, pad=128)
    assert torch.all(gw == 1)


def test_experts_gradients_of_the_last_rows():
    """Rows that end where the data does, an empty segment wherever it lies, offsets behind the rows: taken."""
    D, X = ops.quant_fp8(torch.randn(200, 40), "col"), ops.quant_fp8(torch.randn(200, 70), "block")
    vd, vx = ops.dequant_fp8(D, torch.float64), ops.dequant_fp8(X, torch.float64)
    for off, rows in (([0, 128, 200], [(0, 128), (128, 200)]), ([0, 0, 1000], [(0, 0), (0, 200)]), ([0, 128, 128], [(0, 128), (0, 0)]),
                      ([130, 130, 130], [(0, 0), (0, 0)])):
        gw = torch.ones(2, 40, 70)
        ops.grouped_wgrad_fp8(D, X, torch.tensor(off), gw, pad=128)
        for g, (i, j) in zip(gw, rows):
            torch.testing.assert_close(g.double(), 1 + vd[i:j].t() @ vx[i:j], rtol=1e-5, atol=1e-4)



@pytest.mark.parametrize("out,c,apart", [
    (((4, 8), (8, 1), 8), ((4, 8), (8, 1), 0), False),                       # a row further down
    (((4, 8), (8, 1), 3), ((4, 8), (8, 1), 0), False),                       # three elements further on
    (((4, 8), (20, 1), 4), ((4, 8), (20, 1), 0), False),                     # columns that meet
    (((4, 8), (8, 1), 0), ((4, 8), (0, 1), 8), False),                       # one of the result's rows for all
    (((4, 8), (8, 1), 0), ((4, 8), (16, 1), 0), False),                      # the same place with other strides
    (((4, 8), (8, 1), 0), ((4, 8), (8, 1), 0), True),                        # the result itself
    (((4, 8), (20, 1), 0), ((4, 8), (20, 1), 8), True),                      # columns beside it
    (((4, 8), (20, 1), 12), ((4, 8), (20, 1), 0), True),
    (((4, 8), (8, 1), 0), ((4, 8), (8, 1), 32), True),                       # rows behind it
    (((4, 8), (8, 1), 0), ((4, 8), (0, 1), 32), True),
    (((4, 8), (8, 1), 0), ((4, 8), (1, 4), 0), True),                        # (columns that lie apart are copied first)
])
def test_c_over_the_result(out, c, apart):
    """C is read while the result is written: what lies partly over it is refused, what lies beside it or is the result itself is taken."""
    torch.manual_seed(0)
    base = torch.randn(200)
    a, b = _m("row", 4, 8), _m("block", 8, 8)
    d, c = base.as_strided(*out), base.as_strided(*c)
    if not apart:
        with pytest.raises(ValueError, match="over the result"):
            ops.gemm_fp8(a, b, beta=1.0, c=c, out=d)
        return
    want = 8 + c.clone()
    assert torch.equal(ops.gemm_fp8(a, b, beta=1.0, c=c, out=d), want) and torch.equal(d, want)


def test_a_single_row_of_c_has_no_stride():
    base = torch.randn(40)
    a, b = _m("row", 1, 8), _m("block", 8, 8)
    out, c = base.as_strided((1, 8), (8, 1), 4), base.as_strided((1, 8), (30, 1), 4)
    want = 8 + c.clone()
    assert torch.equal(ops.gemm_fp8(a, b, beta=1.0, c=c, out=out), want)
    with pytest.raises(ValueError, match="over the result"):
        ops.gemm_fp8(a, b, beta=1.0, c=base.as_strided((1, 8), (30, 1), 5), out=out)


def test_offsets_of_64_bits_do_not_wrap():
    """Offsets beyond 32 bits name rows outside of those that there are, not others inside."""
    far = 1 << 32
    X, W = ops.quant_fp8(torch.randn(256, 40), "row"), ops.quant_fp8(torch.randn(2, 24, 40), "block")
    want = torch.full((256, 24), 7.0)
    ops.grouped_gemm_fp8(X, W, torch.tensor([0, 100, 256]), out=want)
    for off, rows in (([0, 100, far + 120], slice(0, 256)), ([0, far + 90, far + 120], None), ([far, far + 10, far + 20], slice(0, 0)),
                      ([-far - 3, 100, far], slice(0, 256))):
        out = torch.full((256, 24), 7.0)
        ops.grouped_gemm_fp8(X, W, torch.tensor(off), out=out)
        if rows is not None:
            assert torch.equal(out[rows], want[rows]) and torch.all(out[rows.stop:] == 7), off
        else:                                                    # the first expert has all rows, the second none
            ref = torch.full((256, 24), 7.0)
            ops.grouped_gemm_fp8(X, W, torch.tensor([0, 256, 256]), out=ref)
            assert torch.equal(out, ref)
    D, X = ops.quant_fp8(torch.randn(256, 24), "col"), ops.quant_fp8(torch.randn(256, 40), "block")
    got, want = torch.zeros(2, 24, 40), torch.zeros(2, 24, 40)
    ops.grouped_wgrad_fp8(D, X, torch.tensor([0, 128, far + 128]), got, pad=128)
    ops.grouped_wgrad_fp8(D, X, torch.tensor([0, 128, 256]), want, pad=128)
    assert torch.equal(got, want)
