"""Models whose products run in 8 bits on the GPU: what every projection and every expert of a training step gives, against 64 bits of
the 16-bit tensors that it was called with, and against 64 bits of the operands that reached the products.

A rounding to e4m3 is off by 2^-4 / sqrt(6) = 0.026 of a value on average (uniform within a step, values spread over a binade), in no
direction.  So a product of two such operands is off, in the 2-norm, by sqrt(2) * 0.026 of the root of the summed squares of its terms;
four times that is allowed, and 2^-8 of the result for its own rounding.  Nothing in its place would be off by the whole norm."""
import pytest
import torch

import flextrain_b200 as ft
from flextrain_b200 import ops
from conftest import build_tiny

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
DIMS = dict(vocab_size=512, n_layers=2, d_model=256, n_heads=4, n_kv_heads=2, head_dim=64, expert_dim=640, ffn_dim=640, num_routed_experts=0,
            num_shared_experts=0, top_k=0, is_causal=True)
MOE = dict(DIMS, expert_dim=192, num_routed_experts=8, top_k=2)
SHARED = dict(MOE, num_shared_experts=1, shared_dim=320)
HYBRID = {"layer_pattern": "1L1F", "gdn": {"n_k_heads": 2, "n_v_heads": 4, "head_k_dim": 64, "head_v_dim": 64}}
SLIDING = {"sliding_window": 32, "layer_pattern": "SF"}
MODELS = [("qwen2", DIMS, None), ("qwen3", DIMS, None), ("gemma3", DIMS, SLIDING), ("gemma4", DIMS, SLIDING), ("qwen3_5", DIMS, HYBRID),
          ("qwen3_moe", MOE, None), ("olmoe", MOE, None), ("qwen3_next", SHARED, HYBRID), ("qwen3_5_moe", SHARED, HYBRID)]


class Checks:
    def __init__(self):
        self.seen, self.worst = {}, 0.0

    def near(self, what, got, a, b, add=None):
        """``got = a @ b (+ add)`` of unrounded ``a`` and ``b`` in 64 bits."""
        a, b, got = a.double(), b.double(), got.double()
        y = a @ b
        want = y if add is None else y + add.double()
        noise = 4 * 2.0 ** -4 / 3 ** 0.5 * (a.square() @ b.square()).sum().sqrt() + 2.0 ** -8 * want.norm() + 1e-30
        assert got.shape == want.shape
        off = float((got - want).norm() / noise)
        assert off <= 1, (what, off)
        self.worst = max(self.worst, off)
        self.seen[what] = self.seen.get(what, 0) + 1

    def exact(self, what, got, a, b, before):
        """``got = a @ b + before`` of the operands' values in 64 bits: a result's rounding, 2^-24 for each block and 2^-16 in one."""
        want, mag = a @ b + before, a.abs() @ b.abs() + before.abs()
        room = (2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24) * want.abs() + (2.0 ** -16 + (a.shape[1] / 128 + 6) * 2.0 ** -24) * mag
        assert torch.all((got.double() - want).abs() <= room), what
        self.seen[what] = self.seen.get(what, 0) + 1


@pytest.fixture
def checks(monkeypatch):
    from flextrain_b200.nn.blocks.ffn_moe import MoEFFN
    from flextrain_b200.nn.blocks.linear import LinearGroup
    k = Checks()
    value = lambda m: m if isinstance(m, torch.Tensor) else ops.dequant_fp8(m, torch.float32)
    fwd, dgrad, wgrad, product, mwgrad = LinearGroup.fwd, LinearGroup.dgrad, LinearGroup.wgrad, MoEFFN._product, MoEFFN._wgrad
    grouped_gemm, grouped_wgrad = ops.grouped_gemm_fp8, ops.grouped_wgrad_fp8

    def fwd_(self, x, params, *, residual=None, out=None):
        got = fwd(self, x, params, residual=residual, out=out)
        if self.fp8:
            add = [t for t in (residual, self.bias(params)) if t is not None]
            k.near("fwd", got, value(x), self.weight(params).t(), sum(t.double() for t in add) if add else None)
            k.seen["bias"] = k.seen.get("bias", 0) + (self.bias(params) is not None)
        return got

    def dgrad_(self, dy, params, **kw):
        got = dgrad(self, dy, params, **kw)
        if self.fp8:
            k.near("dgrad", got, dy, self.weight(params))
        return got

    def wgrad_(self, dy, x, params, grads, *, alpha=1.0):
        names = [g for g in ("g_" + n[2:] for n in self.names) if g in grads]
        before = {g: grads[g].double().clone() for g in names}
        wgrad(self, dy, x, params, grads, alpha=alpha)
        if self.fp8:
            r0 = 0
            for n in self.names:
                rows, g = params[n].shape[0], "g_" + n[2:]
                if g in before:
                    k.near("wgrad", grads[g], alpha * dy[:, r0:r0 + rows].t(), x, before[g])
                r0 += rows

    def product_(self, x, w, offsets, *, trans_w=True, out=None):
        got = product(self, x, w, offsets, trans_w=trans_w, out=out)
        o = offsets.tolist()
        for e, (i, j) in enumerate(zip(o, o[1:])):
            if j > i:
                k.near("experts fwd" if trans_w else "experts dgrad", got[i:j], x[i:j], w[e].t() if trans_w else w[e])
        return got

    def mwgrad_(self, dy, x, offsets, gw):
        before, o = gw.double().clone(), offsets.tolist()
        mwgrad(self, dy, x, offsets, gw)
        for e, (i, j) in enumerate(zip(o, o[1:])):
            k.near("experts wgrad", gw[e], dy[i:j].t(), x[i:j], before[e])

    def grouped_gemm_(x, w, offsets, *, trans_w=True, out=None, alpha=1.0, beta=0.0):
        assert (x.group, w.group, alpha, beta) == ("row", "block", 1.0, 0.0)
        got, vx, vw, o = grouped_gemm(x, w, offsets, trans_w=trans_w, out=out), value(x).double(), value(w).double(), offsets.tolist()
        for e, (i, j) in enumerate(zip(o, o[1:])):
            k.exact("grouped_gemm_fp8", got[i:j], vx[i:j], vw[e].t() if trans_w else vw[e], vx.new_zeros(()))
        return got

    def grouped_wgrad_(dy, x, offsets, gw, *, alpha=1.0, pad=1):
        assert (dy.group, x.group, alpha, pad) == ("col", "block", 1.0, 128)
        before, vd, vx, o = gw.double().clone(), value(dy).double(), value(x).double(), offsets.tolist()
        grouped_wgrad(dy, x, offsets, gw, pad=pad)
        for e, (i, j) in enumerate(zip(o, o[1:])):
            k.exact("grouped_wgrad_fp8", gw[e], vd[i:j].t(), vx[i:j], before[e])
        return gw

    monkeypatch.setattr(LinearGroup, "fwd", fwd_)
    monkeypatch.setattr(LinearGroup, "dgrad", dgrad_)
    monkeypatch.setattr(LinearGroup, "wgrad", wgrad_)
    monkeypatch.setattr(MoEFFN, "_product", product_)
    monkeypatch.setattr(MoEFFN, "_wgrad", mwgrad_)
    monkeypatch.setattr(ops, "grouped_gemm_fp8", grouped_gemm_)
    monkeypatch.setattr(ops, "grouped_wgrad_fp8", grouped_wgrad_)
    return k


@pytest.mark.parametrize("arch,dims,hyper", MODELS, ids=[m[0] for m in MODELS])
@pytest.mark.parametrize("level", [None, 0])
def test_training_step(checks, arch, dims, hyper, level):
    """Biases, norms of heads and rows, sandwich norms, gated attention beside Gated DeltaNet, routed and shared experts; activations
    saved and computed again."""
    ws = ft.WorkingSetConfig.simple(max_seq_len=160, max_global_batch_tokens=640, chunk=320)
    am = build_tiny(arch, dims=dims, hyper=hyper, device="cuda:0", dtype=torch.bfloat16, max_seq_len=160, batch_tokens=640, ws=ws,
                    force_saved_act_level=level, linear_dtype=FP8)
    g = torch.Generator().manual_seed(1)
    for _, _, name, t in am.named_master_params():
        if name.startswith("b_") or "norm" in name:
            t.add_(0.1 * torch.randn(t.shape, generator=g).to(t))
    seqs = ft.SyntheticTokenSource(512, 160, seed=0).get_sequences(640)
    am.fwd_bwd(seqs)
    assert am.step() == 0
    checks.seen.clear()
    ops.reset_backends_used()
    st = am.fwd_bwd(seqs)
    used, s = ops.backends_used(), checks.seen
    assert st.loss == st.loss and am.step() == 0
    layers, chunks = am.layers, 2
    moe = sum(l.moe is not None for l in layers)
    shared = sum(l.moe is not None and l.moe.shared is not None for l in layers)
    attn, ffn = sum(l.attn is not None for l in layers), sum(l.ffn is not None for l in layers)
    groups = 2 * (attn + ffn + shared)
    members = 4 * attn + 3 * (ffn + shared)                      # q, k, v, o; gate, up, down
    assert s.get("fwd", 0) >= chunks * groups and s.get("dgrad", 0) == chunks * groups and s.get("wgrad", 0) == chunks * members
    assert (s.get("bias", 0) > 0) == (arch == "qwen2")
    if moe:
        assert s["experts wgrad"] == 2 * chunks * moe * dims["num_routed_experts"]
        assert s["grouped_wgrad_fp8"] == s["experts wgrad"] and s["grouped_gemm_fp8"] >= 2 * 2 * chunks * moe
        assert s["experts fwd"] > 0 and s["experts dgrad"] > 0
    for family in ("quant_fp8", "gemm_fp8") + (("grouped_gemm_fp8", "grouped_wgrad_fp8") if moe else ()):
        assert used[family] == ["ftb"], used
    for scope, l, name, t in am.named_master_params():
        assert torch.isfinite(t).all(), (scope, l, name)
    from flextrain_b200.ops.cuda import device_error_words
    torch.cuda.synchronize()
    assert device_error_words().get("gemm_fp8", 0) == 0
