"""Models whose products run in 8 bits (``linear_dtype``), on the CPU: against a model without it whose 16-bit products get their
operands rounded, under every save tier, with adapters and with experts; against autograd; the plan's memory; what is refused.

The rounded model forms the same fp32 sums from the same operands, in the same order but for the norm's (2^-22 apart).  A value next
to the middle of two e4m3 numbers that falls to the other side there moves what follows, and what follows is rounded again; the two
models are compared where the values agree to the bit or differ by such single steps: 2^-4 of single values."""
import pytest
import torch

import flextrain_b200 as ft
from flextrain_b200 import ops
from flextrain_b200.bench import naive
from conftest import build_tiny

FP8 = torch.float8_e4m3fn
DIMS = dict(vocab_size=512, n_layers=2, d_model=256, n_heads=4, n_kv_heads=2, head_dim=64, expert_dim=640, num_routed_experts=0,
            num_shared_experts=0, top_k=0, is_causal=True)
MOE = dict(DIMS, expert_dim=128, num_routed_experts=4, top_k=2)


def _round(x, group):
    return ops.dequant_fp8(ops.quant_fp8(x.contiguous(), group), torch.float32)


def _seqs(am):
    return ft.SyntheticTokenSource(512, 128, seed=0).get_sequences(256)


def _rel(a, b):
    return float((a.double() - b.double()).norm() / (b.double().norm() + 1e-30))


def _grads(am):
    bm = am.buffers
    return lambda scope, l: {"embed": bm.embed_grads(), "head": bm.head_grads()}.get(scope) or bm.grads(l)


def _rounded_products(monkeypatch):
    """The products of models without ``linear_dtype`` round their operands from here on."""
    from flextrain_b200.nn.blocks.ffn_moe import MoEFFN
    from flextrain_b200.nn.blocks.linear import LinearGroup
    pads = lambda x, off: torch.cat([x[:int(off[-1])], torch.zeros_like(x[int(off[-1]):])])      # (rows behind the last segment)
    monkeypatch.setattr(MoEFFN, "_product", lambda self, x, w, off, *, trans_w=True, out=None: ops.grouped_gemm(
        _round(pads(x, off), "row"), _round(w, "block"), off, trans_w=trans_w, out=out))
    monkeypatch.setattr(MoEFFN, "_wgrad", lambda self, dy, x, off, gw: ops.grouped_wgrad(
        _round(pads(dy, off), "col"), _round(pads(x, off), "block"), off, gw, pad=128))
    monkeypatch.setattr(LinearGroup, "fwd", lambda self, x, params, *, residual=None, out=None: ops.linear_fwd(
        _round(x, "row"), _round(self.weight(params), "block"), bias=self.bias(params), residual=residual, out=out))
    monkeypatch.setattr(LinearGroup, "dgrad", lambda self, dy, params, *, out=None, accumulate=False: ops.linear_dgrad(
        _round(dy, "row"), _round(self.weight(params), "block"), out=out, accumulate=accumulate))
    monkeypatch.setattr(ops, "linear_wgrad", lambda dy, x, gw, *, alpha=1.0, accumulate=True: ops.gemm(
        _round(dy, "col"), _round(x, "block"), trans_a=True, alpha=alpha, beta=1.0, out=gw))

    def glu_fwd(x, w, kind="swiglu", *, x13=None):
        F, y = w.shape[0] // 2, ops.linear_fwd(_round(x, "row"), _round(w, "block"), out=x13)
        return y, ops.glu_fwd(y[:, :F], y[:, F:], kind)

    def glu_bwd(dy, w2, x13, kind="swiglu"):
        F = w2.shape[1]
        dg, du, act = ops.glu_bwd(ops.linear_dgrad(_round(dy, "row"), _round(w2, "block")), x13[:, :F], x13[:, F:], kind)
        return torch.cat([dg, du], 1), act
    monkeypatch.setattr(ops, "linear_glu_fwd", glu_fwd)
    monkeypatch.setattr(ops, "linear_glu_bwd", glu_bwd)


def _same(am, other, only=""):
    seen = 0
    for scope, l, name, _ in am.named_master_params():
        a, b = (_grads(m)(scope, l).get("g_" + name[2:]) for m in (am, other))
        assert (a is None) == (b is None)
        if a is not None and only in name:
            assert _rel(a, b) <= 2.0 ** -4 * 2.0 ** -7, (scope, l, name)
            seen += 1
    return seen


@pytest.mark.parametrize("arch", ["llama", "qwen2", "qwen3", "gemma2"])
@pytest.mark.parametrize("level", [None, 0, 2])
def test_dense(monkeypatch, arch, level):
    """Biases, norms of heads, sandwich norms; activations saved and computed again."""
    am, other = (build_tiny(arch, dims=DIMS, force_saved_act_level=level, **kw) for kw in (dict(linear_dtype=FP8), {}))
    plain = other.fwd_bwd(_seqs(other)).loss
    other = build_tiny(arch, dims=DIMS, force_saved_act_level=level)
    st = am.fwd_bwd(_seqs(am))
    _rounded_products(monkeypatch)
    st2 = other.fwd_bwd(_seqs(other))
    assert abs(st.loss - st2.loss) < 1e-5 and abs(st.loss - plain) > 1e-5      # (the rounding is there)
    assert _same(am, other) > 20


def test_adapters(monkeypatch):
    """LoRA: the merged weight in 8 bits forward and for the input's gradient, the adapters' own gradients in full."""
    am, other = (build_tiny("llama", dims=DIMS, lora_targets="all", lora_rank=8, lora_alpha=16.0, **kw) for kw in (dict(linear_dtype=FP8), {}))
    for m in (am, other):
        g = torch.Generator().manual_seed(1)
        for scope, l, name, t in m.named_master_params():
            if name.endswith("_lora_b"):
                t.copy_(0.05 * torch.randn(t.shape, generator=g))
    st = am.fwd_bwd(_seqs(am))
    _rounded_products(monkeypatch)
    assert abs(st.loss - other.fwd_bwd(_seqs(other)).loss) < 1e-5
    assert _same(am, other, "_lora_") == 2 * 7 * 2


@pytest.mark.parametrize("shared", [0, 1])
def test_experts(monkeypatch, shared):
    dims = dict(MOE, num_shared_experts=shared)
    am, other = build_tiny("qwen3_moe", dims=dims, linear_dtype=FP8), build_tiny("qwen3_moe", dims=dims)
    assert am.layers[0].moe.fp8 and (am.layers[0].moe.shared is not None) == bool(shared)
    st = am.fwd_bwd(_seqs(am))
    _rounded_products(monkeypatch)
    assert abs(st.loss - other.fwd_bwd(_seqs(other)).loss) < 1e-5
    assert _same(am, other) > 20


class _Linear8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(x, w)
        return _round(x, "row") @ _round(w, "block").t()

    @staticmethod
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        return _round(dy, "row") @ _round(w, "block"), _round(dy, "col").t() @ _round(x, "block")


def _lin8(P, l, name, x, lora_scale=None):
    w = P[("layer", l, name)]
    a = P.get(("layer", l, name + "_lora_a"))
    if a is not None:
        w = w + lora_scale * (P[("layer", l, name + "_lora_b")] @ a)
    return _Linear8.apply(x, w)


def test_against_autograd(monkeypatch):
    """Straight-through gradients of rounded operands.  This oracle's sums are formed in another order, so that its roundings are
    others, too: a rounding's error is 2^-4 of a value at most and 0.026 of it on average (2^-4 / sqrt(6)), and a gradient goes
    through 2 layers of 7 products with two rounded operands each, there and back: sqrt(56) * 0.026 = 0.19."""
    am = build_tiny("llama", dims=DIMS, linear_dtype=FP8)
    seqs = _seqs(am)
    P = naive.clone_params(am)
    monkeypatch.setattr(naive, "_lin", _lin8)
    loss = naive.naive_loss(am, P, seqs)
    loss.backward()
    st = am.fwd_bwd(seqs)
    assert abs(st.loss - float(loss)) < 0.02 * float(loss)
    for (scope, l, name), p in P.items():
        assert _rel(_grads(am)(scope, l)["g_" + name[2:]], p.grad) < 0.19, (scope, l, name)


def test_steps_and_evaluation():
    """Weights that change are used as they are: a second step's loss is that of its own weights."""
    am = build_tiny("llama", dims=DIMS, linear_dtype=FP8)
    seqs = _seqs(am)
    am.fwd_bwd(seqs)
    assert am.step() == 0
    st = am.fwd_bwd(seqs)
    fresh = build_tiny("llama", dims=DIMS, linear_dtype=FP8)
    for (_, _, _, a), (_, _, _, b) in zip(fresh.named_master_params(), am.named_master_params()):
        a.copy_(b)
    assert abs(fresh.fwd_bwd(seqs).loss - st.loss) < 1e-6


@pytest.mark.parametrize("dims,arch", [(DIMS, "llama"), (MOE, "qwen3_moe")])
def test_the_plan_counts_what_products_hold(dims, arch):
    from flextrain_b200.core.working_set import _fp8_bytes, _workspace_bytes
    am, other = build_tiny(arch, dims=dims, linear_dtype=FP8), build_tiny(arch, dims=dims)
    for chunk in (1, 128, 5000):
        c = am.layers[0].cfg
        more = _workspace_bytes(am.layers, am.head, chunk) - _workspace_bytes(other.layers, other.head, chunk)
        assert more == _fp8_bytes(c, chunk) > 0
        size = lambda m: m.data.numel() + 4 * m.scale.numel()
        z = lambda *s: torch.zeros(*s)
        if c.ffn is not None:
            w, x, dy = z(2 * c.ffn.ffn_dim, c.d_model), z(chunk, c.d_model), z(chunk, 2 * c.ffn.ffn_dim)
            assert size(ops.quant_fp8(w, "block")) + size(ops.quant_fp8(x)) <= more
            assert size(ops.quant_fp8(w, "block")) + size(ops.quant_fp8(dy)) <= more
            assert size(ops.quant_fp8(x, "col")) + size(ops.quant_fp8(dy, "col")) <= more
        else:
            w = z(c.moe.num_experts, 2 * c.moe.expert_dim, c.d_model)
            rows = ops.ref.moe_rows_bound(chunk, c.moe.top_k, c.moe.num_experts, 128)
            assert size(ops.quant_fp8(w, "block")) + size(ops.quant_fp8(z(rows, c.d_model))) <= more


@pytest.mark.parametrize("kw,err", [(dict(linear_dtype=torch.float16), ValueError), (dict(linear_dtype=torch.float8_e5m2), ValueError),
                                    (dict(linear_dtype=FP8, dtype=torch.float64), ValueError),
                                    (dict(linear_dtype=FP8, tp=2), NotImplementedError), (dict(linear_dtype=FP8, ep=2), NotImplementedError),
                                    (dict(linear_dtype=FP8, world_size=2), NotImplementedError)])
def test_refusals(kw, err):
    with pytest.raises(err):
        build_tiny("llama", dims=DIMS, **kw)
    assert build_tiny("llama", dims=DIMS, linear_dtype=torch.float32).layers[0].cfg.linear_fp8 is False


@pytest.mark.parametrize("device", ["cuda:0", "cuda", torch.device("cuda", 0)])
def test_full_precision_on_a_gpu_is_refused_when_the_model_is_built(device):
    """The norm and the quantisers' products write bf16 there; a model of another type says so before anything is allocated."""
    for kw in (dict(linear_dtype=FP8, device=device), dict(linear_dtype=FP8, device=device, plan_only=True)):
        with pytest.raises(ValueError, match="on the CPU"):
            build_tiny("llama", dims=DIMS, **kw)
    assert ft.from_dims(DIMS, arch="llama", optimizer=ft.AdamW(lr=1e-3), max_seq_len=128, max_global_batch_tokens=256, device=device,
                        max_gpu_mem_bytes=64 << 30, max_host_mem_bytes=8 << 30, linear_dtype=FP8, plan_only=True) is not None
