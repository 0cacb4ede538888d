"""Models whose products run in 8 bits on the GPU: every product of a training step, with the operands and views that the layers
hand it, against 64 bits; every family on the package's kernels."""
import pytest
import torch

import flextrain_b200 as ft
from flextrain_b200 import ops
from conftest import build_tiny

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
DIMS = dict(vocab_size=512, n_layers=2, d_model=512, n_heads=4, n_kv_heads=2, head_dim=128, expert_dim=1152, num_routed_experts=0,
            num_shared_experts=0, top_k=0, is_causal=True)
MOE = dict(DIMS, expert_dim=256, num_routed_experts=8, top_k=2)


def _model(arch, dims, **kw):
    ws = ft.WorkingSetConfig.simple(max_seq_len=160, max_global_batch_tokens=640, chunk=320)
    return build_tiny(arch, dims=dims, device="cuda:0", dtype=torch.bfloat16, max_seq_len=160, batch_tokens=640, ws=ws, **kw)


@pytest.mark.parametrize("arch,dims,kw", [("llama", DIMS, {}), ("qwen3", DIMS, {}), ("gemma2", DIMS, {}), ("qwen3_moe", MOE, {}),
                                          ("llama", DIMS, dict(lora_targets="all", lora_rank=16)),
                                          ("llama", DIMS, dict(force_saved_act_level=0))])
def test_training_step(monkeypatch, arch, dims, kw):
    """The sums of a product of K terms: 2^-24 for each block of 128 and 128 * 2^-23 in a block, of the terms' magnitudes; the result's
    rounding 2^-8 of it, of what is added to it included."""
    seen = {"fwd": 0, "dgrad": 0, "wgrad": 0}
    real = ops.gemm_fp8

    def checked(a, b, *, trans_a=False, trans_b=False, alpha=1.0, beta=0.0, c=None, bias=None, out=None, out_dtype=None):
        A, B = (ops.dequant_fp8(m, torch.float32).double() for m in (a, b))
        A, B = A.t() if trans_a else A, B.t() if trans_b else B
        add = (c if c is not None else out).double().clone() * beta if beta else torch.zeros((), device="cuda")
        add = add + (bias.double() if bias is not None else 0)
        got = real(a, b, trans_a=trans_a, trans_b=trans_b, alpha=alpha, beta=beta, c=c, bias=bias, out=out, out_dtype=out_dtype)
        want, mag = alpha * A @ B + add, abs(alpha) * A.abs() @ B.abs() + add.abs()
        room = 2.0 ** -8 * want.abs() + (2.0 ** -16 + (A.shape[1] / 128 + 6) * 2.0 ** -24) * mag
        assert got.shape == want.shape and torch.all((got.double() - want).abs() <= room)
        seen["wgrad" if trans_a else "fwd" if trans_b else "dgrad"] += 1
        return got

    am = _model(arch, dims, linear_dtype=FP8, **kw)
    seqs = ft.SyntheticTokenSource(512, 160, seed=0).get_sequences(640)
    am.fwd_bwd(seqs)
    am.step()
    monkeypatch.setattr(ops, "gemm_fp8", checked)
    ops.reset_backends_used()
    st = am.fwd_bwd(seqs)
    used = ops.backends_used()
    for family in ("quant_fp8", "gemm_fp8") + (("grouped_gemm_fp8", "grouped_wgrad_fp8") if dims is MOE else ("rmsnorm_fp8_fwd",)):
        assert used[family] == ["ftb"], used
    products = 2 * 2 * (2 if dims is MOE else 4)                   # layers, chunks, projections
    assert seen["fwd"] >= products and seen["dgrad"] == products
    assert seen["wgrad"] == (0 if "lora_targets" in kw else products)
    assert st.loss == st.loss and am.step() == 0
    for scope, l, name, t in am.named_master_params():
        assert torch.isfinite(t).all(), (scope, l, name)
    from flextrain_b200.ops.cuda import device_error_words
    torch.cuda.synchronize()
    assert device_error_words().get("gemm_fp8", 0) == 0


@pytest.mark.parametrize("arch,dims", [("llama", DIMS), ("qwen3_moe", MOE)])
def test_steps_are_the_same_twice(arch, dims):
    """Nothing depends on an order of additions: two models from one seed stay the same to the bit."""
    a, b = _model(arch, dims, linear_dtype=FP8), _model(arch, dims, linear_dtype=FP8)
    seqs = ft.SyntheticTokenSource(512, 160, seed=0).get_sequences(640)
    for _ in range(2):
        assert a.fwd_bwd(seqs).loss == b.fwd_bwd(seqs).loss
        for (_, l, name, _), (scope, _, _, _) in zip(a.named_master_params(), b.named_master_params()):
            if scope == "layer" and name.startswith("w_") and "norm" not in name:
                assert torch.equal(a.buffers.grads(l)["g_" + name[2:]], b.buffers.grads(l)["g_" + name[2:]]), (l, name)
        a.step(), b.step()
