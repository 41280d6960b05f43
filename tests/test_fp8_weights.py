"""8-bit weights without a GPU: kernels stand in for themselves, what is looked at is when rows are made, from what, and what is held meanwhile."""
import gc
import os

import pytest
import torch

import fp8_reference as R


@pytest.fixture
def kernels(monkeypatch):
    """Quantisation in torch operations, the products by names alone -> the list of what was called."""
    from flash_stu_2_b200 import ops
    calls = []

    def quantize(w):
        calls.append("quantize")
        q, e = R.quantize(w.double())
        return ops.Fp8Rows(q.to(torch.float8_e4m3fn), R.pieces((e + 127).to(torch.uint8)).view(torch.float8_e8m0fnu), w.shape[1])

    def linear(x, W, *, W2=None, resid=None, out=None, overlap=False):
        calls.append(overlap)
        return x if W2 is not None else resid

    class Stream:
        def synchronize(self):
            calls.append("wait")

    monkeypatch.setattr(ops, "quantize_fp8", quantize)
    monkeypatch.setattr(ops, "rmsnorm_fp8", lambda x, w, eps, add=None: x)
    monkeypatch.setattr(ops, "linear_fp8", linear)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: Stream())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return calls


def make(**kw):
    """-> an MLP in 8 bits of width 32"""
    import flash_stu_2_b200 as F
    cfg = F.FlashSTUConfig(**{**dict(n_embd=32, n_layers=2, n_heads=4, seq_len=64, window_size=8, vocab_size=97, mlp_scale=4, num_eigh=8,
                                     torch_dtype=torch.bfloat16, mlp_fp8=True), **kw})
    return F.Fp8MLP(cfg, dtype=torch.bfloat16)


def step(mlp, calls):
    del calls[:]
    x = torch.zeros(1, 32, dtype=torch.bfloat16)
    mlp.apply_residual(x, x, x, norm_w=torch.ones(32, dtype=torch.bfloat16), overlap=True)
    return list(calls)


def of(mlp, k=1):
    return mlp.rows()[k].dequantize()


def test_an_mlp_made_and_moved_in_inference_mode(kernels):
    """Its parameters tell of their changes as any others do: rows are made once, and again behind a change."""
    with torch.inference_mode():
        mlp = make().to(torch.float64).to(torch.bfloat16)
    assert step(mlp, kernels) == ["quantize"] * 3 + ["wait", True, True] and step(mlp, kernels) == [True, True]
    before = of(mlp).clone()
    with torch.inference_mode():
        mlp.load_state_dict({k: 2 * v for k, v in mlp.state_dict().items()})
        assert torch.equal(of(mlp), 2 * before)
    with torch.no_grad():
        mlp.up_proj.weight.mul_(2)
    assert torch.equal(of(mlp), 4 * before)


@pytest.mark.parametrize("how", ["replaced", "assigned", "data"])
def test_parameters_that_do_not_tell_of_their_changes(kernels, how):
    """Inference tensors have no version: every call makes its rows from what they hold, in front of its products, and keeps none."""
    mlp = make()
    with torch.inference_mode():
        state = {k: v.clone() for k, v in mlp.state_dict().items()}
        if how == "replaced":
            mlp.up_proj.weight = torch.nn.Parameter(state["up_proj.weight"])
        elif how == "assigned":
            mlp.load_state_dict(state, assign=True)
        else:
            mlp.up_proj.weight.data = state["up_proj.weight"]
    assert step(mlp, kernels) == ["quantize"] * 3 + [False, False] == step(mlp, kernels)
    before = of(mlp).clone()
    with torch.inference_mode():
        mlp.up_proj.weight.mul_(2)
    assert torch.equal(of(mlp), 2 * before)
    with torch.inference_mode():
        mlp.up_proj.weight.mul_(2)
        assert torch.equal(of(mlp), 4 * before)
