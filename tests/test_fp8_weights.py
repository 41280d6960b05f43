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


def stored(t):
    """Tells whether a tensor's memory is still somebody's."""
    import weakref
    return weakref.ref(t.untyped_storage())


def alive(refs):
    gc.collect()
    return [r() is not None for r in refs]


def test_a_model_that_leaves_a_device_holds_nothing_there(kernels):
    """Neither the weights that rows were made from nor the rows; a move that changes nothing keeps both."""
    mlp = make()
    rows = mlp.rows()
    refs = [stored(p.data) for p in mlp.parameters()] + [stored(t) for r in rows for t in (r.data, r.scales)]
    mlp.to("cpu")
    assert mlp.rows() is rows and alive(refs) == [True] * 9
    del rows
    mlp.to("meta")
    assert alive(refs) == [False] * 9


@pytest.mark.parametrize("how", ["assigned", "replaced", "data", "type"])
def test_weights_that_are_replaced_are_not_held(kernels, how):
    """Not until the next call, and not while that makes the rows of their successors; the rows stay where they are."""
    mlp = make()
    rows = mlp.rows()
    before = of(mlp).clone()
    old = stored(mlp.up_proj.weight.data)
    twice = (2 * mlp.up_proj.weight.detach()).clone()
    if how == "assigned":
        mlp.load_state_dict({**{k: v.clone() for k, v in mlp.state_dict().items()}, "up_proj.weight": twice}, assign=True)
    elif how == "replaced":
        mlp.up_proj.weight = torch.nn.Parameter(twice)
    elif how == "data":
        mlp.up_proj.weight.data = twice
    else:
        twice = mlp.to(torch.float32).up_proj.weight.detach().mul_(2)
    assert alive([old]) == [False]
    assert mlp.rows()[1] is rows[1] and torch.equal(of(mlp), 2 * before)


def test_one_matrix_at_a_time(kernels, monkeypatch):
    """A renewal has the new rows of one matrix beside the old ones of all."""
    from flash_stu_2_b200 import ops
    made, most, quantize = [], [0], ops.quantize_fp8

    def counted(w):
        r = quantize(w)
        made.append(stored(r.data))
        most[0] = max(most[0], sum(alive(made)))
        return r

    monkeypatch.setattr(ops, "quantize_fp8", counted)
    mlp = make()
    mlp.rows()
    most[0] = 0
    with torch.no_grad():
        mlp.up_proj.weight.mul_(2)
    mlp.rows()
    assert most[0] == 3 + 1


def test_another_weight_in_the_same_memory(kernels):
    """Told by what holds the memory, not by its address: a new weight where one that is gone was."""
    mlp = make()
    held = mlp.up_proj.weight.data
    first = of(mlp).clone()
    memory = held.untyped_storage()
    # another tensor over the same bytes: the same storage, the same version
    mlp.up_proj.weight.data = held.view(128, 32)
    assert mlp.rows()[1] is mlp.rows()[1] and torch.equal(of(mlp), first)
    del held, memory
    for value in range(8):
        mlp.up_proj.weight.data = torch.empty(0, dtype=torch.bfloat16)
        mlp.up_proj.weight.data = torch.full((128, 32), 2.0 ** value, dtype=torch.bfloat16)
        assert bool((of(mlp) == 2.0 ** value).all())


def test_a_first_call_that_fails_leaves_nothing_behind(kernels, monkeypatch):
    """Rows of which one could not be made are no model's rows: the next call makes them all."""
    from flash_stu_2_b200 import ops
    mlp = make()
    first = of(mlp).clone()
    quantize, left = ops.quantize_fp8, [1]

    def fails(w):
        if left[0] == 0:
            raise torch.OutOfMemoryError("no room")
        left[0] -= 1
        return quantize(w)

    with torch.no_grad():
        for p in mlp.parameters():
            p.mul_(2)
    monkeypatch.setattr(ops, "quantize_fp8", fails)
    with pytest.raises(torch.OutOfMemoryError):
        mlp.rows()
    monkeypatch.setattr(ops, "quantize_fp8", quantize)
    assert torch.equal(of(mlp), 2 * first) and torch.equal(of(mlp, 2), R.values(quantize(mlp.down_proj.weight.detach())).float())


def test_first_calls_of_two_threads(kernels, monkeypatch):
    """Both get the rows that are kept: a graph that one of them captures next reads memory that stays."""
    import threading
    from flash_stu_2_b200 import ops
    quantize, inside, go = ops.quantize_fp8, threading.Semaphore(0), threading.Event()

    def slow(w):
        inside.release()
        go.wait(10)
        return quantize(w)

    monkeypatch.setattr(ops, "quantize_fp8", slow)
    mlp, got = make(), []
    threads = [threading.Thread(target=lambda: got.append(mlp.rows())) for _ in range(2)]
    threads[0].start()
    assert inside.acquire(timeout=10)
    threads[1].start()
    inside.acquire(timeout=0.5)   # (the second one is inside too, or waits)
    go.set()
    for t in threads:
        t.join()
    assert got[0] is got[1] is mlp.rows()
