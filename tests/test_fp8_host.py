"""8-bit rows without a GPU: the layout, what is refused, and the reference that the GPU tests compare with."""
import torch
import pytest

import fp8_reference as R


def made(rows, cols, seed=0):
    from flash_stu_2_b200 import ops
    g = torch.Generator().manual_seed(seed)
    q, e = R.quantize((torch.randn(rows, cols, generator=g) * torch.exp2(torch.randint(-20, 20, (rows, 1), generator=g).float())).double())
    return ops.Fp8Rows(q.to(torch.float8_e4m3fn), R.pieces((e + 127).to(torch.uint8)).view(torch.float8_e8m0fnu), cols)


@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 300), (128, 512), (131, 1111)])
def test_layout(rows, cols):
    r = made(rows, cols)
    r_scales = r.scales.view(torch.uint8)
    plain = r.block_scales()
    assert plain.shape == (rows, (cols + 127) // 128) and r.shape == (rows, cols) and r.dequantize().shape == (rows, cols)
    for row in {0, rows // 2, rows - 1}:
        for k in {0, plain.shape[1] - 1}:
            byte = int(r_scales[row // 128, k // 4, row % 32, row // 32 % 4, k % 4])
            assert float(plain[row, k]) == 2.0 ** (byte - 127)
    assert torch.equal(R.values(r), r.dequantize().double())


def test_reference_quantisation_is_the_nearest():
    """Against every number of the format: the scale is the smallest that fits, each value goes to the nearest, ties to the even one."""
    g = torch.Generator().manual_seed(1)
    v = (torch.randn(20, 256, generator=g).double() * 10).float().double()
    v[0, 0], v[1, :128] = 448.0, 0.0
    q, e = R.quantize(v)
    numbers = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    order = numbers[~numbers.isnan()].unique()
    top = R.blocks(v.abs()).amax(2)
    assert bool((top <= 448 * R.power(e)).all()) and bool(((top > 224 * R.power(e)) | (e == -127)).all())
    z = (R.blocks(v) * R.power(-e)[:, :, None]).reshape(-1, 1)
    assert bool(((q.reshape(-1, 1) - z).abs() <= (order[None] - z).abs().amin(1, keepdim=True)).all())


def test_check_rows_notices():
    """A wrong value, a wrong scale and a byte where no row is do not pass."""
    from flash_stu_2_b200 import ops
    g = torch.Generator().manual_seed(2)
    v = torch.randn(9, 200, generator=g).double()
    q, e = R.quantize(v.float().double())

    def rows(q=q, e=e, touch=None):
        s = R.pieces((e + 127).to(torch.uint8))
        if touch:
            s[touch] = 100
        return ops.Fp8Rows(q.to(torch.float8_e4m3fn), s.view(torch.float8_e8m0fnu), 200)

    R.check_rows(rows(), v, v.abs() * 2.0 ** -20)
    wrong = q.clone()
    wrong[3, 7] *= 1.25
    for bad in (rows(wrong), rows(q / 2, e + 1), rows(touch=(0, 0, 9, 0, 0)), rows(touch=(0, 0, 0, 0, 2))):
        with pytest.raises(AssertionError):
            R.check_rows(bad, v, v.abs() * 2.0 ** -20)


def test_no_cpu_path():
    from flash_stu_2_b200 import ops
    x = torch.zeros(2, 256)
    r = made(2, 256)
    for call in (lambda: ops.quantize_fp8(x), lambda: ops.rmsnorm_fp8(x, x[0]), lambda: ops.linear_fp8(r, r), lambda: ops.linear_fp8(r, r, W2=r)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(ValueError, match="contiguous rows of 250"):
        ops.linear_fp8(ops.Fp8Rows(r.data, r.scales[:, :0], 250), r)
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        ops.linear_fp8(ops.Fp8Rows(x, r.scales, 256), r)


def test_argument_errors_of_the_library():
    """Checked on the host before any CUDA call; the addresses are dummies."""
    from flash_stu_2_b200 import _lib
    lib, a = _lib.load(), 0x10000
    assert lib.stu_quantize_fp8(None, a, a, 1, 128, 128, 1, None) == -5
    assert lib.stu_quantize_fp8(a, a, a, 1, 0, 128, 1, None) == -2 and lib.stu_quantize_fp8(a, a, a, -1, 128, 128, 1, None) == -2
    assert lib.stu_quantize_fp8(a, a + 8, a, 1, 128, 128, 1, None) == -3 and lib.stu_quantize_fp8(a, a, a, 1, 128, 128, 2, None) == -1
    assert lib.stu_quantize_fp8(a, a, a, 0, 128, 128, 1, None) == 0
    assert lib.stu_rmsnorm_fp8(a, a, a, None, a, a, 1, 128, 128, 128, 128, 1e-6, 1, None) == -5
    assert lib.stu_rmsnorm_fp8(a, None, a, None, a, a, 1, 32769, 32769, 0, 0, 1e-6, 1, None) == -2
    assert lib.stu_rmsnorm_fp8(a, None, a, None, a, a + 4, 1, 128, 128, 0, 0, 1e-6, 1, None) == -3
    args = lambda **k: [{**dict(x=a, xs=a, w=a, ws=a, w2=None, w2s=None, r=None, ldr=0, y=a, ldy=8, ys=None, M=4, N=8, K=128, flags=0, st=None), **k}[n]
                        for n in ("x", "xs", "w", "ws", "w2", "w2s", "r", "ldr", "y", "ldy", "ys", "M", "N", "K", "flags", "st")]
    call = lambda **k: lib.stu_linear_fp8(*args(**k))
    assert call(xs=None) == -5 and call(w2=a) == -5 and call(w2=a, w2s=a) == -5
    assert call(N=0) == -2 and call(K=0) == -2 and call(M=-1) == -2 and call(K=2 ** 31 - 100) == -2
    assert call(w2=a, w2s=a, ys=a, r=a) == -4 and call(flags=1) == -4
    assert call(ws=a + 4) == -3 and call(w2=a, w2s=a, ys=a, y=a + 8) == -3
    assert call(M=0) == 0


def _config(tmp_path, **kw):
    import os
    import flash_stu_2_b200 as F
    path = os.path.join(tmp_path, "phi.pt")
    F.save_spectral_filters(F.get_spectral_filters(64, 8, dtype=torch.float32, device="cpu"), path, metadata={"seq_len": 64, "K": 8})
    return F.FlashSTUConfig(**{**dict(n_embd=32, n_layers=4, n_heads=4, seq_len=64, window_size=8, vocab_size=97, mlp_scale=4, num_eigh=8,
                                      torch_dtype=torch.bfloat16, filter_path=path), **kw})


def test_models_with_an_8_bit_mlp(tmp_path):
    """The switch is the configuration's, survives a round trip, changes no checkpoint, and bfloat16 alone has it."""
    import flash_stu_2_b200 as F
    from flash_stu_2_b200.token_step import layer_supported
    plain, cfg = _config(str(tmp_path)), _config(str(tmp_path), mlp_fp8=True)
    assert not plain.mlp_fp8 and cfg.mlp_fp8 and F.FlashSTUConfig.from_dict(cfg.to_dict()).mlp_fp8 and not F.FlashSTUConfig.from_dict(plain.to_dict()).mlp_fp8
    a, b = F.FlashSTU(plain), F.FlashSTU(cfg)
    assert all(type(layer.mlp) is F.MLP for layer in a.layers) and all(type(layer.mlp) is F.Fp8MLP for layer in b.layers)
    assert list(a.state_dict()) == list(b.state_dict())
    b.load_state_dict(a.state_dict())
    assert all(layer_supported(layer) for layer in a.layers) and not any(layer_supported(layer) for layer in b.layers)
    assert type(F.FlashSTUBlock(d_model=64, sequence_length=128, num_filters=8, mlp_fp8=True).layer.mlp) is F.Fp8MLP
    assert type(F.FlashSTUBlock(d_model=64, sequence_length=128, num_filters=8).layer.mlp) is F.MLP
    with pytest.raises(NotImplementedError, match="bfloat16"):
        F.FlashSTU(_config(str(tmp_path), mlp_fp8=True, torch_dtype=torch.float32))


def test_tensor_parallelism_refuses_an_8_bit_mlp(tmp_path):
    import torch.distributed as dist
    from flash_stu_2_b200.tensor_parallel import TensorParallelFlashSTU
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/rendezvous", rank=0, world_size=1)
    try:
        with pytest.raises(NotImplementedError, match="8 bits"):
            TensorParallelFlashSTU(_config(str(tmp_path), mlp_fp8=True), {}, "cpu")
    finally:
        dist.destroy_process_group()


def test_addresses_inside_of_an_element_are_refused():
    from flash_stu_2_b200 import _lib
    lib, a = _lib.load(), 0x10000
    assert lib.stu_quantize_fp8(a + 1, a, a, 1, 128, 128, 1, None) == -3 and lib.stu_quantize_fp8(a + 2, a, a, 1, 128, 128, 0, None) == -3
    for k in range(4):   # x, add, w, sum
        p = [a] * 4
        p[k] += 1
        assert lib.stu_rmsnorm_fp8(*p, a, a, 1, 128, 128, 128, 128, 1e-6, 1, None) == -3
    assert lib.stu_linear_fp8(a, a, a, a, None, None, None, 0, a + 1, 8, None, 4, 8, 128, 0, None) == -3
    assert lib.stu_linear_fp8(a, a, a, a, None, None, a + 1, 8, a, 8, None, 4, 8, 128, 0, None) == -3


def test_linear_takes_8_bit_rows():
    from flash_stu_2_b200 import ops
    r, t = made(2, 256), torch.zeros(2, 256)
    for call in (lambda: ops.linear_fp8(t, r), lambda: ops.linear_fp8(r, t), lambda: ops.linear_fp8(r, r, W2=t)):
        with pytest.raises(TypeError, match="Fp8Rows"):
            call()


def test_when_8_bit_weights_are_made(tmp_path, monkeypatch):
    """Their kernels stand in for themselves: what is made when, that it is there before anyone reads it ahead of the kernel in front, and what a capture keeps."""
    import copy
    import pickle
    import flash_stu_2_b200 as F
    from flash_stu_2_b200 import ops
    calls, capturing = [], [False]

    class Stream:
        def synchronize(self):
            calls.append("wait")

    def quantize(w):
        calls.append("quantize")
        q, e = R.quantize(w.double())
        return ops.Fp8Rows(q.to(torch.float8_e4m3fn), R.pieces((e + 127).to(torch.uint8)).view(torch.float8_e8m0fnu), w.shape[1])

    def linear(x, W, *, W2=None, resid=None, out=None, overlap=False):
        calls.append(overlap)
        return x if W2 is not None else resid

    monkeypatch.setattr(ops, "quantize_fp8", quantize)
    monkeypatch.setattr(ops, "rmsnorm_fp8", lambda x, w, eps, add=None: x)
    monkeypatch.setattr(ops, "linear_fp8", linear)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: Stream())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    mlp = F.FlashSTU(_config(str(tmp_path), mlp_fp8=True)).layers[0].mlp
    x, norm = torch.zeros(1, 32, dtype=torch.bfloat16), torch.ones(32, dtype=torch.bfloat16)

    def step():
        del calls[:]
        mlp.apply_residual(x, x, x, norm_w=norm, overlap=True)
        return list(calls)

    made, kept = ["quantize"] * 3, [True, True]
    capturing[0] = True
    assert step() == made + [False, False] == step() and mlp._rows is None   # the graph's own, never read ahead of the kernels that make them
    capturing[0] = False
    assert step() == made + ["wait"] + kept and step() == kept
    rows = mlp.rows()
    capturing[0] = True
    assert step() == kept
    capturing[0] = False
    with torch.no_grad():
        mlp.up_proj.weight.mul_(2)
    before = rows[1].dequantize().clone()
    assert step() == made + ["wait"] + kept and mlp.rows()[1] is rows[1] and torch.equal(rows[1].dequantize(), 2 * before)   # in place
    mlp.up_proj.weight.data.mul_(2)   # (leaves no trace)
    assert step() == kept
    mlp.rows(again=True)
    assert torch.equal(rows[1].dequantize(), 4 * before)
    with torch.no_grad():
        mlp.gate_proj.weight.data = mlp.gate_proj.weight.data.t().contiguous().t()   # the same numbers elsewhere
    assert step() == made + ["wait"] + kept
    mlp.down_proj.weight = torch.nn.Parameter(torch.zeros(32, 64, dtype=torch.bfloat16))
    assert step() == made + ["wait"] + kept and mlp.rows()[2].shape == (32, 64)
    for other in (copy.deepcopy(mlp), pickle.loads(pickle.dumps(mlp))):
        assert other._rows is None and mlp._rows is not None
        assert other.rows()[0] is not mlp.rows()[0] and torch.equal(other.rows()[0].dequantize(), mlp.rows()[0].dequantize())
    with pytest.raises(ValueError, match="norm_w"):
        mlp.apply_residual(x, x, x, add=x)


def test_a_weight_at_the_address_of_one_that_is_gone(tmp_path, monkeypatch):
    """The weights that rows were made from are kept with their addresses: nothing else is ever there."""
    import weakref
    import flash_stu_2_b200 as F
    from flash_stu_2_b200 import ops
    monkeypatch.setattr(ops, "quantize_fp8", lambda w: ops.Fp8Rows(w[:1, :1].clone(), torch.zeros(1), w.shape[1]))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: type("S", (), {"synchronize": lambda self: None})())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    mlp = F.FlashSTU(_config(str(tmp_path), mlp_fp8=True)).layers[0].mlp
    for value in range(8):
        mlp.up_proj.weight.data = torch.empty(0, dtype=torch.bfloat16)
        mlp.up_proj.weight.data = torch.full((128, 32), float(value), dtype=torch.bfloat16)
        assert bool((mlp.rows()[1].data == value).all())
    gone = weakref.ref(mlp)
    del mlp
    import gc
    gc.collect()
    assert gone() is None


def test_the_device_that_is_launched_on(monkeypatch):
    from types import SimpleNamespace
    from flash_stu_2_b200 import ops
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    on = lambda i: SimpleNamespace(device=torch.device("cuda", i))
    assert ops._elsewhere(on(0), None, on(0)) is None
    assert ops._elsewhere(on(1), None, on(1)) == torch.device("cuda", 1)
    with pytest.raises(RuntimeError, match="several devices"):
        ops._elsewhere(on(0), on(1))


def test_8_bit_weights_made_in_inference_mode(tmp_path, monkeypatch):
    """What a call in inference mode made is renewed by one outside of it, and the other way around."""
    import flash_stu_2_b200 as F
    from flash_stu_2_b200 import ops
    monkeypatch.setattr(ops, "quantize_fp8", lambda w: ops.Fp8Rows(w.float().clone(), torch.zeros(1), w.shape[1]))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: type("S", (), {"synchronize": lambda self: None})())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    mlp = F.FlashSTU(_config(str(tmp_path), mlp_fp8=True)).layers[0].mlp
    for first, then in ((torch.inference_mode, torch.no_grad), (torch.no_grad, torch.inference_mode)):
        with first():
            before = mlp.rows()[0].data.clone()
        with torch.no_grad():
            mlp.gate_proj.weight.mul_(2)
        with then():
            assert torch.equal(mlp.rows()[0].data, 2 * before)
