"""Rings of 4 bits and packed prompts without a GPU: the layout, what is refused, and the reference that the GPU tests compare with."""
import math

import pytest
import torch

import kv4_reference as R


@pytest.mark.parametrize("hd", [8, 40, 64, 72, 128])
def test_reference_numbers_are_near(hd):
    """Every value is at most half a step off, the step at most 1/15 of the range and of what rounding lowest and step adds to it."""
    g = torch.Generator().manual_seed(hd)
    x = (torch.randn(300, hd, generator=g) * torch.exp2(torch.randint(-30, 30, (300, 1), generator=g).float()) + 3 * torch.randn(300, 1, generator=g)).double()
    for piece in x.split(64, -1):
        low, step, n = R.numbers(piece)
        assert bool((low <= piece.amin(-1, keepdim=True)).all()) and bool(((n >= 0) & (n <= 15)).all())
        assert bool(((low + step * n - piece).abs() <= step * (0.5 + 2.0 ** -18)).all())
        lo, hi = piece.amin(-1, keepdim=True), piece.amax(-1, keepdim=True)
        assert bool((step <= ((hi - lo) + lo.abs() * 2.0 ** -7) / 15 * (1 + 2.0 ** -7) + 2.0 ** -126).all())


def test_reference_layout():
    """Bytes and values are each other's inverse, and lie where the layout says."""
    g = torch.Generator().manual_seed(1)
    for hd in (8, 32, 48, 64, 80, 128):
        x = torch.randn(2, 3, 32, hd, generator=g)
        ring = R.ring_bytes(x)
        assert ring.shape == (2, 3, 32 * {32: 20, 64: 36, 128: 72}[R.width(hd)])
        assert torch.equal(R.values(ring, hd), R.held(x))
    words = ring.view(torch.int32)[1, 2, 5 * 16:6 * 16]            # slot 5 of heads of 128: 16 words
    _, _, n = R.numbers(x[1, 2, 5, 64:].double())
    assert [int(words[2 * 3 + 1]) >> 4 * s & 15 for s in range(8)] == n[24:32].long().tolist()


def test_reference_specials():
    for special in (math.nan, math.inf, -math.inf):
        x = torch.randn(1, 128)
        x[0, 70] = special
        back = R.held(x)
        assert bool(back[0, 64:].isnan().all()) and bool(back[0, :64].isfinite().all())
    x = torch.full((1, 64), 3.0e38)
    x[0, 0] = -3.0e38                                               # a range past fp32's
    assert bool(R.held(x).isnan().all())
    assert torch.equal(R.held(torch.full((1, 24), -0.1875)), torch.full((1, 24), -0.1875, dtype=torch.float64))


def test_check_notices():
    out = torch.zeros(3, 4, dtype=torch.float64)
    R.check(out.float(), out, out + 1e-9)
    for bad in (out + 1e-3, torch.full((3, 4), math.nan, dtype=torch.float64)):
        with pytest.raises(AssertionError):
            R.check(bad.float(), out, out + 1e-9)


def test_no_cpu_path():
    from flash_stu_2_b200 import ops
    k4, v4 = ops.kv4_rings(2, 32, 1, 64, "cpu")
    qkv, pos, cu = torch.zeros(2, 1, 4 * 64), torch.zeros(2, 2, dtype=torch.int32), torch.tensor([0, 1, 2], dtype=torch.int32)
    for call in (lambda: ops.swa_packed(qkv[:, 0], cu, None, 2, kv_heads=1), lambda: ops.kv4_write(qkv, k4, v4, pos, 2),
                 lambda: ops.kv4_write(qkv[:, 0], k4, v4, pos, 2, cu_seqlens=cu), lambda: ops.kv4_read(k4, v4, 64, torch.float32),
                 lambda: ops.kv4_step(qkv, k4, v4, pos, None, 2, 31)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_kv4_rings():
    from flash_stu_2_b200 import ops
    for hd, row in ((8, 20), (32, 20), (40, 36), (64, 36), (72, 72), (128, 72)):
        k4, v4 = ops.kv4_rings(3, 48, 2, hd, "cpu")
        assert k4.shape == v4.shape == (3, 2, 48 * row) and k4.dtype == torch.uint8 and not bool(k4.any())
    assert [ops.kv4_slots(w) for w in (0, 1, 15, 16, 1024, 1039)] == [16, 16, 16, 32, 1040, 1040]
    for bad in ((2, 40, 1, 64), (2, 0, 1, 64), (2, 16, 0, 64)):
        with pytest.raises(ValueError):
            ops.kv4_rings(*bad, "cpu")
    for hd in (0, 4, 20, 136):
        with pytest.raises(NotImplementedError):
            ops.kv4_rings(2, 32, 1, hd, "cpu")


def test_refusals():
    from flash_stu_2_b200 import ops
    k4, v4 = ops.kv4_rings(2, 32, 1, 64, "cpu")
    qkv, pos, cu = torch.zeros(2, 1, 4 * 64), torch.zeros(2, 2, dtype=torch.int32), torch.tensor([0, 1, 2], dtype=torch.int32)
    slopes = torch.zeros(2)

    def step(qkv=qkv, k4=k4, v4=v4, pos=pos, slopes=slopes, H=2, window=31, softcap=0.0):
        ops.kv4_step(qkv, k4, v4, pos, slopes, H, window, softcap)

    def write(qkv=qkv, k4=k4, v4=v4, pos=pos, H=2, cu=None):
        ops.kv4_write(qkv, k4, v4, pos, H, cu_seqlens=cu)

    def packed(qkv=qkv[:, 0], cu=cu, slopes=slopes, H=2, window=None, softcap=0.0, kv_heads=1, out=None):
        ops.swa_packed(qkv, cu, slopes, H, window, softcap, kv_heads, out)

    cases = [
        (TypeError, lambda: step(qkv=qkv.half())), (TypeError, lambda: step(k4=k4.int())), (TypeError, lambda: step(pos=pos.long())),
        (ValueError, lambda: step(qkv=qkv[:1])), (ValueError, lambda: step(qkv=qkv[:, 0])), (ValueError, lambda: step(qkv=torch.zeros(2, 2, 256))),
        (ValueError, lambda: step(H=3)), (ValueError, lambda: step(k4=k4[:, :, :-36], v4=v4[:, :, :-36])), (ValueError, lambda: step(v4=v4[:1])),
        (ValueError, lambda: step(k4=k4[0], v4=v4[0])), (ValueError, lambda: step(window=32)), (ValueError, lambda: step(window=-1)),
        (ValueError, lambda: step(softcap=-1.0)), (ValueError, lambda: step(softcap=math.inf)), (ValueError, lambda: step(softcap=math.nan)),
        (ValueError, lambda: step(slopes=slopes.double())), (ValueError, lambda: step(slopes=torch.zeros(3))), (ValueError, lambda: step(pos=pos[:1])),
        (ValueError, lambda: step(pos=torch.zeros(2, 4, dtype=torch.int32)[:, ::2])), (NotImplementedError, lambda: step(qkv=torch.zeros(2, 1, 4 * 60))),
        (NotImplementedError, lambda: step(qkv=torch.zeros(2, 1, 4 * 144))),
        (ValueError, lambda: write(qkv=qkv[:, 0])), (ValueError, lambda: write(cu=cu)), (ValueError, lambda: write(qkv=qkv[:, 0], cu=cu[:2])),
        (TypeError, lambda: write(qkv=qkv[:, 0], cu=cu.long())), (ValueError, lambda: write(qkv=torch.zeros(3, 1, 256))), (ValueError, lambda: write(H=0)),
        (TypeError, lambda: write(qkv=qkv.double())), (ValueError, lambda: write(k4=k4[0])),
        (TypeError, lambda: packed(qkv=qkv[:, 0].half())), (ValueError, lambda: packed(qkv=qkv)), (ValueError, lambda: packed(kv_heads=0)),
        (ValueError, lambda: packed(kv_heads=3)), (ValueError, lambda: packed(H=3)), (TypeError, lambda: packed(cu=cu.long())),
        (ValueError, lambda: packed(cu=cu[None])), (ValueError, lambda: packed(cu=cu[:0])), (ValueError, lambda: packed(window=-1)),
        (ValueError, lambda: packed(softcap=-2.0)), (ValueError, lambda: packed(softcap=math.nan)), (ValueError, lambda: packed(slopes=slopes[:1])),
        (ValueError, lambda: packed(qkv=torch.zeros(2, 4 * 160))), (ValueError, lambda: packed(out=torch.zeros(2, 64))),
        (ValueError, lambda: packed(out=torch.zeros(2, 128, dtype=torch.bfloat16))), (ValueError, lambda: packed(out=torch.zeros(128, 2).T)),
        (ValueError, lambda: packed(cu=torch.zeros(6, dtype=torch.int32)[::2])),
        (TypeError, lambda: ops.kv4_read(k4, v4, 64, torch.float16)), (ValueError, lambda: ops.kv4_read(k4, v4, 32, torch.float32)),
        (NotImplementedError, lambda: ops.kv4_read(k4, v4, 12, torch.float32)),
    ]
    for error, call in cases:
        with pytest.raises(error):
            call()


def test_argument_errors_without_a_gpu():
    from flash_stu_2_b200 import _lib
    lib = _lib.load()
    a = 0x10000   # stands for an aligned device address; the checks return before anything dereferences it
    assert lib.stu_kv4_step(None, 512, a, a, a, None, a, 1, 2, 1, 64, 16, 15, 0.0, 1, None, 1, None) == -5
    assert lib.stu_kv4_step(a, 512, a, a, a, None, a, 1, 2, 1, 64, 16, 16, 0.0, 1, None, 1, None) == -2
    assert lib.stu_kv4_step(a, 512, a, a, a, None, a, 1, 3, 2, 64, 16, 15, 0.0, 1, None, 1, None) == -2
    assert lib.stu_kv4_step(a, 512, a, a, a, None, a, 1, 2, 1, 64, 24, 15, 0.0, 1, None, 1, None) == -2
    assert lib.stu_kv4_step(a, 512, a, a, a, None, a, 1, 2, 1, 60, 16, 15, 0.0, 1, None, 1, None) == -4
    assert lib.stu_kv4_step(a, 512, a, a, a, None, a, 1, 2, 1, 64, 16, 15, 0.0, 1, None, 2, None) == -1
    assert lib.stu_kv4_step(a, 512, a + 4, a, a, None, a, 1, 2, 1, 64, 16, 15, 0.0, 1, None, 1, None) == -3
    assert lib.stu_kv4_write(a, 255, a, a, a, None, 1, 1, 2, 1, 64, 16, 1, None) == -2
    assert lib.stu_kv4_write(a, 256, a, a, a, None, 2, 3, 2, 1, 64, 16, 1, None) == -2
    assert lib.stu_kv4_read(a, a, a + 8, a, 1, 1, 64, 16, 1, None) == -3
    assert lib.stu_swa_packed(a, 255, a, 1, None, a, 128, 5, 2, 1, 64, -1, 0.0, None, 1, None) == -2
    assert lib.stu_swa_packed(a, 256, a, 0, None, a, 128, 5, 2, 1, 64, -1, 0.0, None, 1, None) == -2
    assert lib.stu_swa_packed(a, 800, a, 1, None, a, 400, 5, 2, 1, 200, -1, 0.0, None, 1, None) == -4
    assert lib.stu_swa_packed(a, 256, a, 1, None, None, 128, 5, 2, 1, 64, -1, 0.0, None, 1, None) == -5


def test_models_without_a_gpu(tmp_path):
    import flash_stu_2_b200 as F
    from flash_stu_2_b200.modules import Packed
    from flash_stu_2_b200.token_step import layer_supported

    def config(**kw):
        return F.FlashSTUConfig(**{**dict(n_embd=64, n_heads=4, n_layers=2, seq_len=64, window_size=20, vocab_size=11, mlp_scale=2, num_eigh=4), **kw})

    assert config().kv_bits is None and F.FlashSTUConfig.from_dict(config(kv_bits=4).to_dict()).kv_bits == 4
    attn = F.Attention(config(kv_bits=4))
    k4, v4, pos = attn.new_cache(3, "cpu")
    assert k4.shape == v4.shape == (3, 4, 32 * 20) and pos.shape == (3, 2)
    assert F.FlashSTUBlock(d_model=64, sequence_length=64, num_filters=4, use_attention=True, kv_bits=4).layer.attn.kv_bits == 4
    layer = F.AttentionLayer(config(kv_bits=4))
    assert not layer_supported(layer) and layer_supported(F.AttentionLayer(config()))
    for bad in (dict(kv_bits=8), dict(kv_bits=4, n_embd=48)):
        with pytest.raises(NotImplementedError):
            F.Attention(config(**bad))
    p = Packed([3, 0, 5], "cpu")
    assert p.cu.tolist() == [0, 3, 3, 8] and p.cu.dtype == torch.int32
    for bad in ([], [-1, 2]):
        with pytest.raises(ValueError):
            Packed(bad, "cpu")


def test_tensor_parallelism_refuses_a_cache_in_4_bits(tmp_path):
    import torch.distributed as dist
    import flash_stu_2_b200 as F
    from flash_stu_2_b200.tensor_parallel import TensorParallelFlashSTU
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/rendezvous", rank=0, world_size=1)
    try:
        with pytest.raises(NotImplementedError, match="4 bits"):
            TensorParallelFlashSTU(F.FlashSTUConfig(n_embd=64, n_heads=4, n_layers=2, seq_len=64, window_size=20, vocab_size=11, num_eigh=4, kv_bits=4), {}, "cpu")
    finally:
        dist.destroy_process_group()


def test_rows_of_a_write_stay_below_32_bits():
    from flash_stu_2_b200 import _lib
    lib = _lib.load()
    a = 0x10000   # as above: refused before anything dereferences it (a + 4: were the rows allowed, the ring's alignment would refuse the call)
    most = 0x7ff00000
    assert lib.stu_kv4_write(a, 256, a + 4, a, a, None, 1, most, 2, 1, 64, 16, 1, None) == -3
    assert lib.stu_kv4_write(a, 256, a + 4, a, a, None, 1, most + 1, 2, 1, 64, 16, 1, None) == -2
