"""What the host knows of a cache's positions once its tensors have been made anew (reordered, cloned, joined), and the calls that need them all alike."""
from types import SimpleNamespace

import pytest
import torch

from flash_stu_2_b200 import FlashSTU, modules
from flash_stu_2_b200.modules import STU


def ragged(*t):
    """Positions that nothing is known of on the host, as index_select leaves them."""
    pos = modules.new_pos(len(t), "cpu")
    pos[:, 0] = torch.tensor(t, dtype=torch.int32)
    return pos.index_select(0, torch.arange(len(t)))


def test_the_furthest_position_counts():
    for t in ((5, 250, 7), (250, 5, 7), (3,), (4, 4)):
        pos = ragged(*t)
        assert modules.host_pos(pos) == max(t) and modules.uniform_pos(pos) == (len(set(t)) == 1)
    assert modules.common_pos(ragged(9, 9)) == 9 and modules.common_pos(modules.new_pos(2, "cpu")) == 0
    noted = modules.new_pos(2, "cpu")
    noted._host_t, noted._uniform = 8, False
    for pos in (ragged(9, 8), ragged(0, 1, 0), noted):
        with pytest.raises(ValueError, match="different positions"):
            modules.common_pos(pos)


@pytest.mark.parametrize("t", [(5, 250), (250, 5), (0, 3)])
def test_models_refuse_several_tokens(t):
    model = SimpleNamespace(training=False, config=SimpleNamespace(dropout=0.0), tok_emb=SimpleNamespace(weight=None), layers=())
    ids = SimpleNamespace(is_cuda=True, shape=(2, 3))
    with pytest.raises(ValueError, match="different positions"):
        FlashSTU._backbone(model, ids, [None, (None, ragged(*t))], True)


@pytest.mark.parametrize("t", [(5, 25), (25, 5)])
def test_layers_refuse_one_position_for_all(t):
    """Layers called by themselves: a prefill's histories go where one number says, and so does every step of the full variant and of the single branch."""
    stu = SimpleNamespace(use_approx=True, use_hankel_L=False, capacity=100, K=4, seq_len=100, cache_len=None, Lh=56, prepared=lambda: (None,) * 3,
                          prepared_full=lambda: (None, None))
    x, hist = torch.zeros(2, 3, 8), torch.zeros(2, 8, 2, 56)
    for call in (lambda: STU.add_to_residual(stu, x, x, (hist, ragged(*t))),
                 lambda: STU.layer_prefill(stu, x, (hist, ragged(*t)), True, None, None, None),
                 lambda: STU.full_forward(stu, x, None, x, (hist, ragged(*t))),
                 lambda: STU.full_decode_step(stu, x[:, 0], None, x[:, 0], (hist, ragged(*t)))):
        with pytest.raises(ValueError, match="different positions"):
            call()


def test_the_furthest_position_is_held_to_the_capacity():
    stu = SimpleNamespace(use_approx=True, use_hankel_L=False, capacity=100, seq_len=100, prepared=lambda: (None,) * 3)
    for t in ((100, 5), (5, 100)):
        with pytest.raises(ValueError, match="exceeds the capacity"):
            STU.decode_step(stu, torch.zeros(2, 8), None, 1e-6, (torch.zeros(2, 8, 2, 56), ragged(*t)), torch.zeros(2, 8))


@pytest.mark.parametrize("kv_bits", [None, 4])
@pytest.mark.parametrize("last", [10, 63, 200])
def test_streams_count_what_rings_hold(monkeypatch, kv_bits, last):
    """The bytes of keys and values that steps up to position `last` read, by the window and not by the rings' second axis (of 4 bits: heads)."""
    import flash_stu_2_b200 as F
    from flash_stu_2_b200.stream_ahead import StreamAhead
    asked = []
    monkeypatch.setattr(StreamAhead, "supported", staticmethod(lambda *a: True))
    monkeypatch.setattr(StreamAhead, "sms", staticmethod(lambda *a: asked.append(a) or 0))
    monkeypatch.setattr("flash_stu_2_b200.stream_ahead._sm_count", lambda dev: 148)
    cfg = F.FlashSTUConfig(n_embd=64, n_heads=4, n_layers=2, seq_len=256, window_size=63, vocab_size=11, mlp_scale=2, num_eigh=4, kv_bits=kv_bits,
                           torch_dtype=torch.bfloat16)
    m = F.FlashSTU(cfg)
    past = [layer.stu.new_cache(16, "cpu") if hasattr(layer, "stu") else layer.attn.new_cache(16, "cpu") for layer in m.layers]
    assert StreamAhead.plan(m.layers, past, 16, last, 1000) is None
    row = 4 * 20 if kv_bits else 64 * 2                      # bytes of a position's keys: heads of 16 in 4 bits are 20, a row of 64 bf16 128
    assert asked[0][6] == 2 * 16 * row * min(last, 64)


def test_steps_of_too_many_sequences_are_refused():
    from flash_stu_2_b200 import ops
    k4, v4 = ops.kv4_rings(65536, 16, 1, 8, "cpu")
    qkv, pos = torch.zeros(65536, 1, 24), torch.zeros(65536, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="65535"):
        ops.kv4_step(qkv, k4, v4, pos, None, 1, 15)
