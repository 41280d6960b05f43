"""Packed prompts and rings of 4 bits at their edges: caches made anew, huge finite values beside others, infinite scores."""
import pytest
import torch

from test_gpu_8_kv4_model import SAME, dev, far, model

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]


# ---------------------------------------------------------------------------------------------------- caches at different positions
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("order", [(2, 0, 1, 3), (1, 2, 3, 0), (3, 3, 2, 0)])
@pytest.mark.parametrize("how", ["reorder", "clone"])
def test_packed_caches_made_anew(dt, order, how):
    """Reordered or cloned caches of packed prompts go on token by token like each prompt alone, and refuse several tokens."""
    m = model(dt)
    lengths = [50, 7, 130, 1]
    ids = torch.randint(97, (1, sum(lengths)), device=dev())
    nxt = torch.randint(97, (4, 6), device=dev())
    cut = [0, 50, 57, 187, 188]
    with torch.no_grad():
        past = m(ids, lengths=lengths, use_cache=True).past_key_values
        if how == "clone":
            past, order = tuple(tuple(t.clone() for t in e) for e in past), (0, 1, 2, 3)
        else:
            past = m._reorder_cache(past, torch.tensor(order, device=dev()))
        before = [[t.clone() for t in e] for e in past]
        with pytest.raises(ValueError, match="different positions"):
            m(nxt[:, :2], past_key_values=past, use_cache=True)
        assert all(torch.equal(a, b) for e, kept in zip(past, before) for a, b in zip(e, kept))     # (nothing has moved on)
        steps = []
        for t in range(6):
            out = m(nxt[:, t:t + 1], past_key_values=past, use_cache=True)
            past = out.past_key_values
            steps.append(out.logits[:, 0])
        for s, of in enumerate(order):
            alone = m(ids[:, cut[of]:cut[of + 1]], use_cache=True).past_key_values
            for t in range(6):
                out = m(nxt[s:s + 1, t:t + 1], past_key_values=alone, use_cache=True)
                alone = out.past_key_values
                assert far(steps[t][s], out.logits[0, 0]) < 4 * SAME[dt]     # (4 bits: a value near the middle of two numbers falls to either side)
    assert past[0][-1][:, 0].tolist() == [lengths[of] + 6 for of in order]


def test_reordered_caches_end_at_the_capacity():
    """The furthest sequence counts, wherever it stands."""
    m = model(torch.bfloat16)
    ids = torch.randint(97, (1, 260), device=dev())
    with torch.no_grad():
        past = m(ids, lengths=[255, 5], use_cache=True).past_key_values
        past = m._reorder_cache(past, torch.tensor([1, 0], device=dev()))
        past = m(ids[:, :2].view(2, 1), past_key_values=past, use_cache=True).past_key_values
        with pytest.raises(ValueError, match="exceeds the capacity"):
            m(ids[:, :2].view(2, 1), past_key_values=past, use_cache=True)
    from flash_stu_2_b200 import ops
    ops.check_status()


def test_layers_by_themselves_refuse_different_positions():
    """A layer's prefill, with and without what the host knows of the positions."""
    m = model(torch.bfloat16)
    ids = torch.randint(97, (1, 60), device=dev())
    x = torch.zeros(2, 3, 256, dtype=torch.bfloat16, device=dev())
    with torch.no_grad():
        past = m(ids, lengths=[7, 53], use_cache=True).past_key_values
        for e in (past[0], tuple(t.clone() for t in past[0])):
            with pytest.raises(ValueError, match="different positions"):
                m.layers[0](x, past_key_value=e, use_cache=True)
