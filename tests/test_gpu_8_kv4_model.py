"""Layers and models whose attention layers hold their keys and values in 4 bits, and models that take packed prompts."""
import pytest
import torch

import kv4_reference as R

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]
# Two ways through the same weights differ by the rounding of attention's outputs (and of what follows from them): a few halves of a step per layer.
SAME = {torch.bfloat16: 2e-2, torch.float32: 1e-4}


def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


def model(dt, seed=0, **kw):
    import flash_stu_2_b200 as F
    torch.manual_seed(seed)
    cfg = F.FlashSTUConfig(**{**dict(n_embd=256, n_heads=4, n_layers=4, seq_len=256, window_size=40, vocab_size=97, mlp_scale=2, num_eigh=8, softcap=20.0,
                                     torch_dtype=dt, kv_bits=4), **kw})
    m = F.FlashSTU(cfg).to(dev()).eval()
    with torch.no_grad():   # (a layer's branch is small against the stream, as in a trained model)
        for name, p in m.named_parameters():
            if name.endswith(("c_proj.weight", "down_proj.weight")):
                p.mul_(0.5)
    return m


def far(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("calls", [(30, 1, 1, 1), (1, 1, 1), (100, 60, 1, 7, 1), (400, 3, 1)])
@pytest.mark.parametrize("heads,d", [(4, 256), (2, 256), (4, 160)])
def test_attention_layer_holds_what_it_says(dt, calls, heads, d):
    """Every call attends its own keys and values as they are and those of earlier calls as the rings hold them."""
    import flash_stu_2_b200 as F
    from flash_stu_2_b200 import ops
    torch.manual_seed(1)
    window, B, hd = 50, 2, d // heads
    cfg = F.FlashSTUConfig(n_embd=d, n_heads=heads, n_layers=1, seq_len=512, window_size=window, vocab_size=8, torch_dtype=dt, kv_bits=4, softcap=30.0)
    attn = F.Attention(cfg).to(dev())
    with torch.no_grad():
        attn.c_attn.weight.mul_(3)
    entry, rows = None, []
    t = 0
    for n in calls:
        x = torch.randn(B, n, d, device=dev()).to(dt)
        y, entry = attn.attend(x, entry, True)
        qkv = ops.linear(x.reshape(B * n, d), attn.c_attn.weight).view(B, n, 3, heads, hd)
        rows.append(qkv)
        for b in range(B):
            old = torch.cat([r[b, :, 1:] for r in rows[:-1]], 0) if t else qkv[b, :0, 1:]
            kv = torch.cat([R.held(old.float()), qkv[b, :, 1:].double()], 0)
            behind = torch.arange(t, t + n, device=dev())[:, None] - torch.arange(t + n, device=dev())
            seen = (behind >= 0) & (behind <= window)
            for h in range(heads):
                o, tt = R.attention(qkv[b, :, 0, h].double(), kv[:, 0, h], kv[:, 1, h], behind, seen, float(attn.alibi_slopes[h]), 30.0)
                # (several tokens: the rings' values are rounded to the model's type on their way into the kernel that takes them)
                loose = 2.0 ** -8 if dt == torch.bfloat16 else 2.0 ** -22
                moved = 2 * loose * (tt["terms"] * 2 + 1) if n > 1 else 0.0
                tol = R.tolerance(o, tt, dt, R.WEIGHTS_PACKED[dt], R.TANH[dt]) + tt["a"] * (moved + loose)
                R.check(y[b, :, h * hd:(h + 1) * hd], o, tol)
        t += n
    assert entry[2][:, 0].tolist() == [t] * B and entry[0].dtype == torch.uint8


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("B", [1, 3, 20])
def test_generate(dt, B):
    """Replayed steps are the layers' own; the rings' rounding changes logits by little."""
    m, plain = model(dt), model(dt, kv_bits=None)
    ids = torch.randint(97, (B, 60), device=dev())
    u = torch.rand(30, B)
    want, logits = m.generate(ids, max_length=90, top_k=5, uniforms=u, return_logits=True, cuda_graph=False)
    got, replayed = m.generate(ids, max_length=90, top_k=5, uniforms=u, return_logits=True)
    assert torch.equal(got, want) and torch.equal(logits, replayed)
    past = None
    with torch.no_grad():
        for step in range(30):
            out = m(want[:, :60] if step == 0 else want[:, 59 + step:60 + step], past_key_values=past, use_cache=True)
            past = out.past_key_values
            assert far(out.logits[:, -1], logits[:, step]) < SAME[dt]
        exact = plain(want[:, :60]).logits[:, -1]
        assert far(logits[:, 0], exact) < SAME[dt]          # (a prompt alone: nothing was read from a ring)
        full = plain(want[:, :-1]).logits[:, 59:]
    assert 1e-6 < far(logits, full) < 0.2
    from flash_stu_2_b200 import ops
    ops.check_status()


@pytest.mark.parametrize("dt", DTYPES)
def test_prompt_in_pieces(dt):
    """A prompt read in several calls comes near the one in one."""
    m = model(dt)
    ids = torch.randint(97, (2, 150), device=dev())
    with torch.no_grad():
        whole = m(ids).logits
        past, parts = None, []
        for a, b in ((0, 70), (70, 71), (71, 150)):
            out = m(ids[:, a:b], past_key_values=past, use_cache=True)
            past = out.past_key_values
            parts.append(out.logits)
    assert far(torch.cat(parts, 1), whole) < 0.2 and far(parts[0], whole[:, :70]) < SAME[dt]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("kw", [{}, dict(use_approx=False), dict(use_hankel_L=True), dict(n_heads=2, window_size=300), dict(use_attn=False)])
def test_packed_prompts(dt, kw):
    """Logits of packed prompts are those of each alone."""
    m = model(dt, **kw)
    lengths = [33, 1, 200, 0, 64]
    ids = torch.randint(97, (1, sum(lengths)), device=dev())
    with torch.no_grad():
        got = m(ids, lengths=lengths, use_cache=False).logits
        assert got.shape == (1, sum(lengths), 97)
        at = 0
        for n in lengths:
            if n:
                assert far(got[:, at:at + n], m(ids[:, at:at + n], use_cache=False).logits) < SAME[dt]
            at += n
        # other prompts beside it change nothing in a prompt
        other = ids.clone()
        other[:, 34:234] = torch.randint(97, (1, 200), device=dev())
        again = m(other, lengths=lengths, use_cache=False).logits
        assert torch.equal(again[:, :34], got[:, :34]) and torch.equal(again[:, 234:], got[:, 234:]) and not torch.equal(again, got)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("kw", [{}, dict(use_attn=False), dict(n_embd=192, n_heads=3)])
def test_packed_prompts_then_tokens(dt, kw):
    """The caches of packed prompts of different lengths go on token by token like those of each prompt alone."""
    m = model(dt, **kw)
    lengths = [50, 7, 130, 1]
    ids = torch.randint(97, (1, sum(lengths)), device=dev())
    nxt = torch.randint(97, (4, 12), device=dev())
    with torch.no_grad():
        out = m(ids, lengths=lengths, use_cache=True)
        past, steps = out.past_key_values, []
        for t in range(12):
            out = m(nxt[:, t:t + 1], past_key_values=past, use_cache=True)
            past = out.past_key_values
            steps.append(out.logits[:, 0])
        at = 0
        for s, n in enumerate(lengths):
            alone = m(ids[:, at:at + n], use_cache=True).past_key_values
            for t in range(12):
                out = m(nxt[s:s + 1, t:t + 1], past_key_values=alone, use_cache=True)
                alone = out.past_key_values
                assert far(steps[t][s], out.logits[0, 0]) < 4 * SAME[dt]     # (4 bits: a value near the middle of two numbers falls to either side)
            at += n
        with pytest.raises(ValueError, match="different positions"):
            m(nxt[:, :2], past_key_values=past, use_cache=True)
    from flash_stu_2_b200 import ops
    ops.check_status()


def test_reordered_caches():
    """Beams that change places take their rings along."""
    m = model(torch.bfloat16)
    ids = torch.randint(97, (3, 45), device=dev())
    with torch.no_grad():
        past = m(ids, use_cache=True).past_key_values
        order = torch.tensor([2, 0, 0], device=dev())
        moved = m._reorder_cache(past, order)
        nxt = torch.randint(97, (3, 1), device=dev())
        got = m(nxt, past_key_values=moved, use_cache=True).logits
        want = m(nxt, past_key_values=m(ids[order], use_cache=True).past_key_values, use_cache=True).logits
    assert far(got, want) < SAME[torch.bfloat16]


def test_refusals_of_models():
    m = model(torch.bfloat16)
    ids = torch.randint(97, (1, 10), device=dev())
    with torch.no_grad():
        for lengths in ([4, 5], [11], [-1, 11], []):
            with pytest.raises(ValueError):
                m(ids, lengths=lengths)
        with pytest.raises(ValueError):
            m(ids.expand(2, -1), lengths=[10])
        with pytest.raises(ValueError):
            m(ids, lengths=[10], past_key_values=m(ids, use_cache=True).past_key_values)
        with pytest.raises(ValueError, match="capacity"):
            m(torch.zeros(1, 300, dtype=torch.int64, device=dev()), lengths=[299, 1], use_cache=True)
        with pytest.raises(NotImplementedError, match="4 bits"):
            model(torch.bfloat16, kv_bits=None)(ids, lengths=[3, 7], use_cache=True)
        for kw in (dict(use_approx=False), dict(use_hankel_L=True), dict(stu_enable_mlp_sandwich=True)):
            with pytest.raises(NotImplementedError, match="different positions"):
                model(torch.bfloat16, **kw)(ids, lengths=[3, 7], use_cache=True)
