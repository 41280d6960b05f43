"""Packed prompts and rings of 4 bits at their edges: caches made anew, huge finite values beside others, infinite scores."""
import pytest
import torch

import kv4_reference as R
from test_gpu_7_kv4 import activations, cu_of, gen, slopes_of
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


# ---------------------------------------------------------------------------------------------------- huge finite values
def huge(dt):
    most = torch.finfo(dt).max
    return (most, -most, 3e38, -3e38, 1e36)


def check_rows(got, want, tol, rows):
    R.check(got[rows], want[rows], tol[rows])


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("hd", [64, 128, 40, 13])
@pytest.mark.parametrize("cap,window", [(50.0, None), (0.0, 30)])
def test_packed_huge_values_are_for_those_who_see_them(dt, hd, cap, window):
    """Finite values as large as the type's, in one sequence or at one key: no other sequence and no earlier row has anything of them, and rows that
    are past the key's window neither.  (All but the weights of what is seen are the same for them, so the reference's tolerance is too.)"""
    from flash_stu_2_b200 import ops
    g, H, kv, lengths = gen(hd), 2, 1, (70, 33, 200, 5)
    qkv, cu, slopes = activations(g, sum(lengths), H, kv, hd, dt), cu_of(lengths), slopes_of(H)
    want, tol = R.packed(qkv, lengths, 0, slopes, H, kv, window, cap, dt)
    for value in huge(dt):
        for bad in range(4):
            x = qkv.clone()
            a, b = int(cu[bad]), int(cu[bad + 1])
            x[a:b, H * hd:] = value
            got = ops.swa_packed(x, cu, slopes, H, window, cap, kv_heads=kv)
            check_rows(torch.cat([got[:a], got[b:]]), torch.cat([want[:a], want[b:]]), torch.cat([tol[:a], tol[b:]]), slice(None))
        x = qkv.clone()
        x[150, (H + kv) * hd:] = value              # one value in the third, whose rows are 103 .. 302
        got = ops.swa_packed(x, cu, slopes, H, window, cap, kv_heads=kv)
        some = list(range(150)) + list(range(303, 308)) + (list(range(150 + window + 1, 303)) if window else [])
        check_rows(got, want, tol, some)
        seen, loose = R.packed(x, lengths, 0, slopes, H, kv, window, cap, dt)
        check_rows(got, seen, loose, slice(150, 150 + window + 1 if window else 303))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_packed_huge_values_far_away(dt, hd):
    """A huge value that is seen from so far that ALiBi leaves nothing of it: e^-390 of it is below 10^-130."""
    from flash_stu_2_b200 import ops
    g, H, kv, n = gen(hd + 1), 2, 2, 400
    qkv, cu, slopes = activations(g, n, H, kv, hd, dt), cu_of([n]), torch.tensor([8.0, 4.0], device=dev())
    for cap in (0.0, 50.0):
        want, tol = R.packed(qkv, [n], 0, slopes, H, kv, None, cap, dt)
        for value in huge(dt):
            x = qkv.clone()
            x[96:100, (H + kv) * hd:] = value
            got = ops.swa_packed(x, cu, slopes, H, None, cap)
            check_rows(got, want, tol, list(range(96)) + list(range(200, n)))


@pytest.mark.parametrize("hd", [64, 128, 30])
@pytest.mark.parametrize("cap", [0.0, 50.0])
def test_packed_huge_queries_and_keys(hd, cap):
    """The largest fp32 numbers in queries and keys, where the other side is 0: they add nothing to a score."""
    from flash_stu_2_b200 import ops
    g, H, kv, lengths, dt = gen(hd + 2), 4, 2, (50, 90), torch.float32
    qkv, cu, slopes = activations(g, sum(lengths), H, kv, hd, dt), cu_of(lengths), slopes_of(H)
    x = qkv.view(-1, H + 2 * kv, hd)
    x[:, :H, 5] = 0.0
    x[:, H:H + kv, 7] = 0.0
    want, tol = R.packed(qkv, lengths, 0, slopes, H, kv, 40, cap, dt)
    for value in huge(dt):
        y = qkv.clone().view(-1, H + 2 * kv, hd)
        y[33, H:H + kv, 5] = value
        y[70, :H, 7] = value
        y[139, H + 1, 5] = value
        R.check(ops.swa_packed(y.flatten(1), cu, slopes, H, 40, cap, kv_heads=kv), want, tol)


# ---------------------------------------------------------------------------------------------------- infinite scores
def by_hand(qkv, lengths, slopes, H, kv, window, cap, dt, unseen):
    """R.packed where nobody sees the rows `unseen`."""
    x = qkv.double().view(qkv.shape[0], H + 2 * kv, -1)
    out, tol, at = [], [], 0
    for n in lengths:
        p = torch.arange(n, device=qkv.device)
        behind = p[:, None] - p
        seen = (behind >= 0) & (behind <= window)
        for j in unseen:
            if at <= j < at + n:
                seen[:, j - at] = False
        rows = [R.attention(x[at:at + n, h], x[at:at + n, H + h * kv // H], x[at:at + n, H + kv + h * kv // H], behind, seen, float(slopes[h]), cap)
                for h in range(H)]
        out.append(torch.stack([o for o, _ in rows], 1))
        tol.append(torch.stack([R.tolerance(o, t, dt, R.WEIGHTS_PACKED[dt], R.TANH[dt]) for o, t in rows], 1))
        at += n
    out, tol = torch.cat(out).flatten(1), torch.cat(tol).flatten(1)
    return out, tol


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("hd", [64, 128, 13])
@pytest.mark.parametrize("beside", [False, True])
def test_packed_keys_of_no_weight(dt, hd, beside):
    """Keys whose scores are minus infinity weigh nothing, the first that a row sees and the first of a tile among them; a row that sees only such has no
    result.  beside: NaN in the keys and values of the next sequence, for which rows are computed in another way."""
    from flash_stu_2_b200 import ops
    g, H, kv, lengths, window = gen(hd + 3), 2, 1, (100, 60), 10
    qkv, cu, slopes = activations(g, sum(lengths), H, kv, hd, dt), cu_of(lengths), slopes_of(H)
    x = qkv.view(-1, H + 2 * kv, hd)
    x[:, :H, 3] = x[:, :H, 3].abs() + 1
    none = [0, 1, 22, 53, 54, 85, 99]
    want, tol = by_hand(qkv, lengths, slopes, H, kv, window, 0.0, dt, none)
    x[none, H:H + kv] = 0.0
    x[none, H:H + kv, 3] = float("-inf")
    if beside:
        x[100:, H:] = float("nan")
    got = ops.swa_packed(qkv, cu, slopes, H, window, 0.0, kv_heads=kv)
    assert bool(got[:2].isnan().all()) and bool(got[100:].isnan().all()) == beside
    R.check(got[2:100], want[2:100], tol[2:100])
    if not beside:
        R.check(got[100:], want[100:], tol[100:])


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("hd", [64, 128, 13])
def test_packed_infinite_scores_are_capped(dt, hd):
    """A soft cap makes a finite score of an infinite one, the same as of one that is far past it."""
    from flash_stu_2_b200 import ops
    g, H, kv, lengths, window, cap = gen(hd + 4), 2, 1, (100, 60), 10, 3.0
    qkv, cu, slopes = activations(g, sum(lengths), H, kv, hd, dt), cu_of(lengths), slopes_of(H)
    x = qkv.view(-1, H + 2 * kv, hd)
    x[:, :H, 3] = x[:, :H, 3].abs() + 1
    for sign in (1.0, -1.0):
        for j in (0, 22, 53, 159):
            x[j, H:H + kv] = 0.0
            x[j, H:H + kv, 3] = sign * 60 * hd ** 0.5      # a score of 60 and more: tanh(20) is 1 - 2^-56
        want, tol = R.packed(qkv, lengths, 0, slopes, H, kv, window, cap, dt)
        y = x.clone()
        for j in (0, 22, 53, 159):
            y[j, H:H + kv, 3] = sign * float("inf")
        R.check(ops.swa_packed(y.flatten(1), cu, slopes, H, window, cap, kv_heads=kv), want, tol)
