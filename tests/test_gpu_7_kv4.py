"""Rings of 4 bits, attention over them and over packed prompts, against the definitions in 64 bits (kv4_reference.py says what each may be off)."""
import math

import pytest
import torch

import kv4_reference as R

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]


def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


def gen(seed):
    return torch.Generator(device=dev()).manual_seed(seed)


def activations(g, rows, H, kv, hd, dt):
    """Queries, keys and values: keys with channels of their own level, some of them far off."""
    level = torch.randn(kv * hd, device=dev(), generator=g)
    level[torch.randint(kv * hd, (max(1, kv * hd // 50),), device=dev(), generator=g)] *= 4
    k = torch.randn(rows, kv * hd, device=dev(), generator=g) + level
    q = 1.5 * torch.randn(rows, H * hd, device=dev(), generator=g)
    return torch.cat([q, k, torch.randn(rows, kv * hd, device=dev(), generator=g)], 1).to(dt)


def slopes_of(H):
    return (0.25 * 2.0 ** (-8 * torch.arange(1, H + 1, device=dev(), dtype=torch.float32) / H))


def positions(*t):
    p = torch.zeros(len(t), 2, dtype=torch.int32, device=dev())
    p[:, 0] = torch.tensor(t, dtype=torch.int32)
    return p


def cu_of(lengths, first=0):
    return torch.tensor([first] + list(lengths), device=dev()).cumsum(0).to(torch.int32)


def full_rings(g, B, slots, kv, hd, dt):
    x = activations(g, B * slots, 1, kv, hd, dt)[:, hd:].view(B, slots, 2, kv, hd).permute(2, 0, 3, 1, 4)
    return R.ring_bytes(x[0]), R.ring_bytes(x[1])


def put(ring, x, at, hd):
    """The reference's write: x [tokens, kv, hd] of one sequence at positions at .. into ring [1, kv, ...]."""
    slots = R.parts(ring, hd)[0].shape[2]
    for t in range(max(0, len(x) - slots), len(x)):
        one = R.ring_bytes(x[t][None, :, None].expand(1, -1, 16, -1))      # (a ring of 16 slots, all of them this token)
        for to, made in zip(R.parts(ring, hd), R.parts(one, hd)):
            to[:, :, (at + t) % slots] = made[:, :, 0]


# ---------------------------------------------------------------------------------------------------- write and read
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("H,kv,hd", [(1, 1, 8), (2, 1, 24), (3, 3, 32), (6, 3, 40), (4, 4, 64), (5, 1, 72), (2, 2, 96), (8, 2, 128)])
def test_write_is_exact(dt, H, kv, hd):
    """Several calls: the ring is filled, passed, written over by more tokens than it has slots, and by one token."""
    from flash_stu_2_b200 import ops
    g, B, slots = gen(hd + H), 2, 32
    k4, v4 = ops.kv4_rings(B, slots, kv, hd, dev())
    want, pos, at = [k4.clone(), v4.clone()], positions(0, 7), [0, 7]
    for tokens in (5, 1, 30, 100, 1):
        qkv = activations(g, B * tokens, H, kv, hd, dt).view(B, tokens, -1)
        ops.kv4_write(qkv, k4, v4, pos, H)
        x = qkv.view(B, tokens, H + 2 * kv, hd)
        for b in range(B):
            for i in range(2):
                put(want[i][b:b + 1], x[b, :, H + i * kv:H + (i + 1) * kv], at[b], hd)
            at[b] += tokens
        assert torch.equal(k4, want[0]) and torch.equal(v4, want[1])
        assert pos.tolist() == [[at[0], 0], [at[1], 0]]
    for out in DTYPES:
        for got, ring in zip(ops.kv4_read(k4, v4, hd, out), want):
            assert torch.equal(got, R.values(ring, hd).transpose(1, 2).flatten(2).float().to(out))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("lengths,first,behind", [((3, 0, 50, 1), 0, 0), ((1,), 5, 3), ((0, 0, 17), 2, 1), ((33, 16), 0, 40)])
def test_write_packed(dt, lengths, first, behind):
    """Sequences of none, one and more tokens than slots; rows ahead of the first and behind the last are nobody's."""
    from flash_stu_2_b200 import ops
    g, slots, H, kv, hd = gen(len(lengths)), 16, 4, 2, 80
    B = len(lengths)
    start = [3 * b for b in range(B)]
    qkv = activations(g, first + sum(lengths) + behind, H, kv, hd, dt)
    k4, v4 = full_rings(g, B, slots, kv, hd, dt)
    want, pos, cu = [k4.clone(), v4.clone()], positions(*start), cu_of(lengths, first)
    ops.kv4_write(qkv, k4, v4, pos, H, cu_seqlens=cu)
    x, row = qkv.view(-1, H + 2 * kv, hd), first
    for b, n in enumerate(lengths):
        for i in range(2):
            put(want[i][b:b + 1], x[row:row + n, H + i * kv:H + (i + 1) * kv], start[b], hd)
        row += n
    assert torch.equal(k4, want[0]) and torch.equal(v4, want[1])
    assert pos.tolist() == [[s + n, 0] for s, n in zip(start, lengths)]


@pytest.mark.parametrize("dt", DTYPES)
def test_write_borders(dt):
    """Infinities and NaN, alone and beside others; pieces of one value, of zeros of both signs; the smallest and the largest numbers; ties; ranges that
    pass fp32's; a minimum that rounds down to minus infinity."""
    from flash_stu_2_b200 import ops
    hd, lines = 128, []
    ramp = torch.linspace(-1, 1, 64, dtype=torch.float64)
    for special in (math.nan, math.inf, -math.inf):
        line = torch.cat([ramp, ramp])
        line[70] = special
        lines += [line, torch.full((hd,), special, dtype=torch.float64)]
    for top in (2.0 ** -149, 2.0 ** -133, 2.0 ** -126, 2.0 ** -120, 1.0, 2.0 ** 100, 1.6e38, 3.0e38, 3.38e38, 3.4e38):
        lines += [torch.cat([ramp * top, ramp.abs() * top]), torch.full((hd,), -top, dtype=torch.float64), torch.cat([100 * top + ramp * top, ramp * top - top])]
    lines += [torch.zeros(hd, dtype=torch.float64), -torch.zeros(hd, dtype=torch.float64), torch.cat([torch.zeros(64), -torch.zeros(64)]).double()]
    mixed = torch.zeros(hd, dtype=torch.float64)
    mixed[::2] *= -1
    lines.append(mixed)
    grid = torch.arange(64, dtype=torch.float64) % 31 / 2     # 0, 0.5, .. 15: the step is 1, every second value a tie
    lines += [torch.cat([grid, grid - 15]), torch.cat([grid * 2.0 ** -60, grid * 2.0 ** 60])]
    x = torch.stack(lines).to(dt).to(dev())
    n = (len(lines) + 15) // 16 * 16
    x = torch.cat([x, x[:1].expand(n - len(x), -1)])
    qkv = torch.cat([torch.zeros_like(x), x, x.flip(1)], 1)[None].contiguous()
    k4, v4 = ops.kv4_rings(1, n, 1, hd, dev())
    ops.kv4_write(qkv, k4, v4, positions(0), 1)
    for ring, v in ((k4, x), (v4, x.flip(1))):
        assert torch.equal(ring, R.ring_bytes(v[None, None]))
    for got, v in zip(ops.kv4_read(k4, v4, hd, torch.float32), (x, x.flip(1))):
        assert torch.equal(got.nan_to_num(7e7), R.held(v)[None].float().nan_to_num(7e7))


@pytest.mark.parametrize("dt", DTYPES)
def test_write_takes_any_rows(dt):
    """Rows off the 16-byte grid, further apart than they are long, of a transposed tensor."""
    from flash_stu_2_b200 import ops
    g, H, kv, hd = gen(5), 2, 2, 64
    plain = activations(g, 2 * 9, H, kv, hd, dt)
    rows = []
    for pad, at in ((8, 0), (3, 1), (5, 2), (16, 8)):
        wide = torch.full((18, plain.shape[1] + pad), math.nan, device=dev(), dtype=dt)
        wide[:, at:at + plain.shape[1]] = plain
        rows.append(wide[:, at:at + plain.shape[1]])
    rows.append(plain.t().contiguous().t())
    made = []
    for r in [plain] + rows:
        for qkv, cu in ((r, cu_of([4, 14])), (r.unflatten(0, (2, 9)), None)):
            k4, v4 = ops.kv4_rings(2, 16, kv, hd, dev())
            ops.kv4_write(qkv, k4, v4, positions(0, 0), H, cu_seqlens=cu)
            made.append((k4, v4))
    for i, (k4, v4) in enumerate(made):
        assert torch.equal(k4, made[i % 2][0]) and torch.equal(v4, made[i % 2][1])


def test_write_nothing():
    from flash_stu_2_b200 import ops
    k4, v4 = full_rings(gen(1), 2, 16, 1, 64, torch.float32)
    before, pos = (k4.clone(), v4.clone()), positions(3, 4)
    ops.kv4_write(torch.zeros(2, 0, 192, device=dev()), k4, v4, pos, 1)
    ops.kv4_write(torch.zeros(0, 192, device=dev()), k4, v4, pos, 1, cu_seqlens=cu_of([0, 0]))
    ops.kv4_write(torch.ones(7, 192, device=dev()), k4, v4, pos, 1, cu_seqlens=cu_of([0, 0], 3))
    assert torch.equal(k4, before[0]) and torch.equal(v4, before[1]) and pos.tolist() == [[3, 0], [4, 0]]


# ---------------------------------------------------------------------------------------------------- one token
STEPS = [  # B, H, kv, hd, window, more slots, positions
    (1, 1, 1, 8, 0, 0, (0,)),
    (1, 1, 1, 64, 15, 0, (1,)),
    (3, 4, 4, 64, 100, 0, (0, 1, 57)),
    (2, 8, 8, 64, 511, 0, (137, 511)),
    (2, 12, 12, 128, 127, 0, (128, 4000)),
    (1, 12, 12, 128, 1024, 0, (5000,)),
    (5, 6, 3, 40, 127, 32, (0, 3, 126, 127, 300)),
    (2, 8, 1, 128, 300, 0, (299, 1000)),
    (2, 16, 2, 128, 40, 100, (39, 777)),
    (1, 5, 1, 64, 2000, 0, (2500,)),
    (2, 11, 1, 72, 65, 0, (30, 70)),
    (1, 40, 2, 32, 700, 0, (1400,)),
    (1, 2, 1, 96, 4095, 0, (100000,)),
    (2, 3, 3, 24, 33, 0, (31, 34)),
    (40, 2, 2, 64, 64, 0, tuple(range(40))),
]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("cap,alibi", [(0.0, False), (50.0, True), (3.0, True)])
@pytest.mark.parametrize("case", range(len(STEPS)))
def test_step(case, cap, alibi, dt):
    from flash_stu_2_b200 import ops
    B, H, kv, hd, window, more, at = STEPS[case]
    g, slots = gen(case), ops.kv4_slots(window + more)
    k4, v4 = full_rings(g, B, slots, kv, hd, dt)
    qkv, pos = activations(g, B, H, kv, hd, dt).view(B, 1, -1), positions(*at)
    slopes = slopes_of(H) if alibi else None
    want, tol = R.step(qkv, k4, v4, pos, slopes, H, window, cap, dt)
    before = k4.clone(), v4.clone()
    got = ops.kv4_step(qkv, k4, v4, pos, slopes, H, window, cap, update_cache=False)
    R.check(got, want, tol)
    assert torch.equal(k4, before[0]) and torch.equal(v4, before[1]) and pos[:, 0].tolist() == list(at)
    kept = ops.kv4_step(qkv, k4, v4, pos, slopes, H, window, cap)
    assert torch.equal(kept, got)
    for ring, x in zip(before, qkv.view(B, H + 2 * kv, hd)[:, H:].split(kv, 1)):
        for b in range(B):
            put(ring[b:b + 1], x[b:b + 1], at[b], hd)
    assert torch.equal(k4, before[0]) and torch.equal(v4, before[1])
    assert pos.tolist() == [[t + 1, 0] for t in at]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("hd,kv,H", [(64, 2, 2), (128, 1, 4), (40, 1, 1)])
def test_step_does_not_look_past_its_window(dt, hd, kv, H):
    """Slots of tokens that are out of the window, or that no token was written to, may hold anything: NaN scales, any numbers."""
    from flash_stu_2_b200 import ops
    g, window = gen(hd), 45
    slots = ops.kv4_slots(window + 50)
    for t in (0, 1, 20, 45, 46, 95, 1000, 1007):
        k4, v4 = full_rings(g, 1, slots, kv, hd, dt)
        qkv, slopes = activations(g, 1, H, kv, hd, dt).view(1, 1, -1), slopes_of(H)
        plain = ops.kv4_step(qkv, k4, v4, positions(t), slopes, H, window, 50.0, update_cache=False)
        assert bool(plain.isfinite().all())
        live = {(t - i) % slots for i in range(1, min(window, t) + 1)}
        dead = torch.tensor([s for s in range(slots) if s not in live], device=dev())
        for ring in (k4, v4):
            rows, scales = R.parts(ring, hd)
            rows[:, :, dead] = 0xff
            scales[:, :, dead] = 0xff
        assert torch.equal(ops.kv4_step(qkv, k4, v4, positions(t), slopes, H, window, 50.0, update_cache=False), plain)
        if live:   # and a NaN that is in the window is seen
            R.parts(k4, hd)[1][:, :, min(live)] = 0xff
            assert bool(ops.kv4_step(qkv, k4, v4, positions(t), slopes, H, window, 50.0, update_cache=False).isnan().all())


@pytest.mark.parametrize("dt", DTYPES)
def test_step_of_extreme_scores(dt):
    """Scores of thousands apart: weights of 0 and 1; a score of the new token far below all others, and far above."""
    from flash_stu_2_b200 import ops
    g, H, kv, hd, window = gen(9), 4, 2, 64, 300
    k4, v4 = full_rings(g, 1, 304, kv, hd, dt)
    for factor in (0.0, 100.0, 3000.0):
        qkv = activations(g, 1, H, kv, hd, dt)
        qkv[:, :H * hd] *= factor
        for sign in (1.0, -1.0):
            qkv[:, H * hd:(H + kv) * hd] *= sign
            for t in (40, 900):
                pos = positions(t)
                want, tol = R.step(qkv[None], k4, v4, pos, None, H, window, 0.0, dt)
                R.check(ops.kv4_step(qkv[None], k4, v4, pos, None, H, window, 0.0, update_cache=False), want, tol)


@pytest.mark.parametrize("dt", DTYPES)
def test_step_streams(dt):
    """Tokens one after the other through a ring that fills up and wraps around: each is what the reference makes of the ring as it then is."""
    from flash_stu_2_b200 import ops
    g, B, H, kv, hd, window = gen(11), 2, 4, 2, 128, 20
    k4, v4 = ops.kv4_rings(B, 32, kv, hd, dev())
    pos, slopes = positions(0, 25), slopes_of(H)
    for _ in range(45):
        qkv = activations(g, B, H, kv, hd, dt).view(B, 1, -1)
        want, tol = R.step(qkv, k4, v4, pos, slopes, H, window, 50.0, dt)
        R.check(ops.kv4_step(qkv, k4, v4, pos, slopes, H, window, 50.0), want, tol)
    assert pos.tolist() == [[45, 0], [70, 0]]


# ---------------------------------------------------------------------------------------------------- packed prompts
PACKED = [  # H, kv, hd, window, lengths, rows ahead, rows behind
    (1, 1, 64, None, (1,), 0, 0),
    (2, 2, 128, 3, (7, 1, 19), 0, 0),
    (4, 4, 64, None, (130, 0, 1, 64), 2, 3),
    (3, 3, 128, 100, (300, 5, 129), 0, 1),
    (8, 2, 128, None, (513,), 0, 0),
    (8, 1, 64, 63, (200, 200, 1, 1, 1, 77), 1, 0),
    (2, 1, 40, 17, (33, 64, 90), 0, 0),
    (4, 2, 128, 0, (5, 140), 0, 0),
    (2, 2, 13, None, (50, 3), 0, 0),
    (5, 5, 96, 1000, (128, 256, 31), 0, 0),
    (12, 12, 128, 1024, (1100, 40), 0, 0),
    (4, 4, 64, 500, tuple([3] * 70), 0, 0),
    (6, 2, 32, 31, (0, 0, 97, 0), 0, 130),
]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("cap,alibi", [(0.0, False), (50.0, True), (3.0, False)])
@pytest.mark.parametrize("case", range(len(PACKED)))
def test_packed(case, cap, alibi, dt):
    from flash_stu_2_b200 import ops
    H, kv, hd, window, lengths, first, behind = PACKED[case]
    N = first + sum(lengths) + behind
    qkv = activations(gen(case), N, H, kv, hd, dt)
    qkv[:first] = math.nan                       # nobody's rows
    qkv[N - behind:] = math.nan
    slopes = slopes_of(H) if alibi else None
    want, tol = R.packed(qkv, lengths, first, slopes, H, kv, window, cap, dt)
    out = torch.full((N, H * hd), 7.0, device=dev(), dtype=dt)
    got = ops.swa_packed(qkv, cu_of(lengths, first), slopes, H, window, cap, kv_heads=kv, out=out)
    assert got is out
    assert bool((out[:first] == 7).all()) and bool((out[N - behind:] == 7).all())
    R.check(out[first:N - behind], want[first:N - behind], tol[first:N - behind])


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("hd", [64, 128, 40])
def test_packed_sequences_do_not_touch(dt, hd):
    """NaN and infinities in the keys and values of one sequence are in no other's rows.  (Rows that share a tile with them may be computed in another
    way, so each is held to the reference's tolerance, which is the same for both, and not to the other's bits.)"""
    from flash_stu_2_b200 import ops
    g, H, kv, lengths = gen(hd), 2, 1, (70, 33, 200, 5)
    qkv, cu, slopes = activations(g, sum(lengths), H, kv, hd, dt), cu_of(lengths), slopes_of(H)
    want, tol = R.packed(qkv, lengths, 0, slopes, H, kv, None, 50.0, dt)
    for bad in range(4):
        for value in (math.nan, math.inf):
            x = qkv.clone()
            a, b = int(cu[bad]), int(cu[bad + 1])
            x[a:b, H * hd:] = value
            got = ops.swa_packed(x, cu, slopes, H, None, 50.0, kv_heads=kv)
            assert bool(got[a:b].isnan().all())
            R.check(torch.cat([got[:a], got[b:]]), torch.cat([want[:a], want[b:]]), torch.cat([tol[:a], tol[b:]]))
    want, tol = R.packed(qkv, lengths, 0, slopes, H, kv, 8, 50.0, dt)
    x = qkv.clone()
    x[90, H * hd:] = math.nan                      # a key in the middle of the second: the rows from it on that see it
    got = ops.swa_packed(x, cu, slopes, H, 8, 50.0, kv_heads=kv)
    assert got.isnan().any(1).nonzero().flatten().tolist() == list(range(90, 99))
    R.check(torch.cat([got[:90], got[99:]]), torch.cat([want[:90], want[99:]]), torch.cat([tol[:90], tol[99:]]))


@pytest.mark.parametrize("dt", DTYPES)
def test_packed_takes_any_rows(dt):
    from flash_stu_2_b200 import ops
    g, H, hd, lengths = gen(3), 2, 64, (150, 40)
    plain, cu = activations(g, 190, H, H, hd, dt), cu_of((150, 40))
    want, tol = R.packed(plain, lengths, 0, slopes_of(H), H, H, 100, 50.0, dt)
    for pad, at in ((8, 0), (3, 1), (5, 2), (16, 8)):
        wide = torch.full((190, plain.shape[1] + pad), math.nan, device=dev(), dtype=dt)
        wide[:, at:at + plain.shape[1]] = plain
        out = torch.full((190, H * hd + pad), 7.0, device=dev(), dtype=dt)
        ops.swa_packed(wide[:, at:at + plain.shape[1]], cu, slopes_of(H), H, 100, 50.0, out=out[:, at:at + H * hd])
        R.check(out[:, at:at + H * hd], want, tol)
        assert bool((out[:, :at] == 7).all()) and bool((out[:, at + H * hd:] == 7).all())
    R.check(ops.swa_packed(plain.t().contiguous().t(), cu, slopes_of(H), H, 100, 50.0), want, tol)


def test_packed_nothing():
    from flash_stu_2_b200 import ops
    assert ops.swa_packed(torch.zeros(0, 192, device=dev()), cu_of([0]), None, 1).shape == (0, 64)
    out = torch.full((5, 64), 7.0, device=dev())
    ops.swa_packed(torch.zeros(5, 192, device=dev()), cu_of([0, 0], 2), None, 1, out=out)
    ops.swa_packed(torch.zeros(5, 192, device=dev()), cu_of([]), None, 1, out=out)
    assert bool((out == 7).all())


# ---------------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("hd", [64, 128, 48])
def test_prompts_then_tokens(dt, hd):
    """Prompts of different lengths in one call, their keys and values into rings, then tokens: every step is the reference's over what the rings hold, and
    near what attention over the exact keys and values would be."""
    from flash_stu_2_b200 import ops
    g, H, kv, window, lengths = gen(hd), 4, 2, 150, (200, 1, 149, 64)
    slots, cu, slopes = ops.kv4_slots(window), cu_of(lengths), slopes_of(H)
    qkv = activations(g, sum(lengths), H, kv, hd, dt)
    want, tol = R.packed(qkv, lengths, 0, slopes, H, kv, window, 50.0, dt)
    R.check(ops.swa_packed(qkv, cu, slopes, H, window, 50.0, kv_heads=kv), want, tol)
    k4, v4 = ops.kv4_rings(4, slots, kv, hd, dev())
    pos = positions(0, 0, 0, 0)
    ops.kv4_write(qkv, k4, v4, pos, H, cu_seqlens=cu)
    assert pos[:, 0].tolist() == list(lengths)
    for _ in range(3):
        new = activations(g, 4, H, kv, hd, dt).view(4, 1, -1)
        want, tol = R.step(new, k4, v4, pos, slopes, H, window, 50.0, dt)
        R.check(ops.kv4_step(new, k4, v4, pos, slopes, H, window, 50.0), want, tol)
    keys, _ = ops.kv4_read(k4, v4, hd, torch.float32)
    x = qkv.view(-1, H + 2 * kv, hd)[int(cu[2]):int(cu[3]), H:H + kv].float().flatten(1)      # the third prompt: all of it is there
    step = (x.unflatten(1, (kv, hd)).amax(2) - x.unflatten(1, (kv, hd)).amin(2)).amax() / 15
    assert float((keys[2, :149] - x).abs().max()) <= float(step) * 0.6


@pytest.mark.parametrize("dt", DTYPES)
def test_calls_repeat(dt):
    """The same call twice gives the same bits."""
    from flash_stu_2_b200 import ops
    g, H, kv, hd = gen(2), 8, 2, 128
    qkv, cu = activations(g, 700, H, kv, hd, dt), cu_of((300, 399, 1))
    a, b = (ops.swa_packed(qkv, cu, slopes_of(H), H, 200, 50.0, kv_heads=kv) for _ in range(2))
    assert torch.equal(a, b)
    k4, v4 = full_rings(g, 3, 2000, kv, hd, dt)
    pos = positions(5000, 10, 1999)
    a, b = (ops.kv4_step(qkv[:3, None], k4, v4, pos, slopes_of(H), H, 1999, 50.0, update_cache=False) for _ in range(2))
    assert torch.equal(a, b)


@pytest.mark.parametrize("dt", DTYPES)
def test_streams_and_graphs(dt):
    """On a stream of its own, and replayed from a graph: new inputs in the same memory, positions moving on."""
    from flash_stu_2_b200 import ops
    g, H, kv, hd, window = gen(4), 4, 4, 64, 100
    slots, slopes = ops.kv4_slots(window), slopes_of(H)
    prompt, cu = activations(g, 160, H, kv, hd, dt), cu_of((90, 70))
    tokens = [activations(g, 2, H, kv, hd, dt).view(2, 1, -1) for _ in range(4)]

    def run(packed, one):
        k4, v4 = ops.kv4_rings(2, slots, kv, hd, dev())
        pos = positions(0, 0)
        outs = [packed(prompt, k4, v4, pos)]
        for t in tokens:
            outs.append(one(t, k4, v4, pos))
        return outs, k4, v4, pos

    def packed(x, k4, v4, pos):
        y = ops.swa_packed(x, cu, slopes, H, window, 50.0)
        ops.kv4_write(x, k4, v4, pos, H, cu_seqlens=cu)
        return y

    def one(t, k4, v4, pos):
        return ops.kv4_step(t, k4, v4, pos, slopes, H, window, 50.0)

    want = run(packed, one)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(packed, one)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want[0], got[0])) and all(torch.equal(a, b) for a, b in zip(want[1:], got[1:]))

    held = {}

    def replayed(t, k4, v4, pos):
        if not held:
            held["t"], keep = t.clone(), (k4.clone(), v4.clone(), pos.clone())
            torch.cuda.synchronize()
            held["graph"] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(held["graph"]):
                held["out"] = one(held["t"], k4, v4, pos)
            for to, was in zip((k4, v4, pos), keep):
                assert torch.equal(to, was)      # (capturing runs nothing)
        held["t"].copy_(t)
        held["graph"].replay()
        return held["out"].clone()

    got = run(packed, replayed)
    assert all(torch.equal(a, b) for a, b in zip(want[0], got[0])) and all(torch.equal(a, b) for a, b in zip(want[1:], got[1:]))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("slopes", [(-0.25, -0.01, 0.0, 3.0), (40.0, -3.0, 0.5, 1e-6)])
def test_packed_takes_any_slopes(dt, slopes):
    """Slopes that lift far keys, and such as leave a row its own key alone."""
    from flash_stu_2_b200 import ops
    g, lengths = gen(21), (400, 130)
    qkv, sl = activations(g, 530, 4, 4, 64, dt), torch.tensor(slopes, device=dev())
    for window in (None, 300):
        want, tol = R.packed(qkv, lengths, 0, sl, 4, 4, window, 0.0, dt)
        R.check(ops.swa_packed(qkv, cu_of(lengths), sl, 4, window), want, tol)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("alibi", [False, True])
def test_packed_of_extreme_scores(dt, alibi):
    """Scores of thousands apart, larger ones behind smaller ones and before them: weights of 0 and 1, rows whose first keys are far above all that follow."""
    from flash_stu_2_b200 import ops
    g, H, hd, lengths = gen(22), 2, 64, (700, 65)
    for factor in (0.0, 30.0, 1000.0):
        qkv = activations(g, 765, H, H, hd, dt)
        qkv[:, :H * hd] *= factor
        for rising in (True, False):
            x = qkv.clone()
            ramp = torch.linspace(0.1, 1, 765, device=dev())
            x[:, H * hd:2 * H * hd] *= (ramp if rising else ramp.flip(0))[:, None].to(dt)
            slopes = slopes_of(H) if alibi else None
            want, tol = R.packed(x, lengths, 0, slopes, H, H, None, 0.0, dt)
            R.check(ops.swa_packed(x, cu_of(lengths), slopes, H), want, tol)


@pytest.mark.parametrize("cap", [1.0, 8.0, 40.0])
def test_packed_caps_of_every_size(cap):
    """Scores below a fifth of the cap, below half of it and above, in one tile and apart: each row by the form that its scores call for."""
    from flash_stu_2_b200 import ops
    g, H, hd, lengths = gen(23), 2, 128, (300, 200)
    qkv = activations(g, 500, H, H, hd, torch.bfloat16)
    qkv[100:, :H * hd] *= 0.02
    qkv[200:260, :H * hd] *= 10
    want, tol = R.packed(qkv, lengths, 0, slopes_of(H), H, H, 150, cap, torch.bfloat16)
    R.check(ops.swa_packed(qkv, cu_of(lengths), slopes_of(H), H, 150, cap), want, tol)


def test_offsets_past_32_bits():
    """Rows of qkv and rings behind more than 2^32 bytes."""
    from flash_stu_2_b200 import ops
    g, H, kv, hd, dt = gen(31), 12, 12, 128, torch.bfloat16
    N, tail = 720000, 300
    qkv = torch.zeros(N, (H + 2 * kv) * hd, device=dev(), dtype=dt)                  # 6.6 GB
    qkv[N - tail:] = activations(g, tail, H, kv, hd, dt)
    out = ops.swa_packed(qkv, cu_of([N - tail, tail]), slopes_of(H), H, 40, 50.0)
    alone = ops.swa_packed(qkv[N - tail:].clone(), cu_of([tail]), slopes_of(H), H, 40, 50.0)
    assert float((out[N - tail:].double() - alone.double()).norm() / alone.double().norm()) < 2.0 ** -7 and not bool(out[:N - tail].any())
    B, slots = 64, 80016
    k4, v4 = ops.kv4_rings(B, slots, kv, hd, dev())                                   # 4.4 GB each
    one = ops.kv4_rings(1, slots, kv, hd, dev())
    pos, pos1 = positions(*([slots - 3] * B)), positions(slots - 3)
    rows = activations(g, 8, H, kv, hd, dt)
    ops.kv4_write(rows.expand(B, 8, -1), k4, v4, pos, H)
    ops.kv4_write(rows[None], *one, pos1, H)
    new = activations(g, 1, H, kv, hd, dt)[None]
    got, want = ops.kv4_step(new.expand(B, 1, -1), k4, v4, pos, slopes_of(H), H, 100, 50.0), ops.kv4_step(new, *one, pos1, slopes_of(H), H, 100, 50.0)
    assert float((got[-1].double() - want[0].double()).norm() / want.double().norm()) < 2.0 ** -7
    assert torch.equal(k4[-1], one[0][0]) and torch.equal(v4[-1], one[1][0]) and torch.equal(k4[0], k4[-1])
    del qkv, out
    k, v = ops.kv4_read(k4[-2:], v4[-2:], hd, dt)
    k1, v1 = ops.kv4_read(*one, hd, dt)
    assert torch.equal(k[1:], k1) and torch.equal(v[1:], v1)
