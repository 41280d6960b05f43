"""Attention over packed prompts and over caches of 4 bits as a program calls them: cases that can be timed and compared.

  prompt   attention of whole prompts of different lengths, packed behind one another: causal, sliding window, ALiBi, soft cap, grouped heads
  store    the keys and values of packed prompts into rings of 4 bits, which are then read back as values (the next chunk of a prompt reads them so)
  read     rings of 4 bits as values
  step     attention of one new token per sequence over its ring of 4 bits; with `keep` the ring takes its key and value in

A ring [batch, kv heads, slots * row] of bytes holds for each slot a row of 4-bit numbers and, behind all rows, for each slot and piece of a row
its lowest value and its step, both bf16.  A row is 32, 64 or 128 numbers wide (the head's dimensions rounded up); more than 64 dimensions are two
pieces, 64 and the rest.  Of a row of one piece word i holds dimensions 8 i .. 8 i + 7, of two pieces word 2 i + p those of piece p, the first in
the lowest bits.  The token at position t is in slot t % slots.  The number n stands for lowest + n * step.  All arithmetic of a stored number is
defined in fp32, rounding by rounding: lowest = the piece's minimum rounded down to bf16, step = (maximum - lowest) * fp32(1/15) rounded up to
bf16, but at least 2^-126 where it is not 0, n = (x - lowest) * (1 / step) to the nearest even, in 0 .. 15.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------- the cases
def _prompt(name, heads, kv, hd, window, cap, alibi, dtype, lengths):
    return dict(name=name, kind="prompt", heads=heads, kv=kv, hd=hd, window=window, cap=cap, alibi=alibi, dtype=dtype, lengths=lengths)


def _step(name, heads, kv, hd, window, cap, alibi, dtype, batch, filled, keep):
    return dict(name=name, kind="step", heads=heads, kv=kv, hd=hd, window=window, cap=cap, alibi=alibi, dtype=dtype, batch=batch, filled=filled,
                keep=keep)


RAGGED = "2048,1311,77,640,1999,1024,333,5,1536,810,1,2047,129,256,1100,904"


def listed():
    return [
        # three short questions at once on the 24-layer model: latency is all that counts
        _prompt("prompt_tiny_bf16", 12, 12, 128, 1024, 50.0, True, "bf16", "7,1,19"),
        # the prefill of a serving batch: sixteen prompts of all lengths on the same model
        _prompt("prompt_batch_bf16", 12, 12, 128, 1024, 50.0, True, "bf16", RAGGED),
        # texts of odd lengths that are scored together, 12 heads of 64
        _prompt("prompt_score_bf16", 12, 12, 64, 512, 50.0, True, "bf16", "1999,37,2500,1,640,801,3333"),
        # one long document, every position sees all before it, eight query heads share a key head
        _prompt("prompt_long_bf16", 16, 2, 128, 0, 0.0, False, "bf16", "16384"),
        # the small fp32 model: two prompts
        _prompt("prompt_small_fp32", 8, 8, 64, 512, 50.0, True, "fp32", "128,700"),
        # the keys and values of that serving batch into the layer's rings
        dict(name="store_batch_bf16", kind="store", heads=12, kv=12, hd=128, window=1024, dtype="bf16", lengths=RAGGED),
        # heads of an odd size, prompts shorter and longer than the ring
        dict(name="store_odd_fp32", kind="store", heads=6, kv=3, hd=40, window=127, dtype="fp32", lengths="3,1,250"),
        # the rings of 32 conversations, read back ahead of the next chunk of their prompts
        dict(name="read_batch_bf16", kind="read", heads=12, kv=12, hd=128, window=1024, dtype="bf16", batch=32),
        # one interactive conversation: a token's latency
        _step("step_one_bf16", 12, 12, 128, 1024, 50.0, True, "bf16", 1, 5000, True),
        # a token of 32 conversations
        _step("step_batch_bf16", 12, 12, 128, 1024, 50.0, True, "bf16", 32, 5000, True),
        # a token of 64 long conversations with grouped heads
        _step("step_long_bf16", 16, 2, 128, 16384, 0.0, False, "bf16", 64, 20000, True),
        # two sequences of the small fp32 model near their beginning, a candidate token that is looked at and not kept
        _step("step_small_fp32", 8, 8, 64, 512, 50.0, True, "fp32", 2, 137, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges.  None does more work than the long ones above."""
    kind = rng.choice(["prompt", "prompt", "prompt", "store", "read", "step", "step", "step"])
    hd = rng.choice([64, 64, 128, 128, 128, 8 * rng.randint(2, 16)])
    kv = rng.choice([1, 2, 3, 4, 8, 12])
    heads = kv * rng.choice([1, 1, 2, 4, 5, 8])
    c = dict(kind=kind, heads=heads, kv=kv, hd=hd, window=_log(rng, 16, 8192), dtype=rng.choice(["bf16", "bf16", "bf16", "fp32"]))
    if kind in ("prompt", "step"):
        c.update(cap=rng.choice([0.0, 50.0, 50.0]), alibi=rng.random() < 0.7)
    if kind in ("prompt", "store"):
        longest = _log(rng, 1, 8192 if c["dtype"] == "bf16" else 1500)
        most, lengths = 3 * 10 ** 11, []
        for _ in range(_log(rng, 1, 24)):
            n = max(1, min(longest, int(longest * (0.05 + rng.random()))))
            # (the plain form computes every sequence as long as the longest, for all pairs)
            if (len(lengths) + 1) * longest ** 2 * heads > 4 * 10 ** 9 or 2 * heads * hd * longest ** 2 * (len(lengths) + 1) > most:
                break
            lengths.append(n)
        c["lengths"] = ",".join(map(str, lengths or [min(longest, 512)]))
        if kind == "prompt" and rng.random() < 0.2:
            c["window"] = 0
    else:
        slots = c["window"] + 1
        c["batch"] = max(1, min(_log(rng, 1, 64), 2 * 10 ** 9 // (slots * kv * hd * 8)))
    if kind == "step":
        c["keep"] = rng.random() < 0.7
        c["filled"] = slots + 15 + rng.randrange(5000) if c["keep"] else _log(rng, 1, 2 * slots)   # (a ring that is not full would fill up from pass to pass)
    return c


# ---------------------------------------------------------------------------------------------------- rings in elementary operations
def _slots(case):
    return -(-(case["window"] + 1) // 16) * 16


def _row(hd):
    """(numbers in a row, pieces)"""
    return (32 if hd <= 32 else 64 if hd <= 64 else 128), (2 if hd > 64 else 1)


def _bf16_toward(x, up):
    """fp32 x rounded to bf16 upwards or downwards, in fp32."""
    bits = x.contiguous().view(torch.int32)
    cut = bits & -65536
    away = (bits != cut) & ((bits >= 0) == up)
    return torch.where(away, cut + 65536, cut).view(torch.float32)


def _quantized(x):
    """fp32 x [..., hd] -> (rows of bytes [..., width / 2], scales of bytes [..., 4 * pieces])"""
    hd = x.shape[-1]
    width, pieces = _row(hd)
    cells = torch.nn.functional.pad(x, (0, width - hd)).unflatten(-1, (pieces, width // pieces))
    there = (torch.arange(width, device=x.device) < hd).view(pieces, -1)
    low = _bf16_toward(torch.where(there, cells, math.inf).amin(-1), False)
    high = torch.where(there, cells, -math.inf).amax(-1)
    step = _bf16_toward((high - low) * torch.tensor(1 / 15, dtype=torch.float32, device=x.device), True)
    step = torch.where(step > 0, step.clamp(min=2.0 ** -126), step)
    bad = ~(torch.isfinite(low) & torch.isfinite(step) & torch.isfinite(cells).all(-1))
    low, step = torch.where(bad, math.nan, low), torch.where(bad, 0.0, step)
    inverse = torch.where(step > 0, 1 / step, 0.0)
    n = torch.round((cells - low[..., None]) * inverse[..., None]).clamp(0, 15)
    n = torch.where(bad[..., None] | ~there, 0.0, n).to(torch.uint8)
    rows = n[..., 0::2] | n[..., 1::2] << 4                                   # [..., pieces, bytes]
    rows = rows.unflatten(-1, (-1, 4)).transpose(-3, -2).flatten(-3)           # words of the pieces in turn
    return rows, torch.stack([low, step], -1).to(torch.bfloat16).view(torch.uint8).flatten(-2)


def _parts(ring, hd):
    """(rows [B, kv, slots, bytes], scales [B, kv, slots, 4 * pieces]) of a ring, as views."""
    width, pieces = _row(hd)
    slots = ring.shape[2] // (width // 2 + 4 * pieces)
    cut = slots * (width // 2)
    return ring[:, :, :cut].unflatten(2, (slots, width // 2)), ring[:, :, cut:].unflatten(2, (slots, 4 * pieces))


def _values(ring, hd):
    """What a ring stands for, fp32 [B, kv, slots, hd]."""
    width, pieces = _row(hd)
    rows, scales = _parts(ring, hd)
    words = rows.unflatten(-1, (-1, pieces, 4)).transpose(-3, -2).flatten(-2)   # [..., pieces, bytes]
    n = torch.stack([words & 15, words >> 4], -1).flatten(-2).float()
    s = scales.contiguous().view(torch.bfloat16).float().unflatten(-1, (pieces, 2))
    return (s[..., 0:1] + n * s[..., 1:2]).flatten(-2)[..., :hd]


# ---------------------------------------------------------------------------------------------------- state
def _activations(gen, rows, case):
    """Queries, keys and values of a layer: keys with channels of their own level, some of them far off, scores of a few units."""
    H, kv, hd = case["heads"], case["kv"], case["hd"]
    q = 1.5 * torch.randn(rows, H * hd, device="cuda", generator=gen)
    level = torch.randn(kv * hd, device="cuda", generator=gen)
    level[torch.randint(kv * hd, (max(1, kv * hd // 50),), device="cuda", generator=gen)] *= 4
    k = torch.randn(rows, kv * hd, device="cuda", generator=gen) + level
    v = torch.randn(rows, kv * hd, device="cuda", generator=gen) * torch.exp(0.3 * torch.randn(rows, 1, device="cuda", generator=gen))
    return torch.cat([q, k, v], 1).to(DTYPES[case["dtype"]])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s, kind, H, kv, hd = {"case": case}, case["kind"], case["heads"], case["kv"], case["hd"]
    width, pieces = _row(hd)
    if kind in ("prompt", "store"):
        lengths = [int(n) for n in case["lengths"].split(",")]
        s["longest"] = max(lengths)
        s["cu"] = torch.tensor([0] + lengths, device="cuda").cumsum(0).to(torch.int32)
        s["qkv"] = _activations(gen, sum(lengths), case)
    if kind in ("prompt", "step"):
        s["slopes"] = 0.25 * 2.0 ** (-8 * torch.arange(1, H + 1, device="cuda", dtype=torch.float32) / H) if case["alibi"] else None
    batch = len(lengths) if kind == "store" else case.get("batch", 0)
    if batch:
        shape = (batch, kv, _slots(case) * (width // 2 + 4 * pieces))
        s["pos"] = torch.zeros(batch, 2, dtype=torch.int32, device="cuda")
        s["k4"], s["v4"] = (torch.zeros(shape, dtype=torch.uint8, device="cuda") for _ in range(2))
    if kind in ("read", "step"):   # full rings, whatever `filled` says: what lies behind the filled part is never looked at
        for b in range(batch):
            one = _activations(gen, _slots(case), case).float()[:, H * hd:].view(-1, 2, kv, hd)
            for i, name in enumerate(("k4", "v4")):
                for part, made in zip(_parts(s[name], hd), _quantized(one[:, i].transpose(0, 1).contiguous())):
                    part[b] = made
        s["qkv"] = _activations(gen, batch, case).view(batch, 1, -1)
    if kind == "step":   # sequences of a batch stand at different positions
        s["pos"][:, 0] = case["filled"]
        if case["keep"]:
            s["pos"][:, 0] += torch.randint(1000, (batch,), device="cuda", generator=gen, dtype=torch.int32)
    return s


# ---------------------------------------------------------------------------------------------------- one pass
def _split(qkv, case):
    """fp32 q [..., heads, hd], k, v [..., kv, hd]"""
    H, kv, hd = case["heads"], case["kv"], case["hd"]
    rows = qkv.float().unflatten(-1, (H + 2 * kv, hd))
    return rows[..., :H, :], rows[..., H:H + kv, :], rows[..., H + kv:, :]


def _softmax_rows(s, case, bias, there):
    """Scores s [..., queries, keys] -> weights, in place."""
    s *= 1 / math.sqrt(case["hd"])
    if case["cap"]:
        s.mul_(1 / case["cap"]).tanh_().mul_(case["cap"])
    if bias is not None:
        s -= bias
    s.masked_fill_(~there, -math.inf)
    s -= s.amax(-1, keepdim=True)
    s.exp_()
    s /= s.sum(-1, keepdim=True)
    return s


def _plain_prompt(s):
    case = s["case"]
    H, kv, hd, T = case["heads"], case["kv"], case["hd"], s["longest"]
    cu = s["cu"].long()
    at = torch.arange(T, device="cuda")
    inside = at < (cu[1:] - cu[:-1])[:, None]                                                  # [S, T]
    rows = torch.where(inside, cu[:-1, None] + at, 0)
    q, k, v = _split(s["qkv"][rows], case)                                                     # [S, T, heads, hd]
    q = q.permute(0, 2, 1, 3).reshape(-1, kv, H // kv * T, hd)
    scores = (q @ k.permute(0, 2, 3, 1)).unflatten(2, (H // kv, T))                            # [S, kv, heads of one, T, T]
    behind = at[:, None] - at
    there = behind >= 0
    if case["window"]:
        there = there & (behind <= case["window"])
    bias = None if s["slopes"] is None else s["slopes"].view(kv, H // kv, 1, 1) * behind
    w = _softmax_rows(scores, case, bias, there)
    o = (w.flatten(2, 3) @ v.permute(0, 2, 1, 3)).view(-1, H, T, hd).permute(0, 2, 1, 3)       # [S, T, H, hd]
    return o[inside].flatten(1).to(s["qkv"].dtype)


def _plain_store(s):
    case = s["case"]
    cu, slots = s["cu"].long(), _slots(case)
    at = torch.arange(slots, device="cuda")
    end = cu[1:] - cu[:-1]
    last = end[:, None] - 1 - (end[:, None] - 1 - at) % slots                                  # the last position that is in this slot
    written = last >= 0
    _, k, v = _split(s["qkv"][torch.where(written, cu[:-1, None] + last, 0)], case)            # [S, slots, kv, hd]
    for name, x in (("k4", k), ("v4", v)):
        for part, made in zip(_parts(s[name], case["hd"]), _quantized(x.transpose(1, 2).contiguous())):
            part.copy_(torch.where(written[:, None, :, None], made, part))
    s["pos"].zero_()
    s["pos"][:, 0] += end
    return _plain_read(s)


def _plain_read(s):
    case = s["case"]
    return tuple(_values(s[name], case["hd"]).transpose(1, 2).flatten(2).to(DTYPES[case["dtype"]]) for name in ("k4", "v4"))


def _plain_step(s):
    case = s["case"]
    H, kv, hd, slots = case["heads"], case["kv"], case["hd"], _slots(case)
    q, k, v = _split(s["qkv"][:, 0], case)                                                     # [B, heads, hd]
    t = s["pos"][:, :1].long()
    behind = (t - 1 - torch.arange(slots, device="cuda")) % slots + 1                          # [B, slots]: how far behind the new token
    there = (behind <= t) & (behind <= case["window"])
    behind, there = (torch.cat([x, x.new_full((len(t), 1), y)], 1) for x, y in ((behind, 0), (there, True)))
    keys, values = (torch.cat([_values(s[name], hd), x[:, :, None]], 2) for name, x in (("k4", k), ("v4", v)))
    scores = q.view(-1, kv, H // kv, hd) @ keys.transpose(2, 3)                                # [B, kv, heads of one, slots + 1]
    bias = None if s["slopes"] is None else s["slopes"].view(kv, H // kv, 1) * behind[:, None, None]
    w = _softmax_rows(scores, case, bias, there[:, None, None])
    o = (w @ values).view(-1, 1, H * hd).to(s["qkv"].dtype)
    if case["keep"]:
        which = torch.arange(len(t), device="cuda")
        for name, x in (("k4", k), ("v4", v)):
            for part, made in zip(_parts(s[name], hd), _quantized(x)):
                part[which, :, t[:, 0] % slots] = made
        s["pos"][:, 0] += 1
    return o


def _own(s):
    from flash_stu_2_b200 import ops
    case = s["case"]
    kind, H, kv, hd = case["kind"], case["heads"], case["kv"], case["hd"]
    if kind == "prompt":
        return ops.swa_packed(s["qkv"], s["cu"], s["slopes"], H, case["window"] or None, case["cap"], kv_heads=kv)
    if kind == "step":
        return ops.kv4_step(s["qkv"], s["k4"], s["v4"], s["pos"], s["slopes"], H, case["window"], case["cap"], update_cache=case["keep"])
    if kind == "store":
        s["pos"].zero_()
        ops.kv4_write(s["qkv"], s["k4"], s["v4"], s["pos"], H, cu_seqlens=s["cu"])
    return ops.kv4_read(s["k4"], s["v4"], hd, DTYPES[case["dtype"]])


def run(state):
    if own:
        out = _own(state)
    else:
        out = {"prompt": _plain_prompt, "store": _plain_store, "read": _plain_read, "step": _plain_step}[state["case"]["kind"]](state)
    if state["case"]["kind"] == "step" and state["case"]["keep"]:
        # the rings as they are held (the bytes: their arithmetic is defined to the last bit, and a program has no use for them as values here)
        return out, state["k4"], state["v4"], state["pos"]
    return out


def _pairs(n, window):
    """Keys that n queries of one sequence see together."""
    w = min(window or n, n)
    return w * (w + 1) // 2 + (n - w) * (w + 1) if w < n else n * (n + 1) // 2


def work(case):
    H, kv, hd = case["heads"], case["kv"], case["hd"]
    size = 4 if case["dtype"] == "fp32" else 2
    held = 2 * kv * (hd / 2 + 4 * _row(hd)[1])          # a token's key and value in 4 bits
    exact = 2 * kv * hd * size                          # ... as values
    if case["kind"] in ("prompt", "store"):
        lengths = [int(n) for n in case["lengths"].split(",")]
    if case["kind"] == "prompt":
        return {"bytes": sum(lengths) * (2 * H + 2 * kv) * hd * size, "flops": 4 * H * hd * sum(_pairs(n, case["window"]) for n in lengths)}
    slots = _slots(case)
    if case["kind"] == "store":
        kept = sum(min(n, slots) for n in lengths)
        return {"bytes": kept * (exact + held) + len(lengths) * slots * (held + exact), "flops": 8 * kept * 2 * kv * hd}
    if case["kind"] == "read":
        return {"bytes": case["batch"] * slots * (held + exact), "flops": 2 * case["batch"] * slots * 2 * kv * hd}
    keys = min(case["filled"], case["window"])
    return {"bytes": case["batch"] * (keys * held + (2 * H + 2 * kv) * hd * size + (held if case["keep"] else 0)),
            "flops": 4 * case["batch"] * H * hd * (keys + 1)}


# ---------------------------------------------------------------------------------------------------- the definition, in 64 bits
def _exact_numbers(x):
    """One piece, float64 [..., dims] of fp32 numbers -> (lowest, step, n): every rounding that the definition names, made from 64 bits."""
    def toward(v, direction):
        m, e = torch.frexp(v)
        return torch.ldexp(direction(m * 256) / 256, e)

    low = toward(x.min(-1, keepdim=True).values, torch.floor)
    spread = (x.max(-1, keepdim=True).values - low).float().double()
    step = toward((spread * float(torch.tensor(1 / 15, dtype=torch.float32))).float().double(), torch.ceil)
    step = torch.where(step > 0, torch.maximum(step, torch.full_like(step, 2.0 ** -126)), step)
    inverse = torch.where(step > 0, (1 / step).float().double(), 0.0)
    scaled = ((x - low).float().double() * inverse).float().double()
    return low, step, torch.round(scaled).clamp(0, 15)


def _exact_back(x):
    """What a key or a value [..., hd] stands for once it has been in a ring."""
    out = []
    for piece in x.split(64, dim=-1):
        low, step, n = _exact_numbers(piece)
        out.append(low + step * n)
    return torch.cat(out, -1)


def _exact_values(ring, case):
    """A ring as float64 [B, kv, slots, hd], number by number."""
    hd, slots = case["hd"], _slots(case)
    width, pieces = (128, 2) if hd > 64 else (64, 1) if hd > 32 else (32, 1)
    words = ring[:, :, :slots * width // 2].long().reshape(*ring.shape[:2], slots, width // 8, 4)
    words = sum(words[..., i] << 8 * i for i in range(4))                      # [B, kv, slots, words of a row]
    scales = ring[:, :, slots * width // 2:].long().reshape(*ring.shape[:2], slots, pieces, 2, 2)
    bits = (scales[..., 0] | scales[..., 1] << 8)
    power = torch.where((bits >> 7 & 255) > 0, (bits >> 7 & 255) - 134, -133)
    whole = torch.where((bits >> 7 & 255) > 0, (bits & 127) + 128, bits & 127)
    scales = (1 - 2 * (bits >> 15)).double() * torch.ldexp(whole.double(), power)
    out = []
    for c in range(hd):
        piece = c // 64
        word = (c % 64) // 8 * pieces + piece
        out.append(scales[..., piece, 0] + scales[..., piece, 1] * (words[..., word] >> 4 * (c % 8) & 15).double())
    return torch.stack(out, -1)


def _exact_attention(q, k, v, slope, behind, case):
    """q [n, hd], k, v [m, hd], behind [n, m] (below 0 or past the window: not seen)."""
    z = q @ k.T / case["hd"] ** 0.5
    if case["cap"]:
        z = case["cap"] * torch.tanh(z / case["cap"])
    z = z - slope * behind
    seen = behind >= 0
    if case["window"]:
        seen &= behind <= case["window"]
    return torch.softmax(torch.where(seen, z, -math.inf), 1) @ v


def exact(case, seed):
    s = prepare(case, seed)
    kind, H, kv, hd, dtype = case["kind"], case["heads"], case["kv"], case["hd"], DTYPES[case["dtype"]]
    if kind == "read":
        return tuple(_exact_values(s[n], case).transpose(1, 2).reshape(case["batch"], _slots(case), kv * hd) for n in ("k4", "v4"))
    x = s["qkv"].double().reshape(-1, H + 2 * kv, hd)
    if kind == "store":
        slots, lengths = _slots(case), [int(n) for n in case["lengths"].split(",")]
        out, first = torch.zeros(2, len(lengths), slots, kv, hd, dtype=torch.float64, device="cuda"), 0
        for i, n in enumerate(lengths):
            t = torch.arange(max(0, n - slots), n, device="cuda")
            for j in range(2):
                out[j, i, t % slots] = _exact_back(x[first + t, H + j * kv:H + (j + 1) * kv])
            first += n
        return tuple(out.flatten(3))
    slopes = [0.0] * H if s["slopes"] is None else s["slopes"].double().tolist()
    if kind == "prompt":
        out, first = torch.empty(x.shape[0], H, hd, dtype=torch.float64, device="cuda"), 0
        for n in map(int, case["lengths"].split(",")):
            for a in range(0, n, 2048):   # queries a .. b - 1, and the keys that any of them sees
                b = min(n, a + 2048)
                lo = max(0, a - case["window"]) if case["window"] else 0
                behind = torch.arange(a, b, device="cuda")[:, None] - torch.arange(lo, b, device="cuda")
                for h in range(H):
                    g = h * kv // H
                    k, v = (x[first + lo:first + b, H + j * kv + g] for j in range(2))
                    out[first + a:first + b, h] = _exact_attention(x[first + a:first + b, h], k, v, slopes[h], behind, case)
            first += n
        return out.flatten(1)
    slots, out = _slots(case), torch.empty(case["batch"], 1, H * hd, dtype=torch.float64, device="cuda")
    for b, t in enumerate(s["pos"][:, 0].tolist()):
        j = torch.arange(max(0, t - case["window"]), t, device="cuda")
        behind = torch.cat([t - j, j.new_zeros(1)])[None]
        one = {n: _exact_values(s[n][b:b + 1], case)[0][:, j % slots] for n in ("k4", "v4")}
        for h in range(H):
            g = h * kv // H
            k, v = (torch.cat([one[n][g], x[b, H + i * kv + g][None]]) for i, n in enumerate(("k4", "v4")))
            out[b, 0, h * hd:(h + 1) * hd] = _exact_attention(x[b, h][None], k, v, slopes[h], behind, case)[0]
    return (out, None, None, None) if case["keep"] else out
