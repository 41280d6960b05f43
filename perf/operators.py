"""The 8-bit operators of the MLP as a program calls them: cases that can be timed and compared.

  quantize   rows to e4m3 with a power-of-two scale for each 128 of a row
  norm       RMSNorm of a residual stream, with or without a branch that is added to it first, to e4m3 rows
  linear     product of two e4m3 operands, alone or added to a residual stream
  gate       GELU(x gate^T) * (x up^T), to e4m3 rows
  mlp        all of them as a layer runs them: x += branch; norm; gate; down projection onto x

Rows of 8-bit values are two tensors, as the framework holds them: the values [rows, columns rounded up to 128], zero behind the columns, and
the scales [rows / 128, columns / 512, 32, 4, 4] (both rounded up): that of row 128 a + 32 b + c and block 4 g + j is at [a, g, c, b, j], 2^-127
(byte 0) where there is no such row or block.
"""
import math

import torch

own = False

EPS = float(torch.finfo(torch.float32).eps)
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # weights of a gate projection on their way into a served model, once per model: fp32 master copies
        dict(name="quantize_weights_fp32", kind="quantize", rows=6144, cols=1536, dtype="fp32"),
        # activations of an odd width that come from elsewhere: four texts of 1999 tokens
        dict(name="quantize_ragged_bf16", kind="quantize", rows=7996, cols=1111, dtype="bf16"),
        # one token of an interactive conversation: latency is all that counts
        dict(name="norm_one_bf16", kind="norm", rows=1, cols=1536, dtype="bf16", add=False),
        # the prefill of 8 sequences of 8192 tokens: attention's branch joins the stream on its way to the MLP
        dict(name="norm_add_prefill_bf16", kind="norm", rows=65536, cols=1024, dtype="bf16", add=True),
        # fp32 stream of an odd width
        dict(name="norm_ragged_fp32", kind="norm", rows=1999, cols=1000, dtype="fp32", add=True),
        # gate and up of one token: weights are streamed once for one row
        dict(name="gate_one", kind="gate", rows=1, cols=1024, out=4096),
        # the same for a serving batch of 32 sequences on the 24-layer model
        dict(name="gate_batch", kind="gate", rows=32, cols=1536, out=6144),
        # the prefill of a batch: 32 prompts of 512 tokens, bound by the tensor cores
        dict(name="gate_prefill", kind="gate", rows=16384, cols=1536, out=6144),
        # down projection of a token step, 8 sequences, over the longest rows (MLP of 12 times the width)
        dict(name="down_batch", kind="linear", rows=8, cols=18432, out=1536, resid=True),
        # one prompt of 333 tokens through matrices of odd sizes
        dict(name="linear_ragged", kind="linear", rows=333, cols=1000, out=1111, resid=False),
        # down projection of a prefill over the longest rows
        dict(name="down_prefill", kind="linear", rows=8192, cols=18432, out=1536, resid=True),
        # a layer's MLP in a token step of 32 sequences, the three calls behind one another
        dict(name="mlp_step", kind="mlp", rows=32, cols=1536, out=18432),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A width: mostly the multiples of 128 that models have, else any number."""
    n = _log(rng, lo, hi)
    return max(128, n // 128 * 128) if rng.random() < 0.6 else n


def draw(rng):
    """One more case of the same ranges.  None does more work than the prefills above."""
    kind = rng.choice(["quantize", "norm", "norm", "linear", "linear", "gate", "gate", "mlp"])
    if kind == "quantize":
        return dict(kind=kind, rows=_log(rng, 1, 8192), cols=_size(rng, 32, 8192), dtype=rng.choice(["bf16", "fp32"]))
    if kind == "norm":
        return dict(kind=kind, rows=_log(rng, 1, 8192), cols=_size(rng, 64, 4096), dtype=rng.choice(["bf16", "bf16", "fp32"]),
                    add=rng.random() < 0.5)
    c = dict(kind=kind, rows=_log(rng, 1, 8192), cols=_size(rng, 100, 4096), out=_size(rng, 100, 8192))
    products = {"linear": 1, "gate": 2, "mlp": 3}[kind]
    c["rows"] = min(c["rows"], 3 * 10 ** 11 // (products * c["cols"] * c["out"]))
    if kind == "linear":
        c["resid"] = rng.random() < 0.5
        if rng.random() < 0.5:
            c["cols"], c["out"] = c["out"], c["cols"]
    return c


# ---------------------------------------------------------------------------------------------------- 8-bit rows in elementary operations
def _up(n, m):
    return -(-n // m) * m


def _power(e):
    """2^e in fp32 for whole -127 <= e <= 127, from its bits."""
    return torch.where(e > -127, (e.to(torch.int32) + 127) << 23, 1 << 22).view(torch.float32)


def _quantized(v):
    """fp32 v [rows, cols] -> (values, scales) in the layout above."""
    rows, cols = v.shape
    v = torch.nn.functional.pad(v, (0, _up(cols, 128) - cols)).view(rows, -1, 128)
    finite = torch.isfinite(v)
    amax = torch.where(finite, v.abs(), 0).amax(dim=2)
    # amax = m * 2^x with 0.5 <= m < 1; 448 = 0.875 * 2^9
    m, x = torch.frexp(amax)
    e = torch.where(amax == 0, -127, x - 9 + (m > 0.875).to(x.dtype)).clamp(min=-127)
    q = torch.where(finite, v * _power(-e)[:, :, None], math.nan).to(torch.float8_e4m3fn).view(rows, -1)
    b = torch.nn.functional.pad((e + 127).to(torch.uint8), (0, _up(e.shape[1], 4) - e.shape[1], 0, _up(rows, 128) - rows))
    b = b.view(b.shape[0] // 128, 4, 32, -1, 4).permute(0, 3, 2, 1, 4).contiguous()
    return q, b.view(torch.float8_e8m0fnu)


def _scales_by_row(scales, rows, blocks):
    b = scales.view(torch.uint8).permute(0, 3, 2, 1, 4)
    return b.reshape(b.shape[0] * 128, -1)[:rows, :blocks].to(torch.int32)


def _values(q, scales, cols):
    """What 8-bit rows stand for, in fp32."""
    e = _scales_by_row(scales, q.shape[0], q.shape[1] // 128) - 127
    return (q.float().view(q.shape[0], -1, 128) * _power(e)[:, :, None]).view(q.shape)[:, :cols]


def _gelu(x):
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))


def _norm(x, weight, add):
    """-> (sum in the stream's type, normalised in fp32)"""
    s = x if add is None else (x.float() + add.float()).to(x.dtype)
    v = s.float()
    return s, v * torch.rsqrt(v.square().mean(dim=1, keepdim=True) + EPS) * weight.float()


# ---------------------------------------------------------------------------------------------------- state
def _stream(gen, rows, cols, dtype):
    """A residual stream: a few channels far above the others, rows of different sizes."""
    wide = torch.exp(0.5 * torch.randn(cols, device="cuda", generator=gen))
    wide[torch.randint(cols, (max(1, cols // 200),), device="cuda", generator=gen)] *= 20
    tall = torch.exp(0.3 * torch.randn(rows, 1, device="cuda", generator=gen))
    return (torch.randn(rows, cols, device="cuda", generator=gen) * wide * tall).to(dtype)


def _weight(gen, out, cols):
    return torch.randn(out, cols, device="cuda", generator=gen) * (torch.exp(0.2 * torch.randn(out, 1, device="cuda", generator=gen)) / math.sqrt(cols))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, rows, cols = case["kind"], case["rows"], case["cols"]
    dtype = DTYPES[case.get("dtype", "bf16")]
    s = {"case": case}
    if kind == "quantize":
        s["x"] = _stream(gen, rows, cols, dtype)
    if kind in ("norm", "mlp"):
        s["x"] = _stream(gen, rows, cols, dtype)
        s["weight"] = (1 + 0.1 * torch.randn(cols, device="cuda", generator=gen)).to(dtype)
        s["add"] = (0.5 * torch.randn(rows, cols, device="cuda", generator=gen)).to(dtype) if case.get("add", True) else None
        s["sum"] = torch.empty_like(s["x"])   # where x + add goes
    if kind in ("linear", "gate"):
        s["a"] = _quantized(_stream(gen, rows, cols, torch.float32))
        s["w"] = _quantized(_weight(gen, case["out"], cols))
        s["w2"] = _quantized(_weight(gen, case["out"], cols)) if kind == "gate" else None
        s["resid"] = _stream(gen, rows, case["out"], torch.bfloat16) if case.get("resid") else None
    if kind == "mlp":
        s["w"] = _quantized(_weight(gen, case["out"], cols))
        s["w2"] = _quantized(_weight(gen, case["out"], cols))
        s["down"] = _quantized(_weight(gen, cols, case["out"]))
    return s


# ---------------------------------------------------------------------------------------------------- one pass
def _linear(a, w, cols, resid):
    y = _values(*a, cols) @ _values(*w, cols).T
    return y.to(torch.bfloat16) if resid is None else (resid.float() + y.to(torch.bfloat16).float()).to(torch.bfloat16)


def _gate(a, w, w2, cols):
    v = _values(*a, cols)
    return _quantized(_gelu(v @ _values(*w, cols).T) * (v @ _values(*w2, cols).T))


def _plain(s):
    case = s["case"]
    kind, cols = case["kind"], case["cols"]
    if kind == "quantize":
        return _quantized(s["x"].float())
    if kind == "linear":
        return _linear(s["a"], s["w"], cols, s["resid"])
    if kind == "gate":
        return _gate(s["a"], s["w"], s["w2"], cols)
    total, v = _norm(s["x"], s["weight"], s["add"])
    q = _quantized(v)
    if kind == "norm":
        return (*q, total) if s["add"] is not None else q
    h = _gate(q, s["w"], s["w2"], cols)
    return _linear(h, s["down"], case["out"], total)


def _own(s):
    from flash_stu_2_b200 import ops
    case = s["case"]
    kind, cols = case["kind"], case["cols"]
    if kind == "quantize":
        q = ops.quantize_fp8(s["x"])
        return q.data, q.scales
    if kind == "linear":
        return ops.linear_fp8(ops.Fp8Rows(*s["a"], cols), ops.Fp8Rows(*s["w"], cols), resid=s["resid"])
    if kind == "gate":
        h = ops.linear_fp8(ops.Fp8Rows(*s["a"], cols), ops.Fp8Rows(*s["w"], cols), W2=ops.Fp8Rows(*s["w2"], cols))
        return h.data, h.scales
    total = s["x"] if s["add"] is None else s["sum"]
    q = ops.rmsnorm_fp8(s["x"], s["weight"], EPS, add=s["add"], out=s["sum"] if s["add"] is not None else None)
    if kind == "norm":
        return (q.data, q.scales, total) if s["add"] is not None else (q.data, q.scales)
    h = ops.linear_fp8(q, ops.Fp8Rows(*s["w"], cols), W2=ops.Fp8Rows(*s["w2"], cols))
    return ops.linear_fp8(h, ops.Fp8Rows(*s["down"], case["out"]), resid=total)


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    kind, rows, cols = case["kind"], case["rows"], case["cols"]

    def held(r, c):
        return r * (_up(c, 128) + _up(c, 128) // 128)

    size = 4 if case.get("dtype") == "fp32" else 2
    if kind == "quantize":
        return {"bytes": rows * cols * size + held(rows, cols), "flops": 3 * rows * cols}
    norm = rows * cols * size * (3 if case.get("add", True) else 1) + cols * size
    if kind == "norm":
        return {"bytes": norm + held(rows, cols), "flops": 7 * rows * cols}
    out = case["out"]
    if kind == "linear":
        return {"bytes": held(rows, cols) + held(out, cols) + rows * out * (4 if case["resid"] else 2), "flops": 2 * rows * cols * out}
    if kind == "gate":
        return {"bytes": held(rows, cols) + 2 * held(out, cols) + held(rows, out), "flops": 4 * rows * cols * out}
    # (the rows between the calls are small against L2; they are not counted)
    return {"bytes": 3 * rows * cols * 2 + 3 * held(out, cols), "flops": 6 * rows * cols * out}


# ---------------------------------------------------------------------------------------------------- the definition, in 64 bits
def _exact_power(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_rows(v):
    """Rows as 8-bit values and scales: every block's power of two by counting, every value to the nearest of the format's numbers."""
    rows, cols = v.shape
    blocks, groups = -(-cols // 128), -(-cols // 512)
    full = v.new_zeros(rows, blocks * 128)
    full[:, :cols] = v
    cells = full.reshape(rows * blocks, 128)
    good = (cells == cells) & (cells.abs() != math.inf)
    top = (cells.abs() * good).nan_to_num(0.0, 0.0).max(dim=1).values
    e = torch.ceil(torch.log2((top / 448).clamp(min=2.0 ** -140))).clamp(min=-127)
    e = e + (top > 448 * _exact_power(e)).double()            # (a logarithm that came out a hair low or high)
    e = (e - (top <= 448 * _exact_power(e - 1)).double()).clamp(min=-127)
    z = cells * _exact_power(-e)[:, None]
    step = _exact_power(torch.frexp(z.abs().clamp(min=2.0 ** -6)).exponent - 4)   # between neighbours of the format
    q = torch.where(good, torch.round(z / step) * step, math.nan).reshape(rows, blocks * 128)
    s = v.new_full((-(-rows // 128) * 128, groups * 4), 2.0 ** -127)
    s[:rows, :blocks] = _exact_power(e).reshape(rows, blocks)
    return q, torch.stack([torch.stack([s[128 * a:128 * a + 128, 4 * g:4 * g + 4].reshape(4, 32, 4).transpose(0, 1) for g in range(groups)])
                           for a in range(s.shape[0] // 128)])


def _exact_product(a, w, cols):
    def opened(q, scales):
        r, groups = q.shape[0], scales.shape[1]
        s = scales.double().permute(0, 3, 2, 1, 4).reshape(-1, 4 * groups)
        return (q.double() * s[:r].repeat_interleave(128, dim=1)[:, :q.shape[1]])[:, :cols]
    return opened(*a) @ opened(*w).mT


def exact(case, seed):
    s = prepare(case, seed)
    kind, cols = case["kind"], case["cols"]

    def gate(a):
        g, u = _exact_product(a, s["w"], cols), _exact_product(a, s["w2"], cols)
        return _exact_rows(g / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * u)   # tanh as a quotient of exponentials

    if kind == "quantize":
        return _exact_rows(s["x"].double())
    if kind == "linear":
        y = _exact_product(s["a"], s["w"], cols)
        return y if s["resid"] is None else y + s["resid"].double()
    if kind == "gate":
        return gate(s["a"])
    x = s["x"].double()
    if s["add"] is not None:
        x = (x + s["add"].double()).to(s["x"].dtype).double()   # the stream is held in its own type
    q = _exact_rows(x / torch.sqrt((x * x).sum(dim=1, keepdim=True) / cols + EPS) * s["weight"].double())
    if kind == "norm":
        return (*q, x) if s["add"] is not None else q
    return x + _exact_product(gate(q), s["down"], case["out"])
