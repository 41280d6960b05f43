"""Rows of 8-bit values, their norm and their products against the definitions in 64 bits (fp8_reference.py says what each may be off)."""
import pytest
import torch

import fp8_reference as R

pytestmark = pytest.mark.gpu

BF16_HALF = torch.finfo(torch.bfloat16).eps / 2
SHAPES = [(1, 128), (1, 1), (3, 100), (5, 512), (127, 129), (128, 513), (130, 1111), (300, 640), (2, 5000), (1, 18432)]


def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


def gen(seed):
    return torch.Generator(device=dev()).manual_seed(seed)


def stream(g, rows, cols, dt):
    """Values over many powers of two, blocks of zeros among them."""
    x = torch.randn(rows, cols, device=dev(), generator=g) * torch.exp2(torch.randint(-12, 13, (rows, 1), device=dev(), generator=g).float())
    x = x * torch.exp(torch.randn(cols, device=dev(), generator=g))
    x[:, cols // 2:cols // 2 + 128] *= (torch.rand(rows, 1, device=dev(), generator=g) < 0.8).float()
    return x.to(dt)


def rows8(g, rows, cols):
    from flash_stu_2_b200 import ops
    return ops.quantize_fp8(stream(g, rows, cols, torch.float32))


def weights8(g, rows, cols):
    from flash_stu_2_b200 import ops
    return ops.quantize_fp8(torch.randn(rows, cols, device=dev(), generator=g) * torch.exp(torch.randn(rows, 1, device=dev(), generator=g)) * cols ** -0.5)


def same_rows(a, b):
    return a.cols == b.cols and torch.equal(a.data.view(torch.uint8), b.data.view(torch.uint8)) and torch.equal(
        a.scales.view(torch.uint8), b.scales.view(torch.uint8))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_is_exact(dt, rows, cols):
    from flash_stu_2_b200 import ops
    x = stream(gen(rows + cols), rows, cols, dt)
    q = ops.quantize_fp8(x)
    want, e = R.quantize(x.double())
    assert torch.equal(q.data.double(), want)
    assert torch.equal(q.scales.view(torch.uint8), R.pieces((e + 127).to(torch.uint8)))
    assert torch.equal(q.dequantize().double(), (R.blocks(want) * R.power(e)[:, :, None]).view(want.shape)[:, :cols])


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_quantize_borders(dt):
    """Maxima on, right below and right above 448 * 2^e; ties between neighbours; the smallest numbers; infinities and NaN beside others and alone;
    zeros of both signs; a maximum below the smallest scale's."""
    from flash_stu_2_b200 import ops
    lines = []
    for top in (448.0, 450.0, 446.0, 1.75, 1.7578125, 2.0 ** -120 * 1.75, 2.0 ** 100):
        line = torch.linspace(-1, 1, 128, dtype=torch.float64) * top
        line[0] = top
        lines.append(line)
    grid = torch.arange(128, dtype=torch.float64)
    lines.append(torch.cat([torch.tensor([448.0]), 16 + grid[:127] / 2]))          # ties among steps of 2
    lines.append(torch.cat([torch.tensor([448.0]), grid[:127] * 2.0 ** -11]))      # below the smallest normal number, ties among steps of 2^-9
    lines.append(torch.full((128,), 2.0 ** -126, dtype=torch.float64))
    lines.append(-torch.zeros(128, dtype=torch.float64))
    for special in (float("inf"), float("-inf"), float("nan")):
        line = torch.linspace(-3, 3, 128, dtype=torch.float64)
        line[[5, 77]] = special
        lines.append(line)
        lines.append(torch.full((128,), special, dtype=torch.float64))
    x = torch.stack(lines).to(dt).to(dev())
    q = ops.quantize_fp8(x)
    want, e = R.quantize(x.double())
    assert torch.equal(q.data.double().nan_to_num(7e7), want.nan_to_num(7e7))
    assert torch.equal(q.scales.view(torch.uint8), R.pieces((e + 127).to(torch.uint8)))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_quantize_takes_any_strides(dt):
    from flash_stu_2_b200 import ops
    g = gen(3)
    wide = stream(g, 40, 700, dt)
    for x in (wide[:, 8:608], wide[:, 3:603], wide[::3, :300], wide.t(), wide.view(4, 10, 700), wide.view(4, 10, 700)[:, ::2, 5:400], wide[7], wide[:1, :9]):
        flat = x.reshape(-1, x.shape[-1])
        assert same_rows(ops.quantize_fp8(x), ops.quantize_fp8(flat.contiguous()))
    assert ops.quantize_fp8(wide[:0]).shape == (0, 700) and ops.quantize_fp8(wide[:0]).dequantize().shape == (0, 700)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("rows,cols", SHAPES + [(1300, 1536), (2500, 1024), (7, 32768), (1184, 2500)])
def test_rmsnorm(dt, add, rows, cols):
    """The stored sum is exact; statistics and scaling in fp32: sums of up to 32768 squares as chains of at most 64, 2^-16 in all."""
    from flash_stu_2_b200 import ops
    g = gen(rows + cols)
    x, w = stream(g, rows, cols, dt), (1 + 0.3 * torch.randn(cols, device=dev(), generator=g)).to(dt)
    branch = stream(g, rows, cols, dt) if add else None
    before = x.clone()
    q = ops.rmsnorm_fp8(x, w, 1e-5, add=branch)
    s = before if not add else (before.float() + branch.float()).to(dt)
    assert torch.equal(x, s)
    v = s.double()
    v = v / torch.sqrt(v.square().mean(1, keepdim=True) + 1e-5) * w.double()
    R.check_rows(q, v, v.abs() * 2.0 ** -16)


def test_rmsnorm_where_the_sum_goes():
    """A separate output, the branch itself, strided rows of every operand; x alone stays as it is; rows of another count give the same rows."""
    from flash_stu_2_b200 import ops
    g = gen(5)
    x, b, w = stream(g, 33, 520, torch.bfloat16), stream(g, 33, 520, torch.bfloat16), torch.rand(520, device=dev(), generator=g).bfloat16()
    want, total = ops.rmsnorm_fp8(x.clone(), w, add=b), (x.float() + b.float()).bfloat16()
    keep, out = x.clone(), torch.full((33, 600), 9.0, device=dev(), dtype=torch.bfloat16)
    assert same_rows(ops.rmsnorm_fp8(x, w, add=b, out=out[:, 40:560]), want) and torch.equal(x, keep)
    assert torch.equal(out[:, 40:560], total) and bool((out[:, :40] == 9).all()) and bool((out[:, 560:] == 9).all())
    b2 = b.clone()
    assert same_rows(ops.rmsnorm_fp8(x, w, add=b2, out=b2), want) and torch.equal(b2, total)
    off = torch.empty(33, 523, device=dev(), dtype=torch.bfloat16)[:, 3:]   # off the 16-byte grid
    off.copy_(x)
    assert same_rows(ops.rmsnorm_fp8(off, w, add=b), want) and torch.equal(off, total)
    assert same_rows(ops.rmsnorm_fp8(x.view(3, 11, 520), w, add=b.view(3, 11, 520), out=torch.empty_like(x).view(3, 11, 520)), want)
    plain = ops.rmsnorm_fp8(x, w)
    assert torch.equal(x, keep)
    many = ops.rmsnorm_fp8(x.repeat(80, 1), w)
    assert torch.equal(many.data.view(torch.uint8)[-33:], plain.data.view(torch.uint8)) and torch.equal(many.block_scales()[-33:], plain.block_scales())
    assert ops.rmsnorm_fp8(x[:0], w, add=b[:0]).shape == (0, 520)


def test_rmsnorm_of_rows_without_a_size():
    """Zeros; a value whose square leaves fp32; infinities and NaN: the row's own, no other's."""
    from flash_stu_2_b200 import ops
    x = torch.randn(6, 300, device=dev(), generator=gen(1))
    x[1] = 0
    x[2, 7] = float("nan")
    x[3, 299] = float("inf")
    q = ops.rmsnorm_fp8(x, torch.ones(300, device=dev()), 1e-6)
    v = x.double()
    v = v / torch.sqrt(v.square().mean(1, keepdim=True) + 1e-6)
    R.check_rows(q, v, v.abs().nan_to_num(0) * 2.0 ** -16)


LINEAR = [(1, 1, 1), (1, 16, 128), (1, 1536, 18432), (2, 5, 100), (7, 129, 129), (8, 1024, 4096), (9, 200, 513), (16, 96, 1000), (17, 33, 640),
          (32, 1536, 1536), (33, 1111, 1000), (64, 128, 2048), (127, 257, 300), (130, 520, 1536), (256, 256, 128), (333, 1111, 1000), (700, 1000, 520),
          (1024, 2048, 1024), (1300, 300, 2000), (2049, 1536, 640), (4100, 260, 384)]


def check_linear(y, x, w, resid=None):
    ref, off = R.product(x, w)
    off = off + (ref.abs() + off) * BF16_HALF
    if resid is not None:
        ref = ref + resid.double()
        off = off + (ref.abs() + off) * BF16_HALF
    bad = ~((y.double() - ref).abs() <= off + 1e-38)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} values, first {bad.nonzero()[0].tolist()}: " \
                                f"{y[tuple(bad.nonzero()[0].tolist())]} for {ref[tuple(bad.nonzero()[0].tolist())]}"


@pytest.mark.parametrize("resid", [False, True])
@pytest.mark.parametrize("M,N,K", LINEAR)
def test_linear(M, N, K, resid):
    from flash_stu_2_b200 import ops
    g = gen(M + N + K)
    x, w = rows8(g, M, K), weights8(g, N, K)
    r = stream(g, M, N, torch.bfloat16) if resid else None
    y = ops.linear_fp8(x, w, resid=r)
    check_linear(y, x, w, r)
    assert torch.equal(ops.linear_fp8(x, w, resid=r), y)


GATE = [(1, 1, 1), (1, 128, 128), (1, 4096, 1024), (2, 5, 100), (8, 640, 129), (9, 200, 513), (16, 1000, 1000), (31, 6144, 1536), (33, 129, 640),
        (64, 1536, 768), (130, 520, 384), (256, 512, 128), (333, 1111, 1000), (1024, 1024, 1024), (1300, 300, 2000), (2049, 2048, 640)]


@pytest.mark.parametrize("M,N,K", GATE)
def test_gate(M, N, K):
    from flash_stu_2_b200 import ops
    g = gen(M + N + K)
    x, w, w2 = rows8(g, M, K), weights8(g, N, K), weights8(g, N, K)
    h = ops.linear_fp8(x, w, W2=w2)
    R.check_rows(h, *R.gate(x, w, w2))
    assert same_rows(ops.linear_fp8(x, w, W2=w2), h)


def test_linear_writes_where_it_is_told():
    """Outputs and residual rows in wider tensors, on and off the 16-byte grid, in place; what lies beside them stays."""
    from flash_stu_2_b200 import ops
    for M, N, K in [(5, 96, 256), (40, 200, 300), (300, 264, 256)]:
        for lead in (8, 3):
            g = gen(M + lead)
            x, w, r = rows8(g, M, K), weights8(g, N, K), stream(g, M, N, torch.bfloat16)
            want = ops.linear_fp8(x, w, resid=r)
            big = torch.full((M, N + 24), 5.0, device=dev(), dtype=torch.bfloat16)
            out = big[:, lead:lead + N]
            assert ops.linear_fp8(x, w, resid=r, out=out) is out
            assert torch.equal(out, want) and bool((big[:, :lead] == 5).all()) and bool((big[:, lead + N:] == 5).all())
            out.copy_(r)
            ops.linear_fp8(x, w, resid=out, out=out)
            assert torch.equal(out, want) and bool((big[:, :lead] == 5).all()) and bool((big[:, lead + N:] == 5).all())
            check_linear(ops.linear_fp8(x, w, out=out), x, w)
    x, w = rows8(gen(1), 4, 256), weights8(gen(2), 8, 256)
    none = ops.Fp8Rows(x.data[:0], x.scales[:0], 256)
    assert ops.linear_fp8(none, w).shape == (0, 8) and ops.linear_fp8(none, w, W2=w).shape == (0, 8)


@pytest.mark.parametrize("M", [3, 40, 400])
def test_nan_stays_in_its_row_and_column(M):
    from flash_stu_2_b200 import ops
    g = gen(M)
    a, b = torch.randn(M, 300, device=dev(), generator=g), torch.randn(140, 300, device=dev(), generator=g)
    a[M - 1, 299] = float("nan")
    b[7, 0] = float("inf")
    x, w = ops.quantize_fp8(a), ops.quantize_fp8(b)
    y = ops.linear_fp8(x, w)
    nan = torch.zeros(M, 140, dtype=torch.bool, device=dev())
    nan[M - 1] = True
    nan[:, 7] = True
    assert torch.equal(torch.isnan(y), nan)
    h = ops.linear_fp8(x, w, W2=w)
    assert torch.equal(torch.isnan(h.data[:, :140].float()), nan)
    fine = torch.isfinite(a).all(1)
    one = ops.linear_fp8(ops.quantize_fp8(a[fine]), w)
    check = ~nan[fine]
    assert torch.equal(one[check], y[fine][check])


@pytest.mark.parametrize("M", [2, 20, 200])
def test_scales_far_apart(M):
    """Operands whose scales differ by 2^100 from block to block: products of tiny and huge blocks are exact powers of two apart."""
    from flash_stu_2_b200 import ops
    g = gen(M)
    up = torch.exp2(torch.tensor([0, 50, -50, 20, -100], device=dev()).float()).repeat_interleave(128)
    a, b = torch.randn(M, 640, device=dev(), generator=g) * up, torch.randn(72, 640, device=dev(), generator=g) / up
    x, w = ops.quantize_fp8(a), ops.quantize_fp8(b)
    check_linear(ops.linear_fp8(x, w), x, w)


@pytest.mark.parametrize("M,d,inter", [(1, 1024, 4096), (32, 512, 1536), (300, 384, 1000)])
def test_an_mlp_of_them(M, d, inter):
    """Norm, gate and up, down onto the stream, one behind the other: within what 8 bits lose of the MLP in 64 bits, and each call against its own inputs.
    Two quantisations of normal values (2^-4 at most, 2^-5.3 in the mean square) and as much of the weights: every product is off by
    less than 2^-4 of its terms' root sum of squares; 4 of them compound to less than 1/8 of the branch's."""
    from flash_stu_2_b200 import ops
    g = gen(M + d)
    x = torch.randn(M, d, device=dev(), generator=g).bfloat16()
    branch, norm = torch.randn(M, d, device=dev(), generator=g).bfloat16(), (1 + 0.1 * torch.randn(d, device=dev(), generator=g)).bfloat16()
    gate, up, down = (torch.randn(*s, device=dev(), generator=g) * s[1] ** -0.5 for s in ((inter, d), (inter, d), (d, inter)))
    wg, wu, wd = (ops.quantize_fp8(t) for t in (gate, up, down))
    total = torch.empty_like(x)
    xn = ops.rmsnorm_fp8(x, norm, add=branch, out=total)
    h = ops.linear_fp8(xn, wg, W2=wu, overlap=True)
    y = ops.linear_fp8(h, wd, resid=total, overlap=True)
    R.check_rows(h, *R.gate(xn, wg, wu))
    check_linear(y, h, wd, total)
    s = (x.float() + branch.float()).bfloat16().double()
    v = s / torch.sqrt(s.square().mean(1, keepdim=True) + ops.RMS_EPS) * norm.double()
    mlp = (R.gelu(v @ gate.double().T) * (v @ up.double().T)) @ down.double().T
    assert float((y.double() - s - mlp).norm() / mlp.norm()) < 0.125


def test_another_stream_and_a_replayed_graph():
    from flash_stu_2_b200 import ops
    g = gen(8)
    M, d, inter = 5, 512, 1024
    xs = [torch.randn(M, d, device=dev(), generator=g).bfloat16() for _ in range(3)]
    norm = torch.ones(d, device=dev(), dtype=torch.bfloat16)
    wg, wu, wd = weights8(g, inter, d), weights8(g, inter, d), weights8(g, d, inter)

    def mlp(x):
        return ops.linear_fp8(ops.linear_fp8(ops.rmsnorm_fp8(x, norm), wg, W2=wu), wd, resid=x)

    want = [mlp(x) for x in xs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [mlp(x) for x in xs]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mlp(static)
    for x, w in zip(xs, want):
        static.copy_(x)
        graph.replay()
        assert torch.equal(out, w)
    # outputs from an arena, as a captured step takes them
    buffer = torch.zeros(1 << 20, dtype=torch.uint8, device=dev())
    with ops.arena(buffer):
        y = mlp(xs[1])
    assert torch.equal(y, want[1])
    assert buffer.data_ptr() <= y.data_ptr() < buffer.data_ptr() + buffer.numel()
    ops.check_status()


def test_refusals():
    from flash_stu_2_b200 import ops
    g = gen(4)
    x, w = rows8(g, 4, 256), weights8(g, 8, 256)
    b = torch.zeros(4, 8, device=dev(), dtype=torch.bfloat16)
    half = torch.zeros(4, 256, device=dev(), dtype=torch.float16)
    for call, error, text in [
            (lambda: ops.quantize_fp8(half), TypeError, "float32 or bfloat16"),
            (lambda: ops.quantize_fp8(b[:, :0]), ValueError, "no columns"),
            (lambda: ops.rmsnorm_fp8(b, torch.ones(8, device=dev())), TypeError, "one type"),
            (lambda: ops.rmsnorm_fp8(b, b[0, :7]), ValueError, "weight"),
            (lambda: ops.rmsnorm_fp8(b, b[0], add=b[:2]), ValueError, "x's shape"),
            (lambda: ops.rmsnorm_fp8(b, b[0], out=b), ValueError, "x \\+ add"),
            (lambda: ops.rmsnorm_fp8(b.t(), b[:, 0].contiguous(), add=b.t()), ValueError, "in place"),
            (lambda: ops.rmsnorm_fp8(torch.zeros(1, 32769, device=dev()), torch.zeros(32769, device=dev())), RuntimeError, "shape"),
            (lambda: ops.linear_fp8(x, weights8(g, 8, 300)), ValueError, "linear_fp8"),
            (lambda: ops.linear_fp8(x, w, W2=weights8(g, 9, 256)), ValueError, "W2"),
            (lambda: ops.linear_fp8(x, w, W2=w, resid=b), ValueError, "added"),
            (lambda: ops.linear_fp8(x, w, resid=b.float()), TypeError, "bfloat16"),
            (lambda: ops.linear_fp8(x, w, out=b[:, :7]), ValueError, "out"),
            (lambda: ops.linear_fp8(x, w, out=b.t().contiguous().t()), ValueError, "contiguous rows"),
            (lambda: ops.linear_fp8(ops.Fp8Rows(x.data[:, :128], x.scales, 128), w), ValueError, "contiguous rows"),
            (lambda: ops.linear_fp8(ops.Fp8Rows(x.data, x.scales[:0], 256), w), ValueError, "scales"),
            (lambda: ops.linear_fp8(ops.Fp8Rows(x.data.float(), x.scales, 256), w), TypeError, "float8_e4m3fn"),
            (lambda: ops.linear_fp8(x, ops.Fp8Rows(w.data[:0], w.scales[:0], 256)), ValueError, "no rows"),
            (lambda: ops.linear_fp8(x, ops.Fp8Rows(w.data.cpu(), w.scales, 256)), RuntimeError, "no CPU path")]:
        with pytest.raises(error, match=text):
            call()
    torch.cuda.synchronize()


@pytest.mark.parametrize("M", [100, 300])
@pytest.mark.parametrize("two", [False, True])
def test_a_wait_that_runs_out(M, two):
    """A CTA alone and a pair of them, plain and gate/up: a first stage that never fills is reported (status 3) within the shortened bound, and the next
    call is as ever."""
    import time
    from flash_stu_2_b200 import _lib, ops
    lib, g = _lib.load(), gen(M)
    x, w, w2 = rows8(g, M, 700), weights8(g, 400, 700), weights8(g, 400, 700)
    call = (lambda: ops.linear_fp8(x, w, W2=w2)) if two else (lambda: ops.linear_fp8(x, w))
    same = same_rows if two else torch.equal
    want = call()
    ops.check_status()
    assert lib.stu_test_inject_wait_expiry(100) == 0
    try:
        t0 = time.monotonic()
        call()
        torch.cuda.synchronize()
        assert time.monotonic() - t0 < 5.0
        with pytest.raises(RuntimeError, match="status 3"):
            ops.check_status()
    finally:
        assert lib.stu_test_inject_wait_expiry(0) == 0
    assert same(call(), want)
    ops.check_status()


# ---------------------------------------------------------------------------------------------------- the models that use them
def plain_mlp(mlp, x, resid, norm_w, eps):
    """resid + an 8-bit MLP of norm(x), from the definitions in 64 bits, rounded where the layer rounds."""
    def rows(v):
        q, e = R.quantize(v)
        return (R.blocks(q) * R.power(e)[:, :, None]).view(q.shape)[:, :v.shape[1]]
    v = x.double()
    v = rows((v / torch.sqrt(v.square().mean(1, keepdim=True) + eps) * norm_w.double()).float().double())
    gate, up, down = (rows(getattr(mlp, n).weight.double()) for n in ("gate_proj", "up_proj", "down_proj"))
    h = rows((R.gelu(v @ gate.T) * (v @ up.T)).float().double())
    return (resid.float() + (h @ down.T).bfloat16().float()).bfloat16()


def model(d=256, layers=4, seed=0, **kw):
    import flash_stu_2_b200 as F
    torch.manual_seed(seed)
    cfg = F.FlashSTUConfig(**{**dict(n_embd=d, n_layers=layers, n_heads=4, seq_len=256, window_size=64, vocab_size=501, mlp_scale=3, num_eigh=8,
                                     torch_dtype=torch.bfloat16, mlp_fp8=True), **kw})
    m = F.FlashSTU(cfg).to(dev()).eval()
    with torch.no_grad():
        for name, p in m.named_parameters():   # branches that are small against the stream, as a trained model's
            if p.dim() == 2:
                p.normal_(0, p.shape[1] ** -0.5 * (0.3 if "down_proj" in name or "c_proj" in name else 1), generator=gen(seed + p.numel()))
    return m


@pytest.mark.parametrize("T", [1, 40, 200])
@pytest.mark.parametrize("attention", [False, True])
def test_a_layer_with_an_8_bit_mlp(T, attention):
    """Prefill and cached steps of a layer against the same layer whose MLP is computed from the definitions; 2e-2 relative is what the layers are held to
    in bf16.  (Both have the same input to the MLP, so that the 8-bit values differ where fp32 sums put a value on the other side of a rounding.)"""
    import flash_stu_2_b200 as F
    from parity import close
    m = model(layers=2)
    layer = m.layers[1 if attention else 0]
    assert type(layer.mlp) is F.Fp8MLP
    x = torch.randn(3, T + 3, 256, device=dev(), generator=gen(T)).bfloat16()

    def run():
        with torch.no_grad():
            y, cache = layer(x[:, :T].clone(), past_key_value=None, use_cache=True)
            out = [y.clone()]
            for t in range(T, T + 3):
                y, cache = layer(x[:, t:t + 1].clone(), past_key_value=cache, use_cache=True)
                out.append(y.clone())
        return torch.cat(out, 1)

    got = run()

    def plain(xn2d, resid2d, out2d, norm_w=None, eps=0.0, overlap=False, add=None):
        if add is not None:
            xn2d += add   # (bf16 + bf16, rounded once)
        out2d.copy_(plain_mlp(layer.mlp, xn2d, resid2d, norm_w, eps))

    layer.mlp.apply_residual = plain
    close(got, run(), 2e-2)


@pytest.mark.parametrize("kw", [dict(), dict(use_approx=False), dict(use_attn=False), dict(stu_enable_mlp_sandwich=True, stu_mlp_hidden_size=128)])
@pytest.mark.parametrize("B", [1, 20])
def test_generate_with_8_bit_mlps(B, kw):
    """A captured step and the layers one by one are the same kernels: the same tokens and logits.  The logits are near the bf16 model's: three 8-bit roundings of
    2^-5.3 in the mean square per MLP (norm, weights, h; the weights' again), whose branches are 0.3 of a stream that grows with them."""
    m = model(**kw)
    ids = torch.randint(0, 501, (B, 30), device=dev(), generator=gen(B))
    with torch.no_grad():
        a, la = m.generate(ids, max_length=50, do_sample=False, return_logits=True)
        b, lb = m.generate(ids, max_length=50, do_sample=False, return_logits=True, cuda_graph=False)
        assert torch.equal(a, b) and torch.equal(la, lb)
        full = m(a, use_cache=False).logits[:, 29:-1].float()
        other = model(mlp_fp8=False, **kw)
        other.load_state_dict(m.state_dict())
        ref = other(a, use_cache=False).logits[:, 29:-1].float()
    # a step and a prefill differ where a bf16 rounding puts an 8-bit value elsewhere: within what the 8 bits lose
    assert float((full - ref).norm() / ref.norm()) < 0.1
    assert float((la.float() - full).norm() / full.norm()) < 0.1


def test_8_bit_weights_follow_the_parameters():
    from flash_stu_2_b200 import ops
    m = model(layers=1)
    mlp, x = m.layers[0].mlp, torch.randn(5, 256, device=dev(), generator=gen(1)).bfloat16()
    with torch.no_grad():
        first = mlp(x)
        assert mlp.rows()[0] is mlp.rows()[0] and torch.equal(mlp(x), first)
        mlp.down_proj.weight.mul_(2)
        assert torch.equal(mlp(x).float(), 2 * first.float())   # a power of two: every rounding is the same
        mlp.gate_proj.weight.data = mlp.gate_proj.weight.data.flip(0).contiguous()
        assert not torch.equal(mlp(x).float(), 2 * first.float())
        assert mlp(x.view(1, 5, 256)).shape == (1, 5, 256)
        want = mlp(x)
        mlp.up_proj.weight.mul_(1)   # new 8-bit rows, made while an arena is open, are not its pieces
        buffer = torch.zeros(1 << 20, dtype=torch.uint8, device=dev())
        with ops.arena(buffer):
            mlp(x)
        buffer.fill_(255)
        assert torch.equal(mlp(x), want)


def test_8_bit_weights_of_a_graph():
    """A first call that is captured makes rows of the graph's own; a graph that reads kept rows reads those of new weights too."""
    from flash_stu_2_b200 import ops
    m = model(layers=1)
    mlp, x = m.layers[0].mlp, torch.randn(5, 256, device=dev(), generator=gen(2)).bfloat16()
    ops.status_word(dev())
    with torch.no_grad():
        want = model(layers=1).layers[0].mlp(x)
        own = torch.cuda.CUDAGraph()
        with torch.cuda.graph(own):
            y = mlp(x)
        assert torch.equal(mlp(x), want)   # nothing has been replayed
        own.replay()
        assert torch.equal(y, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            z = mlp(x)
        graph.replay()
        assert torch.equal(z, want)
        mlp.down_proj.weight.mul_(2)
        assert torch.equal(mlp(x).float(), 2 * want.float())
        for g, out in ((graph, z), (own, y)):
            g.replay()
            assert torch.equal(out.float(), 2 * want.float())
        w = mlp.up_proj.weight
        twice = w.cpu() * 2
        w.data = torch.empty(0, device=dev(), dtype=torch.bfloat16)
        w.data = twice.to(dev())
        assert torch.equal(mlp(x).float(), 4 * want.float())
    ops.check_status()


@pytest.mark.parametrize("M,d,inter", [(1, 512, 1024), (40, 1536, 2048), (700, 1024, 1100)])
def test_two_streams_at_once(M, d, inter):
    """The chain of an MLP on two streams at a time, from threads of their own, many times over: what each gives alone."""
    import threading
    from flash_stu_2_b200 import ops
    g = gen(M)
    wg, wu, wd = weights8(g, inter, d), weights8(g, inter, d), weights8(g, d, inter)
    norm = torch.ones(d, device=dev(), dtype=torch.bfloat16)
    xs = [torch.randn(M, d, device=dev(), generator=g).bfloat16() for _ in range(2)]

    def mlp(x):
        return ops.linear_fp8(ops.linear_fp8(ops.rmsnorm_fp8(x, norm), wg, W2=wu, overlap=True), wd, resid=x, overlap=True)

    want = [mlp(x) for x in xs]
    torch.cuda.synchronize()
    wrong = []

    def run(x, w):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got = [mlp(x) for _ in range(50)]
        stream.synchronize()
        wrong.extend(i for i, y in enumerate(got) if not torch.equal(y, w))

    threads = [threading.Thread(target=run, args=p) for p in zip(xs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    ops.check_status()


@pytest.mark.parametrize("cols", [300, 1536, 4096])
def test_equal_rows_give_equal_rows(cols):
    """Within a call wherever they stand; of the norm and the quantisation whatever stands beside them."""
    from flash_stu_2_b200 import ops
    g = gen(cols)
    one = stream(g, 1, cols, torch.bfloat16)
    w = torch.randn(cols, device=dev(), generator=g).bfloat16()
    a, b = weights8(g, 200, cols), weights8(g, 200, cols)
    norms, quantised = [], []
    for rows in (1, 3, 130, 700, 6000):
        x = one.expand(rows, cols).contiguous()
        q, n = ops.quantize_fp8(x), ops.rmsnorm_fp8(x, w)
        for r in (q, n, ops.linear_fp8(n, a, W2=b)):
            assert bool((r.data.view(torch.uint8) == r.data.view(torch.uint8)[:1]).all()) and bool((r.block_scales() == r.block_scales()[:1]).all())
        y = ops.linear_fp8(n, a)
        assert bool((y == y[:1]).all())
        quantised.append((q.data.view(torch.uint8)[:1], q.block_scales()[:1]))
        norms.append((n.data.view(torch.uint8)[:1], n.block_scales()[:1]))
    for found in (norms, quantised):
        assert all(torch.equal(d, found[0][0]) and torch.equal(s, found[0][1]) for d, s in found)


# up to 64 tokens, and more whose K is long enough to be cut: the forms that have the weights as the 128-row operand, at the edges of their tiles and clusters
CUT = [(17, 300, 2000), (48, 1111, 1536), (64, 257, 4000), (65, 300, 2100), (96, 1, 2177), (128, 128, 2304), (129, 520, 2560), (200, 257, 4096), (300, 520, 2305),
       (384, 1000, 2400), (500, 1100, 9000), (64, 20000, 200)]


@pytest.mark.parametrize("resid", [False, True])
@pytest.mark.parametrize("M,N,K", CUT)
def test_linear_whose_K_is_cut(M, N, K, resid):
    from flash_stu_2_b200 import ops
    g = gen(M + N + K)
    x, w = rows8(g, M, K), weights8(g, N, K)
    big = torch.full((M + 2, N + 9), 5.0, device=dev(), dtype=torch.bfloat16)
    out = big[1:M + 1, 4:4 + N]
    r = stream(g, M, N, torch.bfloat16) if resid else None
    ops.linear_fp8(x, w, resid=r, out=out)
    check_linear(out, x, w, r)
    assert torch.equal(ops.linear_fp8(x, w, resid=r, overlap=True), out)
    big[1:M + 1, 4:4 + N] = 5.0
    assert bool((big == 5).all())
    ops.check_status()


@pytest.mark.parametrize("M,N,K", [(16, 300, 700), (17, 700, 1111), (32, 2000, 300), (32, 18400, 256), (33, 300, 700), (128, 18400, 200)])
def test_gate_of_few_tokens(M, N, K):
    from flash_stu_2_b200 import ops
    g = gen(M + N + K)
    x, w, w2 = rows8(g, M, K), weights8(g, N, K), weights8(g, N, K)
    h = ops.linear_fp8(x, w, W2=w2)
    R.check_rows(h, *R.gate(x, w, w2))
    assert same_rows(ops.linear_fp8(x, w, W2=w2, overlap=True), h)
    ops.check_status()


@pytest.mark.parametrize("M,K,two", [(5, 700, False), (5, 700, True), (30, 2100, False), (30, 2100, True), (50, 2100, False), (100, 2100, False)])
def test_a_wait_that_runs_out_where_K_is_cut(M, K, two):
    from flash_stu_2_b200 import _lib, ops
    lib, g = _lib.load(), gen(M)
    x, w, w2 = rows8(g, M, K), weights8(g, 400, K), weights8(g, 400, K)
    call = (lambda: ops.linear_fp8(x, w, W2=w2)) if two else (lambda: ops.linear_fp8(x, w))
    same = same_rows if two else torch.equal
    want = call()
    ops.check_status()
    assert lib.stu_test_inject_wait_expiry(100) == 0
    try:
        call()
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="status 3"):
            ops.check_status()
    finally:
        assert lib.stu_test_inject_wait_expiry(0) == 0
    assert same(call(), want)
    ops.check_status()


@pytest.mark.parametrize("M", [3, 200])
def test_the_librarys_calls(M):
    """The three calls by addresses, as a host of another kind makes them."""
    from flash_stu_2_b200 import _lib, ops
    lib, g, d, inter, eps = _lib.load(), gen(M), 520, 1100, 1e-5
    stream = torch.cuda.current_stream().cuda_stream
    gate, up, down = (torch.randn(*s, device=dev(), generator=g) * s[1] ** -0.5 for s in ((inter, d), (inter, d), (d, inter)))
    x, branch = (torch.randn(M, d, device=dev(), generator=g).bfloat16() for _ in range(2))
    norm = torch.ones(d, device=dev(), dtype=torch.bfloat16)

    def rows8(n, cols):
        return (torch.empty(n, -(-cols // 128) * 128, dtype=torch.float8_e4m3fn, device=dev()),
                torch.empty(-(-n // 128), -(-cols // 512), 32, 4, 4, dtype=torch.float8_e8m0fnu, device=dev()))

    p = lambda r: (r[0].data_ptr(), r[1].data_ptr())
    weights = []
    for w in (gate, up, down):
        weights.append(rows8(*w.shape))
        assert lib.stu_quantize_fp8(w.data_ptr(), *p(weights[-1]), w.shape[0], w.shape[1], w.stride(0), 0, stream) == 0
    q = [ops.quantize_fp8(w) for w in (gate, up, down)]
    assert all(same_rows(ops.Fp8Rows(*a, b.cols), b) for a, b in zip(weights, q))
    want = x.clone()
    ops.linear_fp8(ops.linear_fp8(ops.rmsnorm_fp8(want, norm, eps, add=branch), q[0], W2=q[1]), q[2], resid=want, out=want)
    xn, h = rows8(M, d), rows8(M, inter)
    assert lib.stu_rmsnorm_fp8(x.data_ptr(), branch.data_ptr(), norm.data_ptr(), x.data_ptr(), *p(xn), M, d, d, d, d, eps, 1, stream) == 0
    assert lib.stu_linear_fp8(*p(xn), *p(weights[0]), *p(weights[1]), None, 0, h[0].data_ptr(), 0, h[1].data_ptr(), M, inter, d, 0, stream) == 0
    assert lib.stu_linear_fp8(*p(h), *p(weights[2]), None, None, x.data_ptr(), d, x.data_ptr(), d, None, M, d, inter, 0, stream) == 0
    assert torch.equal(x, want)
    ops.check_status()


def test_two_devices_at_once_are_refused():
    """Operands on several devices have no kernel; one of them alone is launched where it lies, whichever device is current."""
    from flash_stu_2_b200 import ops
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two CUDA devices")
    g = gen(0)
    x, w = rows8(g, 4, 256), weights8(g, 8, 256)
    want = ops.linear_fp8(x, w)
    there = ops.Fp8Rows(w.data.to("cuda:1"), w.scales.to("cuda:1"), 256)
    with pytest.raises(RuntimeError, match="several devices"):
        ops.linear_fp8(x, there)
    with torch.cuda.device(1):
        assert torch.equal(ops.linear_fp8(x, w), want)
