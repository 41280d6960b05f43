"""8-bit norms and products of many rows: CTAs that take tile after tile and warps that take row after row, every tile and row another; and the activation where its
gates are strongly negative.  Against the definitions in 64 bits."""
import math

import pytest
import torch

import fp8_reference as R
from test_gpu_5_fp8 import check_linear, dev, gen, model, rows8, same_rows, stream, weights8

pytestmark = pytest.mark.gpu


def gelu(g):
    """-> (gelu_tanh in 64 bits, t of exp(-t) in it), as the quotient: the form with tanh cancels where gates are negative (good to 2^-20 at -6 alone, 0 from -7.5 on)."""
    t = 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
    return g / (1 + torch.exp(-t)), t


def gate(x, w, w2, exact=False):
    """-> (gelu_tanh(x w^T) * (x w2^T), what it may be off).  `exact`: sums of one product each, which are exact.
    The activation in fp32, relative: t from two rounded constants and four rounded operations, 6 * 2^-24 of t, which is 3 |t| 2^-23 of exp(-t); the hardware's
    exponential 2 + 1.173 |t| steps of 2^-23 (its documented bound), the sum half a step, the quotient 2 steps, the product with the up value half a step: below
    (5 + 4.2 |t|) 2^-23.  The quotient is 0 where the denominator passes 2^126 (its documented range): |g| 2^-126 at most, twice that with the rounding of t."""
    (g, dg), (u, du) = R.product(x, w), R.product(x, w2)
    if exact:
        dg, du = torch.zeros_like(dg), torch.zeros_like(du)
    a, t = gelu(g)
    h = a * u
    return h, 1.13 * dg * (u.abs() + du) + a.abs() * du + h.abs() * ((5 + 4.2 * t.abs()) * 2.0 ** -23) + g.abs() * u.abs() * 2.0 ** -125


# 74 pairs of CTAs (148 alone) at a time: three to four tiles each, the last ones of odd sizes; K of one k-block, and ends inside of a piece of scales
@pytest.mark.parametrize("resid", [False, True])
@pytest.mark.parametrize("M,N,K", [(4100, 3900, 264), (4100, 3896, 100), (3000, 5000, 700),           # pairs on 256 x 256
                                   (28669, 381, 130), (28669, 376, 128), (56827, 100, 1030)])         # pairs on 256 x 128
def test_linear_of_many_tiles(M, N, K, resid):
    from flash_stu_2_b200 import ops
    g = gen(M + N + K)
    x, w = rows8(g, M, K), weights8(g, N, K)
    r = stream(g, M, N, torch.bfloat16) if resid else None
    y = ops.linear_fp8(x, w, resid=r)
    check_linear(y, x, w, r)
    big = torch.full((M + 2, N + 5), 5.0, device=dev(), dtype=torch.bfloat16)   # off the 16-byte grid, in place
    out = big[1:M + 1, 2:2 + N]
    if resid:
        out.copy_(r)
    ops.linear_fp8(x, w, resid=out if resid else None, out=out)
    assert torch.equal(out, y)
    big[1:M + 1, 2:2 + N] = 5.0
    assert bool((big == 5).all())
    ops.check_status()


@pytest.mark.parametrize("M,N,K", [(2100, 4000, 700), (2100, 3900, 128), (4099, 2049, 264),           # pairs
                                   (379, 18937, 136), (379, 18937, 100)])                             # CTAs alone: three rounds of them, four of pairs
def test_gate_of_many_tiles(M, N, K):
    from flash_stu_2_b200 import ops
    g = gen(M + N + K)
    x, w, w2 = rows8(g, M, K), weights8(g, N, K), weights8(g, N, K)
    h = ops.linear_fp8(x, w, W2=w2)
    R.check_rows(h, *gate(x, w, w2))
    assert same_rows(ops.linear_fp8(x, w, W2=w2), h)
    ops.check_status()


# K of few blocks cut over a cluster, and products on either side of the choice between the kernels
@pytest.mark.parametrize("resid", [False, True])
@pytest.mark.parametrize("M,N,K", [(1, 520, 700), (16, 1000, 1024), (32, 1536, 1536), (48, 768, 1152), (65, 1000, 1024), (200, 520, 700), (129, 1240, 1536), (96, 2048, 2048), (160, 2048, 2048),
                                   (1024, 520, 700), (1024, 1111, 1000), (512, 1536, 3000), (130, 1001, 2560), (700, 1024, 4096)])
def test_linear_near_the_choice(M, N, K, resid):
    from flash_stu_2_b200 import ops
    g = gen(M + N + K)
    x, w = rows8(g, M, K), weights8(g, N, K)
    r = stream(g, M, N, torch.bfloat16) if resid else None
    y = ops.linear_fp8(x, w, resid=r)
    check_linear(y, x, w, r)
    assert torch.equal(ops.linear_fp8(x, w, resid=r, overlap=True), y)
    ops.check_status()


@pytest.mark.parametrize("M,N,K", [(17, 18400, 256), (24, 12300, 300), (24, 18432, 1536), (25, 18400, 256), (20, 1000, 1000), (32, 768, 700)])
def test_gate_near_the_choice(M, N, K):
    from flash_stu_2_b200 import ops
    g = gen(M + N + K)
    x, w, w2 = rows8(g, M, K), weights8(g, N, K), weights8(g, N, K)
    h = ops.linear_fp8(x, w, W2=w2)
    R.check_rows(h, *gate(x, w, w2))
    assert same_rows(ops.linear_fp8(x, w, W2=w2, overlap=True), h)
    ops.check_status()


# bf16 rows without a branch, on the 32-byte grid and on the 16-byte one, of one to four pieces, up to three laps
@pytest.mark.parametrize("rows,cols", [(3600, 512), (9001, 512), (4001, 1024), (4001, 1000), (3555, 328), (2400, 1536), (2501, 1288), (2500, 2048), (5003, 2040), (4999, 1)])
def test_norm_of_many_rows(rows, cols):
    from flash_stu_2_b200 import ops
    g = gen(rows + cols)
    x, w = stream(g, rows, cols, torch.bfloat16), (1 + 0.3 * torch.randn(cols, device=dev(), generator=g)).bfloat16()
    keep = x.clone()
    q = ops.rmsnorm_fp8(x, w, 1e-5)
    assert torch.equal(x, keep)
    v = x.double()
    v = v / torch.sqrt(v.square().mean(1, keepdim=True) + 1e-5) * w.double()
    R.check_rows(q, v, v.abs() * 2.0 ** -16)
    for a in (0, rows // 2, rows - 7):   # a row's result does not depend on how many there are
        few = ops.rmsnorm_fp8(x[a:a + 7], w, 1e-5)
        assert torch.equal(few.data.view(torch.uint8), q.data.view(torch.uint8)[a:a + 7]) and torch.equal(few.block_scales(), q.block_scales()[a:a + 7])
    wide = torch.zeros(rows, cols + 24, device=dev(), dtype=torch.bfloat16)   # rows of a wider tensor
    wide[:, 8:8 + cols].copy_(x)
    assert same_rows(ops.rmsnorm_fp8(wide[:, 8:8 + cols], w, 1e-5), q)


@pytest.mark.parametrize("M", [8, 30, 200, 700])
def test_gates_that_are_strongly_negative(M):
    """Blocks whose gates all lie between -7.3 and -3 or between -9.3 and -4.5, where the activation falls by many powers of two and sets the scale; gates of every size up to where it
    is 0 or the gate itself; every sum is one product, so that the activation alone is seen."""
    from flash_stu_2_b200 import ops
    g = gen(M)
    N = 384
    mant = lambda *s: (8 + torch.randint(0, 8, s, device=dev(), generator=g)).float() / 8
    x, w, w2 = torch.zeros(M, 128, device=dev()), torch.zeros(N, 128, device=dev()), torch.zeros(N, 128, device=dev())
    x[:, 0] = mant(M)                         # 1 .. 1.875
    x[:, 1] = 1
    w[:128, 0] = -2 - mant(128)               # gates -3 .. -7.3
    w[128:256, 0] = -4 - 0.5 * mant(128)      # -4.5 .. -9.3
    w[256:, 0] = mant(128) * torch.exp2(torch.randint(-4, 5, (128,), device=dev(), generator=g).float()) * (torch.randint(0, 2, (128,), device=dev(), generator=g) * 2 - 1)
    w2[:, 1] = mant(N) * torch.exp2(torch.randint(-3, 4, (N,), device=dev(), generator=g).float())
    xq, wq, w2q = ops.quantize_fp8(x), ops.quantize_fp8(w), ops.quantize_fp8(w2)
    assert bool((xq.dequantize()[:, 1] == 1).all())
    R.check_rows(ops.linear_fp8(xq, wq, W2=w2q), *gate(xq, wq, w2q, exact=True))


@pytest.mark.parametrize("B", [1, 3])
def test_generate_behind_a_change_of_the_weights(B):
    """What a model generates with new weights is what one that never had the old ones does; in inference mode, and with weights that tell nobody of their changes, too."""
    ids = torch.randint(0, 501, (B, 20), device=dev(), generator=gen(B))
    run = lambda m: m.generate(ids, max_length=32, do_sample=False, return_logits=True)
    with torch.no_grad():
        m, other = model(layers=2, use_attn=True), model(layers=2, use_attn=True, seed=3)
        want = [run(m), run(other)]
        assert not torch.equal(want[0][1], want[1][1])
        m.load_state_dict(other.state_dict())
        got = run(m)
        assert torch.equal(got[0], want[1][0]) and torch.equal(got[1], want[1][1])
        with torch.inference_mode():
            for layer in m.layers:
                layer.mlp.load_state_dict({k: v.clone() for k, v in layer.mlp.state_dict().items()}, assign=True)
        for factor in (1, 2):
            with torch.inference_mode():
                m.layers[0].mlp.down_proj.weight.mul_(factor)
            with torch.no_grad():
                other.layers[0].mlp.down_proj.weight.mul_(factor)
            a, b = run(m), run(other)
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_memory_behind_a_move():
    """A model whose MLPs are in 8 bits leaves nothing on the device that it is moved from, and runs as before when it is back."""
    import gc
    ids = torch.randint(0, 501, (2, 20), device=dev(), generator=gen(0))
    with torch.no_grad():
        m = model(layers=2, d=512)
        want = m(ids, use_cache=False).logits.clone()
        gc.collect()
        held = torch.cuda.memory_allocated()
        mlps = sum(p.numel() for layer in m.layers for p in layer.mlp.parameters())
        for layer in m.layers:
            layer.mlp.to("cpu")
        assert held - torch.cuda.memory_allocated() >= 3 * mlps
        for layer in m.layers:
            layer.mlp.to(dev())
        assert torch.equal(m(ids, use_cache=False).logits, want)


def test_offsets_that_pass_32_bits():
    """Rows whose bytes lie behind the first 2^31 and 2^32: what the same rows give alone (K of one block: sums do not depend on the form)."""
    from flash_stu_2_b200 import ops
    g = gen(0)
    M, N, last = 550001, 4096, 301
    norm_w = torch.ones(N, device=dev(), dtype=torch.bfloat16)
    x, w, w2 = rows8(g, M, 128), weights8(g, N, 128), weights8(g, N, 128)
    few = ops.quantize_fp8(x.dequantize()[-last:])
    y = ops.linear_fp8(x, w)
    assert torch.equal(y[-last:], ops.linear_fp8(few, w))
    q, n = ops.quantize_fp8(y), ops.rmsnorm_fp8(y, norm_w)
    for rows, alone in ((q, ops.quantize_fp8(y[-last:])), (n, ops.rmsnorm_fp8(y[-last:], norm_w)), (ops.linear_fp8(x, w, W2=w2), ops.linear_fp8(few, w, W2=w2))):
        assert torch.equal(rows.data[-last:].view(torch.uint8), alone.data.view(torch.uint8)) and torch.equal(rows.block_scales()[-last:], alone.block_scales())
    half = y[-last:].clone()
    ops.rmsnorm_fp8(y, norm_w, add=y, out=y)
    assert torch.equal(y[-last:], (2 * half.float()).bfloat16())
    ops.check_status()
