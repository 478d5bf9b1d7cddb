"""Rows times 4-bit weights (``tv_w4_linear``) against the product in 64 bits.

Tolerance per output: a weight (u - 8) * s is rounded once to its 16-bit type
(half a step: 2^-8 of it in bf16, 2^-11 in fp16, and 2^-25 in fp16's subnormal
range), the products are summed in fp32 (at most K / 16 tensor-core steps and
8 CTAs in sequence: below K * 2^-24 of the sum of magnitudes), and the output
is rounded once more."""

from __future__ import annotations

import pytest
import torch

from conftest import cuda_ok

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a CUDA device")]

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SUB = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def weight64(q, s):
    """[N, K] in 64 bits, from the layout's definition."""
    n, words = q.shape
    w = torch.empty(n, words, 8, dtype=torch.float64, device=q.device)
    for i, k in enumerate((0, 2, 4, 6, 1, 3, 5, 7)):
        w[:, :, k] = ((q.long() >> (4 * i)) & 15).double() - 8
    return w.view(n, s.shape[1], -1).mul(s.double()[:, :, None]).view(n, words * 8)


def problem(t, n, k, group, dtype, seed=0, scale=0.02 / 4.6):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(-2 ** 31, 2 ** 31, (n, k // 8), dtype=torch.int32, device="cuda", generator=g)
    s = (scale * (0.5 + torch.rand(n, k // group, device="cuda", generator=g))).to(dtype)
    x = torch.randn(t, k, device="cuda", generator=g).to(dtype)
    return x, q, s


def to_fp8(x):
    s = x.float().abs().amax(-1) / 448
    return (x.float() / s[..., None]).to(torch.float8_e4m3fn), s


def check(y, x, q, s, xs=None):
    w, xd, t = weight64(q, s), x.double(), s.dtype
    if xs is not None:
        xd = xd * xs.double()[:, None]
    want = xd @ w.t()
    mass = xd.abs() @ w.abs().t()
    tol = mass * (HALF[t] + q.shape[1] * 8 * 2.0 ** -24) + xd.abs().sum(1)[:, None] * SUB[t]
    tol = tol + (want.abs() + tol) * HALF[t] + SUB[t]
    off = (y.double() - want).abs()
    assert bool((off <= tol).all()), float((off - tol).max())
    # and far inside it on the whole: errors of either sign average out
    if y.numel() > 256:
        assert float((y.double() - want).norm() / want.norm()) < 2 * HALF[t]


SHAPES = [(1, 64, 256, 128), (1, 6144, 4096, 128), (8, 1000, 704, 32), (17, 129, 1024, 64), (65, 4096, 4096, 128),
          (33, 4099, 14336, 32), (128, 2048, 896, 128), (129, 300, 512, 64), (300, 257, 96, 96), (3, 1, 32, 32),
          (2, 7, 64, 64), (5, 127, 14336, 128), (16, 512, 160, 32), (80, 513, 2080, 32),
          # many tiles: equal runs that cross tiles, rings that wrap; and two token blocks of them
          (48, 40960, 4096, 128), (16, 28672, 4096, 64), (128, 25700, 1056, 32), (200, 13000, 768, 128),
          (1, 40000, 256, 256)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,n,k,group", SHAPES)
def test_matches_the_product(t, n, k, group, dtype):
    from specverify.runtime import w4_linear
    x, q, s = problem(t, n, k, group, dtype, seed=t + n + k)
    y = w4_linear(x, q, s)
    check(y, x, q, s)
    assert torch.equal(y, w4_linear(x, q, s))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,n,k,group", SHAPES[:10])
def test_8_bit_rows(t, n, k, group, dtype):
    from specverify.runtime import w4_linear
    x, q, s = problem(t, n, k, group, dtype, seed=t + n + k + 1)
    x8, xs = to_fp8(x)
    check(w4_linear(x8, q, s, x_scale=xs), x8, q, s, xs)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_nibble_at_every_place(dtype):
    """One-hot rows read single weights back: all sixteen values, every k, exactly (u - 8 and a power of two)."""
    from specverify.runtime import dequantize_w4, w4_linear
    k, n = 256, 144
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randint(-2 ** 31, 2 ** 31, (n, k // 8), dtype=torch.int32, device="cuda", generator=g)
    s = torch.full((n, k // 32), 0.25, device="cuda").to(dtype)
    s *= 2.0 ** torch.randint(-3, 4, s.shape, device="cuda", generator=g)
    y = w4_linear(torch.eye(k, device="cuda").to(dtype), q, s)
    assert torch.equal(y.double().t(), weight64(q, s))
    assert torch.equal(dequantize_w4(q, s).double(), weight64(q, s))
    assert len(torch.unique((weight64(q, s).view(n, -1, 32) / s.double()[:, :, None]))) == 16


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale", [1e-4, 1.0, 50.0])
def test_small_and_large_scales(dtype, scale):
    from specverify.runtime import w4_linear
    x, q, s = problem(9, 200, 512, 64, dtype, seed=3, scale=scale)
    s[5] = 0
    s[7, 2] = -s[7, 2]
    y = w4_linear(x, q, s)
    check(y, x, q, s)
    assert bool((y[:, 5] == 0).all())


def test_quantize_round_trip():
    from specverify import SpecVerifyError
    from specverify.runtime import dequantize_w4, quantize_w4, w4_linear
    for dtype in (torch.bfloat16, torch.float16):
        w = (0.02 * torch.randn(300, 512, device="cuda")).to(dtype)
        w[3, :128] = 0
        q, s = quantize_w4(w, 128)
        assert torch.equal(q.cpu(), quantize_w4(w.cpu(), 128)[0])
        back = weight64(q, s)
        # half a step of the group's scale, the scale rounded to 16 bits (which moves 7 s by 7 half steps of it)
        step = s.double().repeat_interleave(128, 1)
        assert bool(((back - w.double()).abs() <= step * (0.5 + 8 * HALF[dtype])).all())
        assert bool((dequantize_w4(q, s)[3, :128] == 0).all())
        x = torch.randn(4, 7, 512, device="cuda").to(dtype)
        y = w4_linear(x, q, s)
        assert y.shape == (4, 7, 300)
        check(y.view(28, 300), x.view(28, 512), q, s)
    with pytest.raises(SpecVerifyError):
        quantize_w4(w, 48)
    with pytest.raises(SpecVerifyError):
        quantize_w4(w.float(), 128)


def test_strides_and_rows_left_alone():
    from specverify.runtime import w4_linear
    x, q, s = problem(40, 333, 1024, 128, torch.bfloat16)
    want = w4_linear(x, q, s)
    wide = torch.randn(40, 1024 + 9, device="cuda").bfloat16()
    for lead in (0, 1, 8):                      # rows at odd addresses, and with an odd stride
        wide[:, lead:lead + 1024] = x
        assert torch.equal(w4_linear(wide[:, lead:lead + 1024], q, s), want)
    even = torch.randn(80, 1032, device="cuda").bfloat16()
    even[::2, 8:] = x
    assert torch.equal(w4_linear(even[::2, 8:], q, s), want)
    row = x[:1].expand(40, 1024)
    assert torch.equal(w4_linear(row, q, s), w4_linear(x[:1].repeat(40, 1), q, s))
    buf = torch.full((80, 340), 5.0, device="cuda").bfloat16()
    got = w4_linear(x, q, s, out=buf[::2, 3:336])
    assert torch.equal(got, want) and bool((buf[1::2] == 5).all())
    assert bool((buf[:, :3] == 5).all()) and bool((buf[:, 336:] == 5).all())
    # weights and scales as row slices of larger ones
    q2, s2 = torch.zeros(666, 160, dtype=torch.int32, device="cuda"), torch.zeros(666, 11, device="cuda").bfloat16()
    q2[::2, :128], s2[::2, 2:10] = q, s
    assert torch.equal(w4_linear(x, q2[::2, :128], s2[::2, 2:10]), want)
    x8, xs = to_fp8(x)
    w8 = torch.zeros(40, 1027, device="cuda").to(torch.float8_e4m3fn)
    w8[:, 3:] = x8
    assert torch.equal(w4_linear(w8[:, 3:], q, s, x_scale=xs), w4_linear(x8, q, s, x_scale=xs))


def test_infinities_and_nan_stay_in_their_rows():
    from specverify.runtime import w4_linear
    x, q, s = problem(20, 150, 512, 128, torch.bfloat16)
    want = w4_linear(x, q, s)
    x[3, 100] = float("nan")
    x[11, 7] = float("inf")
    y = w4_linear(x, q, s)
    keep = [i for i in range(20) if i not in (3, 11)]
    assert torch.equal(y[keep], want[keep]) and bool(y[3].isnan().all()) and not bool(y[11].isfinite().any())


def test_side_stream_graph_and_empty():
    from specverify.runtime import w4_linear
    x, q, s = problem(65, 640, 2048, 128, torch.bfloat16)
    assert w4_linear(x[:0], q, s).shape == (0, 640)
    x8, xs = to_fp8(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = w4_linear(x, q, s)
    side.synchronize()
    check(y, x, q, s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a = w4_linear(x, q, s)
        b = w4_linear(x8, q, s, x_scale=xs)
    for seed in (5, 6):
        nx = problem(65, 640, 2048, 128, torch.bfloat16, seed)[0]
        x.copy_(nx)
        n8, ns = to_fp8(nx)
        x8.view(torch.uint8).copy_(n8.view(torch.uint8))
        xs.copy_(ns)
        g.replay()
        torch.cuda.synchronize()
        check(a, x, q, s)
        check(b, x8, q, s, xs)


def test_norm_product_chain():
    """The residual's addition and norm in 8 bits, straight into the product: the run of a decoder layer."""
    from specverify.runtime import add_rms_norm, w4_linear
    x, q, s = problem(65, 1024, 4096, 128, torch.bfloat16)
    r = 4 * torch.randn_like(x)
    w = torch.ones(4096, device="cuda").bfloat16()
    y8, scale, h = add_rms_norm(x, r, w, 1e-5, fp8=True)
    check(w4_linear(y8, q, s, x_scale=scale), y8, q, s, scale)
    y, h2 = add_rms_norm(x, r, w, 1e-5)
    assert torch.equal(h, h2)
    a, b = w4_linear(y8, q, s, x_scale=scale).double(), w4_linear(y, q, s).double()
    # e4m3 holds each value to within 2^-4: at most that between the two on the whole
    assert float((a - b).norm() / b.norm()) < 2.0 ** -4


def test_refusals():
    from specverify import SpecVerifyError
    from specverify.runtime import w4_linear
    x, q, s = problem(4, 96, 256, 64, torch.bfloat16)
    x8, xs = to_fp8(x)
    bad = [(x[:, :128], q, s, {}), (x, q[:, :16], s, {}), (x, q, s[:, :3], {}), (x, q[:50], s, {}), (x.half(), q, s, {}),
           (x.float(), q, s.float(), {}), (x, q.long(), s, {}), (x, q, s, dict(x_scale=xs)), (x8, q, s, {}),
           (x8, q, s, dict(x_scale=xs[:2])), (x8, q, s, dict(x_scale=xs.double())),
           (x.t().contiguous().t(), q, s, {}), (x, q.t().contiguous().t(), s, {}), (x.cpu(), q, s, {}),
           (x, q, s, dict(out=torch.empty(4, 95, device="cuda").bfloat16())),
           (x, q, s, dict(out=torch.empty(4, 96, device="cuda"))),
           (x, q, s, dict(out=torch.empty(1, 96, device="cuda").bfloat16().expand(4, 96))),
           (x, torch.zeros(96, 33, dtype=torch.int32, device="cuda")[:, 1:], s, {})]
    for a, b, c, kw in bad:
        with pytest.raises(SpecVerifyError):
            w4_linear(a, b, c, **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,k,group", [(40, 128, 128), (333, 384, 32), (100, 768, 256), (2500, 2048, 128), (48, 4224, 64)])
def test_every_number_of_rows_multiplies_the_same_weights(n, k, group, dtype):
    """A token decoded alone, in a frontier and in a tree sees one model: the weights are those of dequantize_w4, rounded
    once to the 16-bit type, in both kernels.  A row of x with 1 at one k and -1 at another reads the difference of two
    of them; both have at most 11 bits and lie within 2^9 of each other (or are 0), so that it fits fp32's 24 bits and
    is rounded once, to the output."""
    from specverify.runtime import dequantize_w4, w4_linear
    _, q, s = problem(1, n, k, group, dtype, seed=n + k)
    w = dequantize_w4(q, s).double()
    for t in (1, 3, 8, 9, 65, 130):
        g = torch.Generator().manual_seed(t)
        a, b = torch.randint(0, k, (2, t), generator=g)
        b = torch.where(a == b, (b + 1) % k, b)
        b[0] = a[0] ^ 1                             # one pair in one group
        x = torch.zeros(t, k)
        x[torch.arange(t), a] = 1
        x[torch.arange(t), b] = -1
        x = x.cuda()
        want = (w[:, a.cuda()] - w[:, b.cuda()]).t()
        assert torch.equal(want.float().double(), want)
        assert torch.equal(w4_linear(x.to(dtype), q, s), want.float().to(dtype)), t
        xs = torch.full((t,), 0.25, device="cuda")
        assert torch.equal(w4_linear(x.to(torch.float8_e4m3fn), q, s, x_scale=xs), (want / 4).float().to(dtype)), t


# widths of decoders that are no multiple of 2048 along k, groups of 128; one token, a frontier, a tree
@pytest.mark.parametrize("t", [1, 8, 65])
@pytest.mark.parametrize("n,k", [(5120, 5120), (4096, 11008), (3584, 2560), (18944, 3584), (1024, 13824)])
def test_decoder_widths(t, n, k):
    from specverify.runtime import w4_linear
    x, q, s = problem(t, n, k, 128, torch.bfloat16, seed=t + k)
    check(w4_linear(x, q, s), x, q, s)
    x8, xs = to_fp8(x)
    check(w4_linear(x8, q, s, x_scale=xs), x8, q, s, xs)


@pytest.mark.parametrize("t,n,k,group", [(130, 300, 512, 128), (257, 4099, 1056, 32), (600, 1000, 2048, 64)])
def test_8_bit_rows_of_a_prompt(t, n, k, group):
    from specverify.runtime import w4_linear
    x, q, s = problem(t, n, k, group, torch.float16, seed=t)
    x8, xs = to_fp8(x)
    check(w4_linear(x8, q, s, x_scale=xs), x8, q, s, xs)


@pytest.mark.parametrize("t", [3, 20])
@pytest.mark.parametrize("value", [2.0 ** -60, 2.0 ** 110])
def test_small_and_large_rows(t, value):
    """bf16 sums are held times 2^-40; far from 1 they keep fp32's precision all the same (products here of 2^-70 and
    2^-10 times 2^110)."""
    from specverify.runtime import w4_linear
    _, q, s = problem(t, 200, 512, 128, torch.bfloat16, seed=8)
    g = torch.Generator(device="cuda").manual_seed(3)
    x = (value * torch.randn(t, 512, device="cuda", generator=g)).to(torch.bfloat16)
    check(w4_linear(x, q, s), x, q, s)
