"""Residual addition + RMSNorm (``tv_add_rms_norm``) against its formula in 64
bits.

Tolerances.  A rounding is off by at most half a step: 2^-8 of the value in
bf16, 2^-11 in fp16, 2^-4 in e4m3 (and half the smallest subnormal, 2^-25 in
fp16, 2^-10 in e4m3, below the normal range).  The sum of squares is at most
16384 / 512 terms a thread in sequence plus two trees, rsqrtf and three fp32
products: together below 2^-16 of the value.  The 16-bit output is rounded
twice (before and after the weight), the 8-bit one once, at a scale that has
the same fp32 error."""

from __future__ import annotations

import pytest
import torch

from conftest import cuda_ok

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a CUDA device")]

EPS = 1e-5
F32 = 2.0 ** -16
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SUB = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def problem(rows, cols, dtype, seed=0, spread=4.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, device="cuda", generator=g).to(dtype)
    r = (spread * torch.randn(rows, cols, device="cuda", generator=g)).to(dtype)
    w = (1 + 0.2 * torch.randn(cols, device="cuda", generator=g)).to(dtype)
    return x, r, w


def formula(h, w, eps=EPS):
    f = h.double()
    return f / (f.square().mean(1, keepdim=True) + eps).sqrt() * w.double()


def check(x, r, w, out, fp8, eps=EPS):
    h = out[-1]
    assert torch.equal(h, x + r)                       # torch's addition rounds once, from fp32
    want = formula(h, w, eps)
    if not fp8:
        t = x.dtype
        off = (out[0].double() - want).abs()
        tol = want.abs() * ((1 + HALF[t]) ** 2 - 1 + F32) + SUB[t] * (w.double().abs() + 1)
        assert bool((off <= tol).all()), float((off - tol).max())
        return
    y, scale, _ = out
    assert y.dtype == torch.float8_e4m3fn and scale.dtype == torch.float32
    amax = want.abs().amax(1)
    assert bool(((scale.double() - amax / 448).abs() <= amax / 448 * F32).all())
    s = scale.double()[:, None]
    off = (y.double() * s - want).abs()
    tol = want.abs() * (2.0 ** -4 + F32) + s * 2.0 ** -10
    assert bool((off <= tol).all()), float((off - tol).max())
    if want.shape[1]:
        assert bool((y.float().abs().amax(1) >= 416).all())     # the largest value sits at the top of the range


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (1, 8), (65, 4096), (7, 4101), (5, 2052), (2, 8200), (3, 16384),
                                       (2, 16392), (2, 9001), (1, 65536), (301, 640)])
def test_matches_the_formula(rows, cols, dtype, fp8):
    from specverify.runtime import add_rms_norm
    x, r, w = problem(rows, cols, dtype, seed=rows + cols)
    keep = (x.clone(), r.clone())
    out = add_rms_norm(x, r, w, EPS, fp8=fp8)
    check(x, r, w, out, fp8)
    assert torch.equal(x, keep[0]) and torch.equal(r, keep[1])
    again = add_rms_norm(x, r, w, EPS, fp8=fp8)
    for a, b in zip(out, again):
        assert torch.equal(a.view(torch.uint8) if a.dtype == torch.float8_e4m3fn else a,
                           b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_in_place_residual_strides_and_the_two_step_form(dtype):
    from specverify.draft.spec_decode import rms_norm
    from specverify.runtime import add_rms_norm
    x, r, w = problem(65, 4096, dtype)
    y, h = add_rms_norm(x, r, w, EPS)
    two = rms_norm(x + r, w, EPS)
    # same roundings; the sum of squares is taken in another order, which may move a rounding by one step
    assert float((y != two).float().mean()) < 0.01
    inplace = r.clone()
    y2, h2 = add_rms_norm(x, inplace, w, EPS, residual_out=inplace)
    assert h2 is inplace and torch.equal(inplace, h) and torch.equal(y2, y)
    # every other row, unaligned columns, one broadcast row added to all
    big = torch.randn(130, 4099, device="cuda").to(dtype)
    xs = big[::2, 3:]
    check(xs, r, w, add_rms_norm(xs, r, w, EPS), False)
    check(xs, r, w, add_rms_norm(xs, r, w, EPS, fp8=True), True)
    row = x[:1].expand(65, 4096)
    check(row, r, w, add_rms_norm(row, r, w, EPS), False)
    # rows around a strided output stay as they were
    buf = torch.full((130, 4096), 7.0, device="cuda").to(dtype)
    add_rms_norm(x, r, w, EPS, residual_out=buf[::2])
    assert torch.equal(buf[::2], h) and bool((buf[1::2] == 7).all())


def test_zero_nan_inf_and_tiny_rows():
    from specverify.runtime import add_rms_norm
    x, r, w = problem(6, 512, torch.bfloat16)
    x[1] = 0
    r[1] = 0
    x[2, 5] = float("nan")
    x[3, 6] = float("inf")
    x[4] = -r[4]
    x[5] = 1e-30
    r[5] = 0
    y, h = add_rms_norm(x, r, w, 0.0 + 1e-5)
    assert bool((y[1] == 0).all()) and bool((y[4] == 0).all()) and bool(y[2].isnan().all())
    assert bool(y[3, 6].isnan()) and bool((y[3, :6] == 0).all())
    y8, s, _ = add_rms_norm(x, r, w, 1e-5, fp8=True)
    f = y8.float()
    assert bool((f[1] == 0).all()) and s[1] == 0 and s[4] == 0 and bool((f[4] == 0).all())
    assert bool(f[2].isnan().all()) and bool(s[2].isnan()) and bool(s[3].isnan())
    for i in (0, 5):
        check(x[i:i + 1], r[i:i + 1], w, (y8[i:i + 1], s[i:i + 1], h[i:i + 1]), True)
    # a row whose scale is far below the normal range of its reciprocal
    t = torch.full((1, 64), 1e-36, device="cuda").bfloat16()
    y8, s, _ = add_rms_norm(t, torch.zeros_like(t), torch.ones(64, device="cuda").bfloat16(), 1.0, fp8=True)
    assert bool(torch.isfinite(y8.float()).all())
    # eps 0 keeps a tiny row's direction
    t = (torch.arange(1, 65, device="cuda")[None] * 1e-12).bfloat16()
    one = torch.ones(64, device="cuda").bfloat16()
    check(t, torch.zeros_like(t), one, add_rms_norm(t, torch.zeros_like(t), one, 0.0), False, eps=0.0)


def test_empty_side_stream_and_captured_graph():
    from specverify.runtime import add_rms_norm
    x, r, w = problem(33, 1024, torch.float16)
    out = add_rms_norm(x[:0], r[:0], w, EPS, fp8=True)
    assert [tuple(t.shape) for t in out] == [(0, 1024), (0,), (0, 1024)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = add_rms_norm(x, r, w, EPS, fp8=True)
    side.synchronize()
    check(x, r, w, out, True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a = add_rms_norm(x, r, w, EPS)
        b = add_rms_norm(a[0], a[1], w, EPS, fp8=True)
    for seed in (4, 5):
        nx, nr, _ = problem(33, 1024, torch.float16, seed)
        x.copy_(nx)
        r.copy_(nr)
        g.replay()
        torch.cuda.synchronize()
        check(x, r, w, a, False)
        check(a[0], a[1], w, b, True)


def test_refusals():
    from specverify import SpecVerifyError
    from specverify.runtime import add_rms_norm
    x, r, w = problem(4, 64, torch.bfloat16)
    bad = [(x.float(), r.float(), w.float()), (x, r.half(), w), (x, r, w.half()), (x, r[:3], w), (x, r, w[:32]),
           (x[0], r[0], w), (x.t().contiguous().t(), r, w), (x.cpu(), r, w)]
    for args in bad:
        with pytest.raises(SpecVerifyError):
            add_rms_norm(*args, EPS)
    for out in (r.half(), r[:2], r[:1].expand(4, 64)):
        with pytest.raises(SpecVerifyError):
            add_rms_norm(x, r, w, EPS, residual_out=out)
