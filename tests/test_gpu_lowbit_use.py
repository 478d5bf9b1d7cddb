"""The low-bit operators and the residual rule as a program uses them: every
small row count in every form, calls at once on two streams, graphs replayed
side by side, batches around each cluster size, and tensors whose element
offsets pass 32 bits.  Tolerances are those of the operators' own tests."""

from __future__ import annotations

import pytest
import torch

import test_gpu_residual_accept as ra
from conftest import cuda_ok
from test_gpu_w4 import check, problem, to_fp8

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a CUDA device")]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
# one block of 128 k and less, blocks that do not fill a team's warps, ones that do; few and many units;
# rows that do not fit an SM's shared memory
@pytest.mark.parametrize("n,k,group", [(16, 32, 32), (17, 128, 64), (100, 480, 32), (2500, 2048, 128),
                                       (30000, 512, 64), (48, 4224, 128), (33, 14336, 128), (15, 28672, 256)])
def test_few_rows_in_every_form(n, k, group, dtype):
    from specverify.runtime import w4_linear
    for t in range(1, 9):
        x, q, s = problem(t, n, k, group, dtype, seed=t * n + k)
        want = w4_linear(x, q, s)
        check(want, x, q, s)
        wide = torch.zeros(t, k + 3, dtype=dtype, device="cuda")
        wide[:, 1:k + 1] = x                     # rows at odd addresses
        buf = torch.full((2 * t, n + 5), 5.0, dtype=dtype, device="cuda")
        # both ways of reading x sum in the same order where the same kernel takes them
        y = w4_linear(wide[:, 1:k + 1], q, s, out=buf[::2, 2:n + 2])
        check(y, x, q, s)
        assert bool((buf[1::2] == 5).all()) and bool((buf[:, :2] == 5).all()) and bool((buf[:, n + 2:] == 5).all())
        x8, xs = to_fp8(x)
        check(w4_linear(x8, q, s, x_scale=xs), x8, q, s, xs)
        # a row's result does not hang on the rows beside it
        if t > 1:
            assert torch.equal(w4_linear(x[t - 1:], q, s)[0], want[t - 1]) or k > 13000


def chain(seed, rows=65):
    """Residual and norm in 8 bits, the product of it, and the acceptance over its first words."""
    from specverify.draft import accept_residual
    from specverify.runtime import add_rms_norm, w4_linear
    x, q, s = problem(rows, 4096, 2048, 128, torch.bfloat16, seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = torch.randn(rows, 2048, device="cuda", generator=g).bfloat16()
    w = torch.rand(2048, device="cuda", generator=g).bfloat16()
    draft = torch.randint(0, 4096, (rows,), device="cuda", generator=g)
    parent = torch.arange(-1, rows - 2, device="cuda") // 2
    u = torch.rand(rows, device="cuda", generator=g)

    def run():
        y8, scale, h = add_rms_norm(x, r, w, 1e-5, fp8=True)
        logits = w4_linear(y8, q, s, x_scale=scale)
        acc = accept_residual(logits, draft, parent, u)
        return y8.view(torch.uint8), scale, h, logits, acc.result, acc.next_tokens
    return run


def test_calls_at_once_on_two_streams():
    runs = [chain(1), chain(2, 9)]
    want = [[t.clone() for t in run()] for run in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(runs[i]())
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))


def test_graphs_replayed_side_by_side():
    runs = [chain(3), chain(4)]
    want = [[t.clone() for t in run()] for run in runs]
    graphs, outs = [], []
    for run in runs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run())
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        for out in outs:
            for t in out:
                t.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(out, w))


@pytest.mark.parametrize("sampled", [False, True])
# the number of sequences decides how many SMs share one: around every step of that rule
@pytest.mark.parametrize("b,v", [(1, 40000), (7, 40000), (8, 40000), (15, 33000), (16, 33000), (22, 30000),
                                 (23, 25000), (34, 18000), (46, 9000), (75, 9000), (160, 5000)])
def test_batches_around_the_cluster_sizes(b, v, sampled):
    from specverify.draft import accept_residual
    logits, draft, parent, u, q = ra.problem(b, 4, v, 2, torch.bfloat16, sampled, seed=b + v)
    cl, cd, cp, cu, cq = ra.cuda(logits, draft, parent, u, q)
    ra.check(accept_residual(cl, cd, cp, cu, draft_probs=cq), logits, draft, parent, u, q)


def test_drafts_from_the_target_itself():
    """Draft probabilities that are the target's own, rounded: next to nothing is left of p - q."""
    from specverify.draft import accept_residual
    logits, draft, parent, u, _ = ra.problem(6, 5, 3000, 1, torch.float32, True, seed=11)
    q = torch.softmax(logits, -1)
    cl, cd, cp, cu, cq = ra.cuda(logits, draft, parent, u, q)
    acc = accept_residual(cl, cd, cp, cu * 0.999, draft_probs=cq)      # u q < p for all of them: every draft passes
    assert acc.result[:, 2].tolist() == [5] * 6
    for dt in (torch.bfloat16, torch.float16):
        acc = accept_residual(cl, cd, cp, cu, draft_probs=cq.to(dt))
        assert acc.result[:, 0].tolist() == [0] * 6
        assert bool((acc.result[:, 3] >= 0).all()) and bool((acc.result[:, 3] < 3000).all())


def test_offsets_beyond_32_bits():
    from specverify.draft import accept_residual
    from specverify.runtime import add_rms_norm, w4_linear
    # outputs: 20000 x 128256 elements
    x, q, s = problem(20000, 128256, 128, 64, torch.bfloat16, seed=1)
    y = w4_linear(x, q, s)
    for rows in (slice(0, 40), slice(19960, 20000)):
        check(y[rows].contiguous(), x[rows], q, s)
    del y
    # packed weights: 600000 x 4096 words; rows far apart
    n, k = 600000, 32768
    q = torch.randint(-2 ** 31, 2 ** 31, (n, k // 8), dtype=torch.int32, device="cuda")
    s = torch.full((n, k // 128), 0.004, device="cuda").bfloat16()
    for t in (2, 20):
        x = torch.randn(t, k, device="cuda").bfloat16()
        y = w4_linear(x, q, s)
        for cols in (slice(0, 200), slice(n - 333, n)):
            check(y[:, cols].contiguous(), x, q[cols], s[cols])
    del q, s, y
    # logits: 70 sequences of 250 rows over 128256 words
    logits = torch.randn(70, 250, 128256, device="cuda", dtype=torch.bfloat16)
    draft = torch.randint(0, 128256, (70, 250), device="cuda")
    parent = (torch.arange(-1, 248, device="cuda") // 3).expand(70, 249).contiguous()
    u = torch.rand(70, 250, device="cuda")
    acc = accept_residual(logits, draft, parent, u)
    for i in (0, 69):
        one = accept_residual(logits[i].clone(), draft[i], parent[i], u[i])
        assert torch.equal(acc.result[i], one.result.view(-1))
    del logits
    # rows of the norm
    x = torch.randn(300000, 8192, device="cuda", dtype=torch.bfloat16)
    r = torch.randn(300000, 8192, device="cuda", dtype=torch.bfloat16)
    w = torch.rand(8192, device="cuda").bfloat16()
    y8, scale, h = add_rms_norm(x, r, w, 1e-5, fp8=True)
    a8, ascale, ah = add_rms_norm(x[-5:].clone(), r[-5:].clone(), w, 1e-5, fp8=True)
    # h is the same element by element.  The sum of 8192 squares runs over 128 or 512 threads, as the number of rows
    # decides: in any order it is off by less than 8192 * 2^-24 of itself, so the two inverse roots, and with them
    # the scales, differ by less than 2^-11 and a few roundings (2^-20).  8-bit values are off by half a step each:
    # 2^-4 of the value, or 2^-10 of the scale below the normal range.
    assert torch.equal(h[-5:], ah)
    assert bool(((scale[-5:] - ascale).abs() <= (2.0 ** -11 + 2.0 ** -20) * ascale).all())
    a, b = y8[-5:].double() * scale[-5:, None].double(), a8.double() * ascale[:, None].double()
    assert bool(((a - b).abs() <= (2 * 2.0 ** -4 + 2.0 ** -10) * torch.maximum(a.abs(), b.abs())
                 + 2.0 ** -9 * ascale[:, None]).all())


def test_sizes_that_32_bits_do_not_hold_are_refused():
    """The argument blocks' sizes are 32 bits: 2^32 + 4 rows would be taken as four and the rest left unwritten."""
    from specverify import SpecVerifyError
    from specverify.draft import accept_residual
    from specverify.runtime import add_rms_norm, w4_linear
    for rows in (2 ** 31, 2 ** 32 + 4):
        one = torch.ones(1, 1, dtype=torch.bfloat16, device="cuda")
        x, q, s = problem(1, 2, 32, 32, torch.bfloat16)
        calls = [lambda: add_rms_norm(one.expand(rows, 1), one.expand(rows, 1), one[0], 1e-5),
                 lambda: w4_linear(x.expand(rows, 32), q, s),
                 lambda: w4_linear(x.expand(rows, 1, 32), q, s),
                 lambda: accept_residual(torch.zeros(1, 1, 4, device="cuda").expand(rows, 1, 4),
                                         torch.zeros(1, 1, dtype=torch.int64, device="cuda").expand(rows, 1),
                                         torch.zeros(1, 0, dtype=torch.int64, device="cuda").expand(rows, 0),
                                         torch.zeros(1, 1, device="cuda").expand(rows, 1))]
        for call in calls:
            with pytest.raises(SpecVerifyError) as e:
                call()
            assert e.value.status == -7


def test_captured_behind_copies_memsets_and_a_fork():
    """Launches that may start while their predecessor ends, captured where that predecessor is a copy, a memset, two
    kernels on different streams that meet, or one that takes its time."""
    from specverify.draft import accept_residual
    from specverify.runtime import add_rms_norm, w4_linear
    x, q, s = problem(65, 4096, 2048, 128, torch.bfloat16, seed=21)
    few, fq, fs = problem(2, 2048, 2048, 128, torch.bfloat16, seed=22)
    w = torch.rand(2048, device="cuda").bfloat16()
    r = torch.zeros_like(x)
    stage, sums = torch.zeros_like(x), torch.zeros_like(x)
    draft = torch.randint(0, 4096, (65,), device="cuda")
    parent = torch.arange(-1, 63, device="cuda") // 2
    u = torch.rand(65, device="cuda")
    big = torch.randn(4096, 4096, device="cuda")

    def run(side):
        slow = (big @ big)[0, 0] * 0                  # some hundred microseconds
        stage.copy_(x)                                # a memory copy
        sums.zero_()                                  # a memset
        y, h = add_rms_norm(stage, sums, w, 1e-5)
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            z = w4_linear(few + slow.bfloat16(), fq, fs)          # a join of two streams in front of the norm
        logits = w4_linear(y, q, s)
        here.wait_stream(side)
        r[:2] = z
        y8, scale, h2 = add_rms_norm(h, r, w, 1e-5, fp8=True)
        logits2 = w4_linear(y8, q, s, x_scale=scale)
        side.wait_stream(here)
        with torch.cuda.stream(side):
            a = accept_residual(logits, draft, parent, u)
        b = accept_residual(logits2, draft, parent, u)
        here.wait_stream(side)
        return y, h, logits, z, y8.view(torch.uint8), scale, h2, logits2, a.result, b.result

    torch.cuda.synchronize()
    want = [t.clone() for t in run(torch.cuda.Stream())]
    torch.cuda.synchronize()
    y, h, logits = want[:3]
    check(logits, y, q, s)
    check(want[3], few, fq, fs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(torch.cuda.Stream())
    for _ in range(5):
        for t in out:
            t.zero_()
        r.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_calls_from_several_threads():
    import threading
    runs = [chain(5), chain(6, 9), chain(7, 3), chain(8, 130)]
    want = [[t.clone() for t in run()] for run in runs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                out = runs[i]()
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(out, want[i])):
                    bad.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("t,n,k,group,fp8", [(1, 130, 2 ** 20, 128, False), (9, 40, 2 ** 20, 32, True),
                                             (3, 64, 104448 // 3 // 32 * 32, 32, False), (8, 33, 13056, 128, True),
                                             (8, 33, 13088, 32, False), (1, 2 ** 27, 32, 32, False)])
def test_products_at_the_ends_of_their_ranges(t, n, k, group, fp8):
    """The longest k, the most that fits an SM's shared memory and one step more, the most outputs (its last columns
    and some in between)."""
    from specverify.runtime import w4_linear
    x, q, s = problem(t, n, k, group, torch.bfloat16, seed=t)
    x, xs = to_fp8(x) if fp8 else (x, None)
    y = w4_linear(x, q, s, x_scale=xs)
    for lo in sorted({0, n // 2, max(0, n - 500)}):
        cols = slice(lo, lo + 500)
        check(y[:, cols].contiguous(), x, q[cols], s[cols], xs)


def test_a_very_wide_row():
    """2^24 + 5 columns off the 16-byte grid, one CTA a row.  A thread adds 2^15 squares one after another: the sum is
    off by less than 2^15 * 2^-24 of itself and 2^-16 for the rest, its inverse root by half of that."""
    from specverify.runtime import add_rms_norm
    cols = 2 ** 24 + 5
    g = torch.Generator(device="cuda").manual_seed(0)
    x, r = (torch.randn(2, cols, device="cuda", generator=g).bfloat16() for _ in range(2))
    w = torch.rand(cols, device="cuda", generator=g).bfloat16()
    y, h = add_rms_norm(x, r, w, 1e-5)
    assert torch.equal(h, x + r)
    f = h.double()
    want = f / (f.square().mean(1, keepdim=True) + 1e-5).sqrt() * w.double()
    off = 2.0 ** -10 + 2.0 ** -16
    assert bool(((y.double() - want).abs() <= want.abs() * ((1 + off) * (1 + 2.0 ** -8) ** 2 - 1) + 2.0 ** -125).all())


@pytest.mark.parametrize("b,m,v", [(65535, 2, 5), (2, 1024, 257), (1, 2, 4 * 2 ** 20 + 3)])
def test_acceptance_at_the_ends_of_its_ranges(b, m, v):
    """The largest batch and tree, a vocabulary of many blocks a CTA, against the rule on whole tensors in 64 bits:
    a chain whose drafts are all tried in order (every node has one child)."""
    from specverify.draft import accept_residual
    g = torch.Generator(device="cuda").manual_seed(b)
    logits = torch.randn(b, m, v, device="cuda", generator=g)
    p = torch.softmax(logits.double(), -1)
    draft = torch.randint(0, v, (b, m), device="cuda", generator=g)
    draft[:, 1:] = logits[:, :-1].argmax(-1)                       # drafts with a chance
    parent = torch.arange(-1, m - 2, device="cuda").expand(b, m - 1).contiguous()
    u = torch.rand(b, m, device="cuda", generator=g)
    if m > 100:
        u[:, 1:m // 2] *= 1e-3                                     # a path of some length
    acc = accept_residual(logits, draft, parent, u)
    pt = torch.gather(p[:, :-1], 2, draft[:, 1:, None])[..., 0]
    ok = u[:, 1:].double() < pt
    n = ok.long().cumprod(1).sum(1) + 1
    at = torch.arange(b, device="cuda")
    rest = p[at, n - 1].clone()
    has = n < m
    rest[at[has], draft[at[has], n[has]]] = 0
    cdf = rest.cumsum(-1)
    edge = u[:, 0].double() * cdf[:, -1]
    token = torch.searchsorted(cdf, edge[:, None], right=True)[:, 0].clamp(max=v - 1)
    # comparisons within 2^-20 of a border (a fp32 normaliser's few roundings, and for the draw far more than the
    # pairs' error) are left out; they are few
    near = ((u[:, 1:].double() - pt).abs() < 2.0 ** -20 * pt).any(1)
    near |= (cdf - edge[:, None]).abs().amin(1) < 2.0 ** -34
    assert float(near.double().mean()) < 0.01
    keep = ~near
    assert (acc.result[:, 0] == 0).all() and bool(keep.any())
    assert torch.equal(acc.result[keep, 2], n[keep]) and torch.equal(acc.result[keep, 3], token[keep])
