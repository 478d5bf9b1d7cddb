"""Acceptance by the residual rule (``tv_residual_accept``) against a plain
64-bit walk of the tree, node by node and child by child, and against the law
it is there for: the emitted tokens are distributed as the target's own."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import cuda_ok

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a CUDA device")]

NINF = float("-inf")


def softmax64(l, t):
    x = (l - l.max()) / t
    e = np.exp(x)
    return e / e.sum()


def plain_walk(logits, draft, parent, u, q=None, t=1.0, live=None):
    """The rule as it is written: the distribution is updated and normalised at every rejection."""
    live = len(draft) if live is None else live
    node, path = 0, [0]
    while True:
        p = softmax64(logits[node], t)
        dist, nxt = p.copy(), None
        for i in range(1, live):
            if parent[i - 1] + 1 != node:
                continue
            x = draft[i]
            if q is None:
                ok = u[i] < dist[x] if dist[x] > 0 else False
            else:
                ok = u[i] * q[node][x] < dist[x]
            if ok:
                nxt = i
                break
            dist = dist.copy()
            if q is None:
                dist[x] = 0.0
            else:
                dist = np.maximum(dist - q[node], 0.0)
            if dist.sum() > 0:
                dist = dist / dist.sum()
        if nxt is None:
            break
        node = nxt
        path.append(nxt)
    w = dist if dist.sum() > 0 else p
    c = np.cumsum(w)
    token = int(np.searchsorted(c, u[0] * c[-1], side="right"))
    return path, min(token, len(p) - 1)


def level_tree(m, width, rng, per_level=8):
    parent, above, i = [], [-1], 0
    while i < m - 1:
        k = min(per_level, m - 1 - i, len(above) * width)
        parent += sorted(int(x) for x in rng.permutation(np.repeat(above, width))[:k])
        above, i = list(range(i, i + k)), i + k
    return np.array(parent, dtype=np.int64)


def problem(b, m, v, width, dtype, sampled, seed, spread=3.0, t=1.0):
    rng = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    logits = (spread * torch.randn(b, m, v, generator=g)).to(dtype)
    noisy = (logits.double() + 0.7 * torch.randn(b, m, v, generator=g).double()).numpy()
    parent = np.stack([level_tree(m, width, rng) for _ in range(b)]) if m > 1 else np.zeros((b, 0), np.int64)
    draft = rng.integers(0, v, (b, m))
    q = None
    if sampled:
        q = np.stack([[softmax64(noisy[i, j], t) for j in range(m)] for i in range(b)]).astype(np.float32)
    for i in range(b):
        for c in range(1, m):
            p = parent[i, c - 1] + 1
            if sampled:
                cdf = q[i, p].astype(np.float64).cumsum()
                draft[i, c] = min(v - 1, int(np.searchsorted(cdf, rng.random() * cdf[-1], side="right")))
            else:
                rank = int((parent[i, :c - 1] + 1 == p).sum())
                draft[i, c] = np.argsort(-noisy[i, p])[min(rank, v - 1)]
    u = rng.random((b, m), dtype=np.float32)
    return logits, draft, parent, u, q


def check(acc, logits, draft, parent, u, q=None, t=1.0, counts=None):
    res, nxt = acc.result.cpu().numpy(), acc.next_tokens.cpu().numpy()
    b, m = draft.shape
    accepted = 0
    for i in range(b):
        live = m if counts is None else int(counts[i])
        path, token = plain_walk(logits[i].double().numpy(), draft[i], parent[i], u[i].astype(np.float64),
                                 None if q is None else q[i].astype(np.float64), t, live)
        accepted += len(path) - 1
        want = np.full(8 + 2 * m, -1, dtype=np.int64)
        want[:8] = [0, path[-1], len(path), token, 0, 0, 0, 0]
        want[8:8 + len(path)] = path
        want[8 + m:8 + m + len(path)] = draft[i][path]
        assert res[i].tolist() == want.tolist(), i
        only = np.full(m, -1)
        only[path[-1]] = token
        assert nxt[i].tolist() == only.tolist(), i
    return accepted


def cuda(*xs):
    return [None if x is None else (x if torch.is_tensor(x) else torch.from_numpy(x)).cuda() for x in xs]


@pytest.mark.parametrize("sampled", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("b,m,v,width,t", [(1, 1, 1, 1, 1.0), (3, 1, 37, 1, 0.7), (2, 2, 2, 1, 1.0),
                                           (5, 6, 1000, 1, 0.75), (2, 33, 4099, 8, 1.0), (3, 17, 32000, 2, 1.3),
                                           (4, 40, 257, 3, 0.5)])
def test_matches_the_plain_walk(sampled, dtype, b, m, v, width, t):
    from specverify.draft import accept_residual
    logits, draft, parent, u, q = problem(b, m, v, width, dtype, sampled, seed=m * 31 + v, t=t)
    cl, cd, cp, cu, cq = cuda(logits, draft, parent, u, q)
    acc = accept_residual(cl, cd, cp, cu, draft_probs=cq, temperature=t)
    check(acc, logits, draft, parent, u, q, t)
    again = accept_residual(cl, cd, cp, cu, draft_probs=cq, temperature=t)
    assert torch.equal(acc.result, again.result) and torch.equal(acc.next_tokens, again.next_tokens)


@pytest.mark.parametrize("sampled", [False, True])
def test_target_vocabulary_and_single_tree_form(sampled):
    """One 65-row tree over 128256 words, without a batch dimension; the result drives the compaction."""
    from specverify.draft import accept_residual, compact_kv
    b, m, v = 1, 65 if not sampled else 9, 128256
    logits, draft, parent, u, q = problem(b, m, v, 8 if not sampled else 2, torch.bfloat16, sampled, seed=5)
    u[:, 1:] *= 1e-3                                  # a walk of some length
    cl, cd, cp, cu, cq = cuda(logits[0], draft[0], parent[0], u[0], None if q is None else q[0])
    acc = accept_residual(cl, cd, cp, cu, draft_probs=cq)
    path, token = plain_walk(logits[0].double().numpy(), draft[0], parent[0], u[0].astype(np.float64),
                             None if q is None else q[0].astype(np.float64))
    assert len(path) >= 2
    h = acc.to_host()
    assert h["path"] == path and h["next_token"] == token and h["best_candidate"] == draft[0][path].tolist()
    assert h["accept_length"] == len(path) - 1 and int(acc.next_tokens[h["max_id"]]) == token
    kv = torch.randn(4, 20 + m, 64, device="cuda").bfloat16()
    want = kv.clone()
    want[:, 20:20 + len(path)] = kv[:, [20 + i for i in path]]
    compact_kv([kv], 20, acc)
    assert torch.equal(kv, want)


def test_padded_batch_reads_nothing_behind_the_last_node():
    from specverify.draft import accept_residual
    b, m, v = 6, 9, 3001
    logits, draft, parent, u, q = problem(b, m, v, 2, torch.float32, True, seed=3)
    counts = np.array([1, 9, 4, 2, 7, 5], dtype=np.int32)
    lg, dr, pa, un, pr = logits.clone(), draft.copy(), parent.copy(), u.copy(), q.copy()
    for i, c in enumerate(counts):
        lg[i, c:] = float("nan")
        pr[i, c:] = np.nan
        dr[i, c:] = -7
        pa[i, c - 1:] = 10 ** 6
        un[i, c:] = np.nan
    cl, cd, cp, cu, cq, cc = cuda(lg, dr, pa, un, pr, counts)
    acc = accept_residual(cl, cd, cp, cu, draft_probs=cq, counts=cc)
    check(acc, logits, draft, parent, u, q, counts=counts)
    assert [s["accept_length"] for s in acc.to_host()] == [acc.sequence(i).to_host()["accept_length"] for i in range(b)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_and_unaligned_views(dtype):
    from specverify.draft import accept_residual
    b, m, v = 3, 12, 1003
    logits, draft, parent, u, q = problem(b, m, v, 2, dtype, True, seed=9)
    big = torch.full((b, 2 * m, v + 6), float("nan"), dtype=dtype)
    big[:, ::2, 3:3 + v] = logits
    qbig = torch.full((b, m, v + 1), float("nan"))
    qbig[:, :, 1:] = torch.from_numpy(q)
    cb, qb = big.cuda(), qbig.cuda()
    wide = torch.zeros(b, 2 * m, dtype=torch.int64)
    wide[:, :m] = torch.from_numpy(draft)
    uw = torch.zeros(b, m + 3)
    uw[:, 3:] = torch.from_numpy(u)
    acc = accept_residual(cb[:, ::2, 3:3 + v], wide.cuda()[:, :m], *cuda(parent), uw.cuda()[:, 3:],
                          draft_probs=qb[:, :, 1:])
    check(acc, logits, draft, parent, u, q)
    # draft probabilities in 16 bits
    q16 = torch.from_numpy(q).to(torch.bfloat16)
    acc = accept_residual(*cuda(logits, draft, parent, u), draft_probs=q16.cuda())
    check(acc, logits, draft, parent, u, q16.float().numpy())


def one(logits, draft, parent, u, q=None, t=1.0):
    from specverify.draft import accept_residual
    lg = torch.tensor(logits, dtype=torch.float32)
    acc = accept_residual(lg.cuda(), torch.tensor(draft).cuda(), torch.tensor(parent, dtype=torch.int64).cuda(),
                          torch.tensor(u, dtype=torch.float32).cuda(),
                          draft_probs=None if q is None else torch.tensor(q, dtype=torch.float32).cuda(), temperature=t)
    return acc.to_host()


def test_borders_and_masks():
    lo = [0.0, NINF, 0.0, NINF]                       # p = 1/2, 0, 1/2, 0
    # u = 0 draws the first word with any weight, u just below 1 the last
    assert one([[NINF, 0.0, 0.0, NINF]], [0], [], [0.0])["next_token"] == 1
    assert one([[NINF, 0.0, 0.0, NINF]], [0], [], [0.99999994])["next_token"] == 2
    # out-of-range numbers are taken as the ends
    assert one([lo], [0], [], [1.0])["next_token"] == 2
    assert one([lo], [0], [], [float("nan")])["next_token"] == 0
    # a draft of probability 0 is never accepted, one of probability 1 always
    assert one([lo, lo], [0, 1], [-1], [0.0, 0.0])["accept_length"] == 0
    assert one([[NINF, 5.0], lo[:2]], [0, 1], [-1], [0.5, 0.99999994])["path"] == [0, 1]
    # a rejected draft cannot be drawn; the same word again is not accepted
    h = one([lo, lo, lo], [0, 0, 0], [-1, -1], [0.0, 0.6, 0.0])
    assert h["path"] == [0] and h["next_token"] == 2
    # the second sibling is tried with what the first one left: p = 1/2 of 1/2
    h = one([lo, lo, lo], [0, 0, 2], [-1, -1], [0.0, 0.6, 0.999])
    assert h["path"] == [0, 2] and h["best_candidate"] == [0, 2]
    # sampled drafts: p == q is always accepted; p < q leaves (p - q)+
    q = [[0.5, 0.0, 0.5, 0.0]] * 2
    assert one([lo, lo], [0, 2], [-1], [0.3, 0.99], q)["path"] == [0, 1]
    q = [[1.0, 0.0, 0.0, 0.0]] * 2
    h = one([lo, lo], [0, 0], [-1], [0.0, 0.75], q)
    assert h["path"] == [0] and h["next_token"] == 2
    # nothing left after a rejection (u = 1 is outside its range): p itself
    q = [[0.5, 0.0, 0.5, 0.0]] * 2
    assert one([lo, lo], [0, 0], [-1], [0.75, 1.0], q)["next_token"] == 2
    # rows that the walk does not end at may hold anything
    bad = [float("nan")] * 4
    assert one([lo, bad, bad], [0, 1, 3], [-1, -1], [0.1, 0.5, 0.5])["path"] == [0]
    q = [[0.25] * 4, bad]
    assert one([lo, lo], [0, 0], [-1], [0.9, 0.9], q)["path"] == [0, 1]


@pytest.mark.parametrize("row", [[NINF] * 4, [0.0, float("nan"), 0.0, 0.0], [0.0, float("inf"), 0.0, 0.0]])
def test_rows_that_are_no_distribution_are_reported(row):
    from specverify import SpecVerifyError
    from specverify.draft import accept_residual
    ok = [0.0, 1.0, 0.0, 2.0]
    lg = torch.tensor([[ok, ok], [row, ok], [ok, row]]).cuda()
    # sequences 0 and 2 accept their draft and end at their second row
    u = torch.tensor([[0.5, 0.0], [0.5, 0.0], [0.5, 0.0]]).cuda()
    acc = accept_residual(lg, torch.tensor([[0, 3]] * 3).cuda(), torch.tensor([[-1]] * 3).cuda(), u)
    assert acc.sequence(0).to_host()["path"] == [0, 1]
    for i in (1, 2):
        with pytest.raises(SpecVerifyError):
            acc.sequence(i).to_host()
        r = acc.result[i].tolist()
        assert r[0] == -6 and r[2] == 0 and r[3] == -1 and set(r[8:]) == {-1}
        assert acc.next_tokens[i].tolist() == [-1, -1]


def test_bad_trees_are_reported_not_followed():
    from specverify.draft import accept_residual
    g = torch.Generator().manual_seed(0)
    lg = torch.randn(7, 4, 50, generator=g).cuda()
    draft = torch.randint(0, 50, (7, 4), generator=g)
    parent = torch.tensor([[-1, 0, 0]] * 7)
    parent[1, 2] = 3                # past the tree
    parent[2, 1] = 2                # a later node
    parent[3, 0] = -2
    draft[4, 2] = 50
    draft[5, 1] = -1
    counts = torch.tensor([4, 4, 4, 4, 4, 4, 5], dtype=torch.int32)
    acc = accept_residual(lg, draft.cuda(), parent.cuda(), torch.rand(7, 4, generator=g).cuda(), counts=counts.cuda())
    assert acc.result[:, 0].tolist() == [0] + [-6] * 6
    # a draft's own index is another way to say "child of the root"
    same = [accept_residual(lg[:1], draft[:1].cuda(), torch.tensor([p]).cuda(), torch.tensor([[0.5, 0.9, 0.9, 0.9]]).cuda())
            for p in ([-1, -1, 1], [0, 1, 1])]
    assert torch.equal(same[0].result, same[1].result) and same[0].result[0, 0].item() == 0
    counts[6] = 0
    acc = accept_residual(lg, draft.cuda(), parent.cuda(), torch.rand(7, 4, generator=g).cuda(), counts=counts.cuda())
    assert acc.result[6, 0].item() == -6 and acc.result[0, 0].item() == 0


@pytest.mark.parametrize("sampled", [False, True])
def test_emitted_tokens_follow_the_target(sampled):
    """The first emitted token over 40000 sequences with two children each: chi-square against p (7 degrees of
    freedom, 24.3 at p = 0.001), though the drafts come from another distribution."""
    from specverify.draft import accept_residual
    n, v = 40000, 8
    g = torch.Generator().manual_seed(7 + sampled)
    row = torch.tensor([2.0, 1.0, 0.5, 0.0, -1.0, 0.3, 1.5, -0.5])
    lg = row.repeat(n, 3, 1)
    q = torch.softmax(torch.tensor([0.0, 2.0, 0.5, 1.0, 0.0, -1.0, 0.5, 0.0]), -1)
    draft = torch.zeros(n, 3, dtype=torch.int64)
    if sampled:
        draft[:, 1:] = torch.multinomial(q, 2 * n, replacement=True, generator=g).view(n, 2)
    else:
        draft[:, 1:] = torch.tensor([1, 3])
    u = torch.rand(n, 3, generator=g)
    acc = accept_residual(lg.cuda(), draft.cuda(), torch.full((n, 2), -1).cuda(), u.cuda(),
                          draft_probs=q.repeat(n, 3, 1).cuda() if sampled else None)
    res = acc.result.cpu()
    assert (res[:, 0] == 0).all()
    first = torch.where(res[:, 2] == 2, res[:, 8 + 3 + 1], res[:, 3])
    counts = torch.bincount(first, minlength=v).double()
    want = torch.softmax(row.double(), -1) * n
    assert float(((counts - want) ** 2 / want).sum()) < 24.3
    # how often a draft is accepted: p(1) + p(3) for the fixed ones (0.190), at least sum min(p, q) for the sampled
    # ones; four deviations of a share of 40000 draws are at most 4 * 0.5 / 200
    rate, p = float((res[:, 2] == 2).double().mean()), want / n
    if sampled:
        assert float(torch.minimum(p, q.double()).sum()) - 0.01 < rate < 1.0
    else:
        assert abs(rate - float(p[1] + p[3])) < 0.01


def test_side_stream_and_captured_graph():
    from specverify.draft import accept_residual
    sets = [problem(2, 9, 5003, 2, torch.bfloat16, True, seed=s) for s in (1, 2)]
    logits, draft, parent, u, q = (x.cuda() for x in (sets[0][0], *[torch.from_numpy(y) for y in sets[0][1:]]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        acc = accept_residual(logits, draft, parent, u, draft_probs=q)
    side.synchronize()
    check(acc, *sets[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        acc = accept_residual(logits, draft, parent, u, draft_probs=q)
        acc2 = accept_residual(logits, draft, parent, u)
    for s in (sets[1], sets[0]):
        for buf, new in zip((logits, draft, parent, u, q), s):
            buf.copy_(new if torch.is_tensor(new) else torch.from_numpy(new))
        graph.replay()
        torch.cuda.synchronize()
        check(acc, *s)
        check(acc2, *s[:4])


def test_wide_trees_and_empty_batches():
    """1024 nodes, all children of the root with many repeated words; a batch of none."""
    from specverify.draft import accept_residual
    m, v = 1024, 600
    g = torch.Generator().manual_seed(2)
    logits = torch.randn(1, m, v, generator=g)
    draft = torch.randint(0, v, (1, m), generator=g).numpy()
    parent = np.full((1, m - 1), -1)
    u = np.full((1, m), 0.999999, dtype=np.float32)
    acc = accept_residual(*cuda(logits, draft, parent, u))
    check(acc, logits, draft, parent, u)
    acc = accept_residual(logits[:0].cuda(), *cuda(draft[:0], parent[:0], u[:0]))
    assert acc.result.shape == (0, 8 + 2 * m)


def test_refusals():
    from specverify import SpecVerifyError
    from specverify.draft import accept_residual
    lg, d = torch.zeros(2, 3, 10).cuda(), torch.zeros(2, 3, dtype=torch.int64).cuda()
    p, u = torch.full((2, 2), -1).cuda(), torch.zeros(2, 3).cuda()
    ok = dict(draft_probs=None, temperature=1.0, counts=None)
    accept_residual(lg, d, p, u, **ok)
    bad = [((lg.double(), d, p, u), {}), ((lg, d.int(), p, u), {}), ((lg, d, p, u.double()), {}),
           ((lg, d[:, :2], p, u), {}), ((lg, d, p[:, :1], u), {}), ((lg, d, p, u[:1]), {}),
           ((lg[0, 0], d, p, u), {}), ((lg.transpose(1, 2).contiguous().transpose(1, 2), d, p, u), {}),
           ((lg, d, p, u), dict(temperature=0.0)), ((lg, d, p, u), dict(temperature=float("nan"))),
           ((lg, d, p, u), dict(temperature=float("inf"))), ((lg, d, p, u), dict(draft_probs=lg[:1])),
           ((lg, d, p, u), dict(draft_probs=lg.double())),
           ((lg, d, p, u), dict(counts=torch.ones(2, dtype=torch.int64).cuda())),
           ((lg.cpu(), d, p, u), {})]
    for args, kw in bad:
        with pytest.raises(SpecVerifyError):
            accept_residual(*args, **{**ok, **kw})


@pytest.mark.parametrize("t", [0.7, 0.9, 1.3])
def test_draws_next_to_borders_at_temperatures_that_no_float_holds(t):
    """Draws beside the borders of softmax(logits / t) with t in 64 bits.  A temperature rounded to 32 bits is off by
    2^-26 to 2^-24 of itself and moves the borders by some 2^-29 of the sum, all of a row the same way.  The uniform
    numbers here lie between 2^-32 and 2^-29 of the sum from a border; the kernel's own error is that of its weights
    (2^-36 each) and of their sum (the pairs' l parts, below 2^-40), the 80-bit CDF's is below 2^-46."""
    from specverify.draft import accept_residual
    v = 128256
    g = torch.Generator().manual_seed(int(100 * t))
    logits = (3.0 * torch.randn(1, 1, v, generator=g)).to(torch.float16)
    x = logits[0, 0].double().numpy().astype(np.longdouble)
    cdf = np.cumsum(np.exp((x - x.max()) / np.longdouble(t)))
    cdf /= cdf[-1]
    u = cdf[:-1].astype(np.float32)
    far = np.abs(u.astype(np.longdouble) - cdf[:-1])
    u = u[(far > 2.0 ** -32) & (far < 2.0 ** -29) & (u < 1)]
    assert len(u) > 2000
    # numbers near 0 are finer than the borders' errors: only the nearest border decides how far one is
    want = np.searchsorted(cdf, u.astype(np.longdouble), side="right")
    near = np.minimum(np.abs(cdf[np.minimum(want, v - 1)] - u), np.abs(u - cdf[np.maximum(want - 1, 0)]))
    u, want = u[near > 2.0 ** -32], want[near > 2.0 ** -32]
    b = len(u)
    acc = accept_residual(logits.cuda().expand(b, 1, v), torch.zeros(b, 1, dtype=torch.int64, device="cuda"),
                          torch.zeros(b, 0, dtype=torch.int64, device="cuda"), torch.from_numpy(u)[:, None].cuda(),
                          temperature=t)
    assert (acc.result[:, 0] == 0).all()
    wrong = int((acc.result[:, 3].cpu().numpy() != want).sum())
    assert wrong == 0, (wrong, b)
