"""The decode loop on 4-bit projections and with the residual rule: the same
defining properties as with 16-bit weights and matched samples.  The plain
continuation, decoded one token at a time, is what the speculative loop has
to reproduce; at a temperature near zero the residual rule accepts and draws
the argmax.

The two may part where the two largest logits are closer than the roundings
of a one-row and a many-row step: some ten bf16 roundings (2^-8 of a value,
one after another) of logits whose deviation is sqrt(512) = 23 move a logit by
23 * 2^-8 * sqrt(10) = 0.28, so a lead of 1.5 is more than five deviations and
what follows a smaller one is not compared."""

from __future__ import annotations

import pytest
import torch

from conftest import cuda_ok

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a CUDA device")]

PROMPT = 300


def _model(bits=4, fp8=False, group=128):
    from specverify.draft.spec_decode import LlamaShape, SpecDecodeModel
    shape = LlamaShape(hidden=512, layers=4, heads=4, kv_heads=2, head_dim=128, ffn=1024, vocab=1000,
                       draft_vocab=1000, feature_layers=(0, 1, 2))
    m = SpecDecodeModel.from_config(shape, device="cuda", seed=0, max_tokens=1024, draft_ctx=256, weight_bits=bits,
                                    group=group, act_fp8=fp8)
    m.lm_head.normal_(0.0, 1.0, generator=torch.Generator(device="cuda").manual_seed(9))
    return m


def _plain_greedy(m, root, start, n):
    from specverify.runtime import pack_tree_mask
    bits = pack_tree_mask(torch.ones(1, 1, dtype=torch.int8, device="cuda"))[0]
    out, tok = [], root
    for i in range(n):
        hidden, _ = m.verify(torch.tensor([tok], device="cuda"), torch.tensor([start + i], device="cuda"), bits, start + i)
        top = (hidden @ m.lm_head.t()).float()[0].topk(2)
        tok = int(top.indices[0].item())
        out.append((tok, float(top.values[0] - top.values[1])))
    return out


def _same_until_close(got, plain):
    """Tokens equal up to the first that leads by less than 1.5; how many that are."""
    for i, (tok, lead) in enumerate(plain[:len(got)]):
        if lead < 1.5:
            return i
        assert got[i] == tok, (i, lead)
    return len(got)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("acceptance,temperature", [("match", 0.0), ("residual", 1e-4)])
def test_speculative_decode_on_4_bit_weights_equals_the_plain_one(fp8, acceptance, temperature):
    m = _model(fp8=fp8)
    root = m.fill_context(PROMPT, seed=4)
    want = _plain_greedy(m, root, PROMPT, 16)
    r = m.diffspec_generate(PROMPT, max_new_tokens=16, nodes=8, max_depth=4, temperature=temperature, seed=4,
                            acceptance=acceptance)
    assert _same_until_close(r["tokens"], want) >= 3
    assert r["final_length"] == PROMPT + sum(a + 1 for a in r["accepted_per_step"])


@pytest.mark.parametrize("bits", [4, 16])
def test_residual_rule_accepts_the_true_chain_and_compacts_it(bits):
    from specverify.runtime.draft_tree import finalize_tree
    m = _model(bits=bits)
    root = m.fill_context(PROMPT, seed=5)
    plain = _plain_greedy(m, root, PROMPT, 10)
    want = [t for t, _ in plain]
    depth = next((i for i, (_, lead) in enumerate(plain[:6]) if lead < 1.5), 6) - 1
    assert depth >= 1
    tree = finalize_tree(torch.arange(depth, device="cuda"), torch.zeros(depth, 1, dtype=torch.int64, device="cuda"),
                         torch.tensor(want[:depth], device="cuda").view(depth, 1), depth, 1, validate=True)
    m.fill_context(PROMPT, seed=5)
    acc, _, _ = m.step(torch.tensor([root], device="cuda"), torch.zeros(1, 3 * 512, device="cuda", dtype=m.dtype),
                       PROMPT, 1, depth, 1e-4, 0, 0, tree=tree, acceptance="residual")
    h = acc.to_host()
    assert h["accept_length"] == depth and h["best_candidate"][1:] == want[:depth] and h["next_token"] == want[depth]
    rest = _plain_greedy(m, want[depth], PROMPT + depth + 1, 10 - depth - 1)
    _same_until_close([t for t, _ in rest], plain[depth + 1:])


@pytest.mark.parametrize("fp8", [False, True])
def test_graphed_verify_equals_eager_verify(fp8):
    from specverify.runtime import pack_tree_mask
    m = _model(fp8=fp8, group=64)
    m.fill_context(PROMPT, seed=6)
    t = 9
    bits = pack_tree_mask(torch.tril(torch.ones(t, t, dtype=torch.int8, device="cuda")))[0]
    g = torch.Generator(device="cuda").manual_seed(1)
    for start in (PROMPT, PROMPT + 5):
        ids = torch.randint(0, m.shape.vocab, (t,), device="cuda", generator=g)
        pos = start + torch.arange(t, device="cuda")
        h_e, f_e = (x.clone() for x in m.verify(ids, pos, bits, start))
        h_g, f_g = m.verify_graphed(ids, pos, bits, start)
        torch.cuda.synchronize()
        assert torch.equal(h_g, h_e) and torch.equal(f_g, f_e)


def test_4_bit_layers_follow_the_16_bit_formula():
    """One verify step against the same layers in fp32 torch operations on the weights that the 4 bits stand for.
    The bf16 roundings along four layers are those of the 16-bit loop: 2^-8 a value, some ten in a row a layer."""
    from specverify.runtime import dequantize_w4, pack_tree_mask
    m = _model()
    m.fill_context(PROMPT, seed=7)
    t = 5
    bits = pack_tree_mask(torch.tril(torch.ones(t, t, dtype=torch.int8, device="cuda")))[0]
    ids = torch.tensor([3, 99, 500, 7, 12], device="cuda")
    pos = PROMPT + torch.arange(t, device="cuda")
    pool = m.pool.clone()
    h4, _ = m.verify(ids, pos, bits, PROMPT)
    m.pool.copy_(pool)
    m16 = _model(bits=16)
    for a, b in zip(m16.layers, m.layers):
        for w in ("wqkv", "wo", "wgu", "wdown"):
            setattr(a, w, dequantize_w4(*getattr(b, w)))
    m16.pool.copy_(pool)
    m16.embed, m16.lm_head = m.embed, m.lm_head
    h16, _ = m16.verify(ids, pos, bits, PROMPT)
    d = (h4.double() - h16.double()).norm() / h16.double().norm()
    assert float(d) < 40 * 2.0 ** -8                  # forty roundings in the same direction


def test_arguments():
    from specverify.draft.spec_decode import SpecDecodeModel
    with pytest.raises(ValueError):
        _model(bits=8)
    with pytest.raises(ValueError):
        _model(bits=16, fp8=True)
    m = _model()
    with pytest.raises(ValueError):
        m.diffspec_generate(PROMPT, 4, 8, 4, temperature=0.0, acceptance="residual")
    with pytest.raises(ValueError):
        m.diffspec_generate(PROMPT, 4, 8, 4, acceptance="other")
    assert isinstance(m, SpecDecodeModel)


@pytest.mark.parametrize("seed", [0, 2 ** 45 + 3, 2 ** 62])
def test_residual_rule_takes_large_seeds(seed):
    m = _model()
    a = m.diffspec_generate(PROMPT, 4, 8, 4, temperature=1.0, seed=seed, max_steps=2, acceptance="residual")
    b = m.diffspec_generate(PROMPT, 4, 8, 4, temperature=1.0, seed=seed, max_steps=2, acceptance="residual")
    assert a["steps"] >= 1 and a["tokens"] == b["tokens"]


def test_residual_rule_draws_other_numbers_for_every_seed_and_step(monkeypatch):
    """Seeds that agree in their low 43 bits, and a step number that runs past 20 bits: no number is shared (nine of
    24 bits each: by chance two sets have one in common once in 2^17), and the same seed and step repeat theirs."""
    from specverify.draft import spec_decode
    m = _model()
    root = m.fill_context(PROMPT, seed=5)
    feat = torch.zeros(1, 3 * 512, device="cuda", dtype=m.dtype)
    seen = []
    rule = spec_decode.accept_residual

    def record(logits, draft, parent, uniform, **kw):
        seen.append(uniform.tolist())
        return rule(logits, draft, parent, uniform, **kw)

    monkeypatch.setattr(spec_decode, "accept_residual", record)
    runs = [(0, 0), (3, 0), (2 ** 45 + 3, 0), (2 ** 62, 0), (2 ** 63 + 3, 0), (-1, 0), (1, 0), (0, 1), (0, 2 ** 20),
            (0, 2 ** 32), (2 ** 43, 0)]
    for seed, offset in runs + runs[:1]:
        m.step(torch.tensor([root], device="cuda"), feat, PROMPT, 2, 4, 1.0, seed, offset, acceptance="residual")
    assert seen[-1] == seen[0] and len(seen[0]) == 9
    for i in range(len(runs)):
        for j in range(i):
            assert not set(seen[i]) & set(seen[j]), (runs[i], runs[j])


def test_a_step_refuses_an_acceptance_that_it_does_not_know():
    m = _model()
    root = m.fill_context(PROMPT, seed=5)
    before = m.pool.clone()
    for kw in (dict(acceptance="residua", temperature=1.0), dict(acceptance="residual", temperature=0.0)):
        with pytest.raises(ValueError):
            m.step(torch.tensor([root], device="cuda"), torch.zeros(1, 3 * 512, device="cuda", dtype=m.dtype), PROMPT, 2,
                   4, seed=0, offset=0, **kw)
    # refused before anything ran; bitwise, as rows that nothing has written yet may hold NaNs
    assert torch.equal(m.pool.view(torch.int16), before.view(torch.int16))


@pytest.mark.parametrize("bits", [4, 16])
def test_residual_rule_moves_the_accepted_rows_of_every_layer(bits):
    """The cache after a step, row by row: the accepted path's rows lie behind the context in order, in the K and V of
    every layer, bitwise as the verify step wrote them at the tree's rows."""
    from specverify.runtime.draft_tree import finalize_tree
    m = _model(bits=bits)
    root = m.fill_context(PROMPT, seed=5)
    first = _plain_greedy(m, root, PROMPT, 1)[0][0]
    # two children of the root, the second the target's own token: the path skips a row
    other = (first + 1) % m.shape.vocab
    tree = finalize_tree(torch.arange(2, device="cuda"), torch.zeros(1, 2, dtype=torch.int64, device="cuda"),
                         torch.tensor([[other, first]], device="cuda"), 1, 2, validate=True)
    m.fill_context(PROMPT, seed=5)
    state, compact = {}, m._compact

    def watch(start, acc, rows):
        state["before"] = _rows(m, start, rows)
        compact(start, acc, rows)
        state["after"] = _rows(m, start, rows)
    m._compact = watch
    acc, _, _ = m.step(torch.tensor([root], device="cuda"), torch.zeros(1, 3 * 512, device="cuda", dtype=m.dtype), PROMPT,
                       2, 1, 1e-4, 0, 0, tree=tree, acceptance="residual")
    path = acc.to_host()["path"]
    assert path == [0, 2]
    want = state["before"].clone()
    want[..., :2, :] = state["before"][..., path, :]
    assert not torch.equal(state["before"][..., 1, :], state["before"][..., 2, :])
    assert torch.equal(state["after"], want)


def _rows(m, start, rows):
    """K and V of logical rows start .. start + rows of every layer, [layers, 2, kv heads, rows, head_dim]."""
    pos = torch.arange(start, start + rows, device="cuda")
    page = m.page_table.view(-1)[pos // m.page].long()
    return m.pool[:, :, page, :, pos % m.page, :].permute(1, 2, 3, 0, 4).clone()
