"""Argument checks of the low-bit and residual-rule entries, host only (the
pointers are never used: every refusal comes before a launch)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from specverify import SpecVerifyError, _lib

FAKE = 1 << 20


@pytest.fixture(scope="module")
def lib():
    import build
    build.build()
    return _lib.load()


def test_add_rms_norm_checks(lib):
    f = lib.tv_add_rms_norm
    good = dict(x=FAKE, xs=64, r=FAKE, rs=64, w=FAKE, h=FAKE, hs=64, y=FAKE, ys=64, s=None, rows=4, cols=64, eps=1e-5,
                dt=0)

    def call(**kw):
        return f(*{**good, **kw}.values(), None)
    assert call(rows=0) == 0                     # nothing to do
    assert call(rows=-1) == -1 and call(cols=0) == -1
    assert call(dt=2) == -2 and call(dt=7) == -2
    for k in "xrwhy":
        assert call(**{k: None}) == -8, k


def _accept(**kw):
    a = _lib.ResidualAcceptArgs()
    a.logits_dtype, a.batch, a.rows, a.vocab = 0, 2, 3, 100
    a.logits = a.draft = a.parent = a.uniform = a.next_tokens = a.result = FAKE
    a.temperature = 1.0
    a.workspace, a.workspace_bytes = FAKE, 1 << 16
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_residual_accept_checks(lib):
    def call(**kw):
        return lib.tv_residual_accept(ctypes.byref(_accept(**kw)), None)
    assert call(batch=0) == 0
    assert call(batch=-1) == -1 and call(rows=0) == -1 and call(vocab=0) == -1
    assert call(rows=1025) == -7 and call(batch=65536) == -7 and call(vocab=(1 << 30) + 1) == -7
    assert call(logits_dtype=3) == -2 and call(probs=FAKE, probs_dtype=-1) == -2
    for t in (0.0, -1.0, float("nan"), float("inf")):
        assert call(temperature=t) == -6, t
    for k in ("logits", "draft", "parent", "uniform", "next_tokens", "result"):
        assert call(**{k: None}) == -8, k
    assert call(workspace=None) == -5 and call(workspace_bytes=8) == -5
    assert call(workspace=FAKE + 8) == -3
    assert lib.tv_residual_accept(None, None) == -8
    n = ctypes.c_size_t(0)
    assert lib.tv_residual_accept_workspace_size(ctypes.byref(_accept(rows=65, vocab=128256)), ctypes.byref(n)) == 0
    assert n.value == 2 * 65 * 16 * 12 + 16      # 8192 16-bit words a chunk: 16 (max, sum) pairs a row
    assert lib.tv_residual_accept_workspace_size(ctypes.byref(_accept()), None) == -8


def test_cpu_tensors_are_refused():
    from specverify.draft import accept_residual
    from specverify.runtime import add_rms_norm
    x = torch.zeros(2, 8, dtype=torch.bfloat16)
    with pytest.raises(SpecVerifyError):
        add_rms_norm(x, x, x[0], 1e-5)
    with pytest.raises(SpecVerifyError):
        accept_residual(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64), torch.zeros(1, dtype=torch.int64),
                        torch.zeros(2))


def test_w4_linear_checks(lib):
    def args(**kw):
        a = _lib.W4Args()
        a.x_dtype = a.out_dtype = 0
        a.rows, a.n, a.k, a.group = 4, 100, 256, 64
        a.x = a.qweight = a.scales = a.out = FAKE
        a.x_sm, a.q_sn, a.s_sn, a.o_sm = 256, 32, 4, 100
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    def call(**kw):
        return lib.tv_w4_linear(ctypes.byref(args(**kw)), None)
    assert call(rows=0) == 0
    assert call(rows=-1) == -1 and call(n=0) == -1 and call(k=0) == -1
    assert call(group=48) == -1 and call(group=0) == -1 and call(group=96) == -1 and call(group=512) == -1
    assert call(out_dtype=2) == -2 and call(x_dtype=1) == -2 and call(x_dtype=2) == -2
    for k in ("x", "qweight", "scales", "out"):
        assert call(**{k: None}) == -8, k
    assert call(x_dtype=3) == -8                                # e4m3 rows need their scales
    assert call(qweight=FAKE + 4) == -3 and call(q_sn=33) == -3 and call(q_sn=28) == -1
    assert call(k=(1 << 20) + 64, q_sn=1 << 20) == -7 and call(n=(1 << 27) + 1) == -7
    # more than 8 rows that TMA cannot read are staged: 8 bits, off the 16-byte grid, or overlapping
    for kw in (dict(x_dtype=3, x_scale=FAKE), dict(x=FAKE + 2), dict(x_sm=260), dict(x_sm=0)):
        kw["rows"] = 40
        assert call(**kw) == -5, kw
        assert call(**kw, workspace=FAKE, workspace_bytes=40 * 256 * 2 - 1) == -5
        assert call(**kw, workspace=FAKE + 8, workspace_bytes=1 << 20) == -3
    assert call(rows=65535 * 128 + 1) == -7
    assert lib.tv_w4_linear(None, None) == -8
    n = ctypes.c_size_t(0)
    assert lib.tv_w4_workspace_size(ctypes.byref(args()), ctypes.byref(n)) == 0 and n.value == 0
    for rows, need in ((8, 0), (9, 9 * 256 * 2)):
        assert lib.tv_w4_workspace_size(ctypes.byref(args(x_dtype=3, rows=rows)), ctypes.byref(n)) == 0
        assert n.value == need
    assert lib.tv_w4_workspace_size(ctypes.byref(args(rows=1, x_sm=0)), ctypes.byref(n)) == 0 and n.value == 0
    assert lib.tv_w4_workspace_size(None, ctypes.byref(n)) == -8


def test_structs_match_the_header(tmp_path):
    """Size and every field's offset of the two argument blocks, as the host C compiler lays them out."""
    import shutil
    import subprocess
    from pathlib import Path
    if shutil.which("gcc") is None:
        pytest.skip("no host C compiler")
    mirrors = {"tv_residual_accept_args": _lib.ResidualAcceptArgs, "tv_w4_args": _lib.W4Args}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "specverify.h"', "int main(void) {"]
    want = []
    for cname, py in mirrors.items():
        lines.append(f'  printf("%zu\\n", sizeof({cname}));')
        want.append(ctypes.sizeof(py))
        for fname, _ in py._fields_:
            lines.append(f'  printf("%zu\\n", offsetof({cname}, {fname}));')
            want.append(getattr(py, fname).offset)
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run(["gcc", "-I", str(Path(__file__).resolve().parent.parent / "include"), str(src), "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    assert [int(x) for x in out.split()] == want


def test_compaction_takes_one_sequence(lib):
    """A batched result would have every slice moved along its first sequence's path."""
    from specverify.core.kv_cache.paged_kv import PagedKVCache, PagedKVConfig
    from specverify.draft import AcceptResult, compact_kv
    both = AcceptResult(torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 14, dtype=torch.int64), 3)
    with pytest.raises(SpecVerifyError) as e:
        compact_kv([], 0, both)
    assert e.value.status == -1
    compact_kv([], 0, both.sequence(1))
    compact_kv([], 0, AcceptResult(both.next_tokens[:1], both.result[:1], 3))
    cache = PagedKVCache(PagedKVConfig(page_size=4, max_pages=4, num_layers=1, num_heads=1, head_dim=8, device="cpu"))
    cache.allocate_sequence(0, 8)
    for path in (None, [0, 2]):
        with pytest.raises(SpecVerifyError) as e:
            cache.compact_path(0, 2, both, path=path)
        assert e.value.status == -1


def test_add_rms_norm_refuses_rows_that_its_column_index_does_not_hold(lib):
    """A thread steps over a wide row 4096 columns at a time in 32 bits: behind 2^31 - 4096 the index would turn negative."""
    for cols in (2 ** 31 - 1, 2 ** 31 - 4096, 2 ** 30 + 1):
        for y_scale in (None, FAKE):
            assert lib.tv_add_rms_norm(FAKE, cols, FAKE, cols, FAKE, FAKE, cols, FAKE, cols, y_scale, 0, cols, 1e-5, 0,
                                       None) == -7
    assert lib.tv_add_rms_norm(FAKE, 8, FAKE, 8, FAKE, FAKE, 8, FAKE, 8, None, 0, 2 ** 30, 1e-5, 0, None) == 0


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")
def test_compaction_of_each_sequence_of_a_batch():
    from specverify.core.kv_cache.paged_kv import PagedKVCache, PagedKVConfig
    from specverify.draft import accept_residual, compact_kv
    from specverify.draft.tree_verification import AcceptResult
    logits = torch.full((2, 4, 50), -30.0, device="cuda")
    logits[0, 0, 7] = logits[0, 2, 9] = logits[1, 0, 8] = logits[1, 1, 3] = 30.0
    draft = torch.tensor([[0, 1, 7, 9], [0, 8, 5, 3]], device="cuda")
    parent = torch.tensor([[-1, -1, 1], [-1, -1, 0]], device="cuda")
    acc = accept_residual(logits, draft, parent, torch.full((2, 4), 0.5, device="cuda"))
    paths = [h["path"] for h in acc.to_host()]
    assert paths == [[0, 2, 3], [0, 1, 3]]
    kv = torch.randn(2, 3, 20, 64, device="cuda").bfloat16()            # [batch, heads, rows, head_dim]
    want = kv.clone()
    for b, path in enumerate(paths):
        want[b, :, 10:13] = kv[b][:, [10 + i for i in path]]
    for b in range(2):
        compact_kv([kv[b]], 10, acc.sequence(b))
    assert torch.equal(kv, want)
    # a batch of one is one sequence, in the paged cache too
    one = AcceptResult(acc.next_tokens[1:], acc.result[1:], 4)
    caches = []
    for a, path in ((one, None), (acc.sequence(1), paths[1])):
        cache = PagedKVCache(PagedKVConfig(page_size=4, max_pages=8, num_layers=1, num_heads=1, head_dim=64,
                                           dtype=torch.bfloat16, device="cuda"))
        cache.allocate_sequence(0, 16)
        cache.page_pool.copy_(torch.randn(cache.page_pool.shape, generator=torch.Generator().manual_seed(1)))
        assert cache.compact_path(0, 10, a, path=path) == 13
        caches.append(cache.page_pool)
    assert torch.equal(*caches)
