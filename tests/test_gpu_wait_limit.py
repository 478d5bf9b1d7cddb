"""What a 4-bit product's bounded waits leave behind when one runs out: the
helpers of its kernel in one whose barriers nothing completes, the status word
of the public call, and the decode loop's reading of it."""

from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from conftest import ROOT, cuda_ok

gpu = [pytest.mark.gpu, pytest.mark.skipif(not cuda_ok(), reason="needs a CUDA device")]


@pytest.fixture(scope="module")
def waits(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(nvcc).exists():
        pytest.skip("no nvcc")
    lib = tmp_path_factory.mktemp("waits") / "waits.so"
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-shared", "-Xcompiler", "-fPIC",
                    f"-I{ROOT / 'specdiff-ae_b200' / 'csrc'}", f"-I{ROOT / 'include'}",
                    str(Path(__file__).with_name("wait_limit.cu")), "-o", str(lib)], check=True)
    fn = ctypes.CDLL(str(lib)).run_wait_limit
    fn.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_longlong, ctypes.c_void_p]
    return fn


def test_builds(waits):
    assert waits is not None


@pytest.mark.parametrize("with_status", [True, False])
@pytest.mark.usefixtures("waits")
class TestWaits:
    pytestmark = gpu

    def test_a_wait_that_runs_out_is_reported(self, waits, with_status):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = torch.full((3,), -1, dtype=torch.int32, device="cuda")
        rc = waits(status.data_ptr() if with_status else None, out.data_ptr(), 1 << 20,
                   torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert rc == 0 and out.tolist() == [0, 0, 1]            # both gave up; the completed barrier's did not
        assert status.item() == (3 if with_status else 0)       # the first code stays
        assert float(torch.ones(4, device="cuda").sum()) == 4   # the context goes on


class TestStatus:
    pytestmark = gpu

    @pytest.mark.parametrize("rows", [1, 40, 200])
    def test_calls_that_complete_leave_it(self, rows):
        from specverify import SpecVerifyError
        from specverify.runtime import w4_linear
        from test_gpu_w4 import check, problem, to_fp8
        x, q, s = problem(rows, 300, 1024, 128, torch.bfloat16)
        for start in (0, 5):
            status = torch.full((1,), start, dtype=torch.int32, device="cuda")
            check(w4_linear(x, q, s, status=status), x, q, s)
            x8, xs = to_fp8(x)
            check(w4_linear(x8, q, s, x_scale=xs, status=status), x8, q, s, xs)
            assert status.item() == start
        for bad in (torch.zeros(1, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"),
                    torch.zeros(1, dtype=torch.int32)):
            with pytest.raises(SpecVerifyError):
                w4_linear(x, q, s, status=bad)

    def test_the_decode_loop_reads_it(self, monkeypatch):
        from specverify import SpecVerifyError
        from specverify.draft import spec_decode
        from test_gpu_spec_decode_w4 import PROMPT, _model
        args = dict(max_new_tokens=4, nodes=8, max_depth=4, temperature=1.0, seed=0, max_steps=2)
        product = spec_decode.w4_linear

        def gives_up(x, *w, status, **kw):
            status.fill_(2)
            return product(x, *w, status=status, **kw)

        monkeypatch.setattr(spec_decode, "w4_linear", gives_up)
        m = _model()
        with pytest.raises(SpecVerifyError, match="code 2"):
            m.diffspec_generate(PROMPT, **args)
        monkeypatch.setattr(spec_decode, "w4_linear", product)
        m = _model()
        m.status.fill_(3)                    # an earlier run's
        assert m.diffspec_generate(PROMPT, **args)["steps"] >= 1
