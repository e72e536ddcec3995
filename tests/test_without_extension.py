"""The package where the extension module (_calls) is not there or does not fit: the library is built and loaded without
torch's headers, and prompt attention, which needs nothing else, still runs."""
import os
import subprocess
import sys

import pytest
import torch

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "turboquant-mlx_b200")


@pytest.fixture()
def bare(tq, monkeypatch):
    """The package as it is when importing _calls fails."""
    monkeypatch.setattr(tq._lib, "native", None)
    monkeypatch.setattr(tq._lib, "_native_absent", False, raising=False)
    monkeypatch.delattr(tq, "_calls", raising=False)
    monkeypatch.setitem(sys.modules, tq.__name__ + "._calls", None)
    return tq


def test_make_without_torch(tmp_path):
    """A Python without torch: make still builds the library and leaves the module out."""
    python = tmp_path / "python"
    python.write_text(f"#!/bin/sh\nexec {sys.executable} -S -E \"$@\"\n")
    python.chmod(0o755)
    assert subprocess.run([str(python), "-c", "import torch"], capture_output=True).returncode != 0
    r = subprocess.run(["make", "-n", "-B", "-C", PKG, f"PYTHON={python}"], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "-o " + os.path.join(PKG, "libtqb200.so") in r.stdout and "calls.cpp" not in r.stdout
    r = subprocess.run(["make", "-n", "-B", "-C", PKG, f"PYTHON={sys.executable}"], capture_output=True, text=True)
    assert r.returncode == 0 and "calls.cpp" in r.stdout


def test_paged_calls_say_what_is_missing(bare):
    with pytest.raises(RuntimeError, match="_calls.so"):
        bare.copy_pages([torch.zeros(4)], [0], [1])


def test_prompt_refusals(bare):
    x = torch.zeros((1, 2, 3, 128), dtype=torch.float16)
    with pytest.warns(UserWarning, match="_calls.so"), pytest.raises(RuntimeError, match="CUDA tensors only"):
        bare.prefill_attention(x, x, x, 1.0)


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore:_calls.so")
def test_prompt_attention(tq, dev, bare, monkeypatch):
    """The same bits and the same refusals as through the module."""
    q, k, v = [torch.randn((2, n, h, 128), device=dev, dtype=torch.bfloat16).transpose(1, 2) for n, h in ((70, 4), (300, 2), (300, 2))]
    odd = torch.randn((2 * 2 * 300 * 128 + 1,), device=dev).bfloat16()[1:].view(2, 2, 300, 128)       # not 16-byte aligned
    one = torch.randn((1, 1, 128), device=dev).bfloat16().as_strided((1, 1, 1, 128), (3, 5, 7, 1))
    out = torch.empty((2, 70, 4, 128), device=dev, dtype=torch.bfloat16).transpose(1, 2)
    calls = [lambda: bare.prefill_attention(q, k, v, 0.1), lambda: bare.prefill_attention(q, k, v, 0.1, causal=False),
             lambda: bare.prefill_attention(q, k, odd, 0.1, window=50, sinks=3), lambda: bare.prefill_attention(one, one, one, 0.1),
             lambda: bare.prefill_attention(q, k, v, 0.1, window=20, out=out).clone()]
    bad = [lambda: bare.prefill_attention(q.float(), k, v, 0.1), lambda: bare.prefill_attention(q, k.half(), v, 0.1),
           lambda: bare.prefill_attention(q[..., :64], k, v, 0.1), lambda: bare.prefill_attention(q[:, :3], k, v, 0.1),
           lambda: bare.prefill_attention(q, k, v[:, :, :299], 0.1), lambda: bare.prefill_attention(q, k[:1], v[:1], 0.1),
           lambda: bare.prefill_attention(q[0], k, v, 0.1), lambda: bare.prefill_attention(k.repeat(1, 2, 1, 1), q[:, :2], q[:, 2:], 0.1),
           lambda: bare.prefill_attention(q, k, v, 0.1, window=-1), lambda: bare.prefill_attention(q, k, v, 0.1, sinks=2),
           lambda: bare.prefill_attention(q, k, v, 0.1, window=4, causal=False), lambda: bare.prefill_attention(q, k, v, -1.0),
           lambda: bare.prefill_attention(q, k, v, 0.1, out=out.float()), lambda: bare.prefill_attention(q, k, v, 0.1, out=out[:, :3])]

    def run():
        for f in bad:
            with pytest.raises(ValueError):
                f()
        with pytest.raises(RuntimeError, match="CUDA"):
            bare.prefill_attention(q, k.cpu(), v, 0.1)
        return [f() for f in calls]

    assert bare._lib.native is None
    mine = run()
    assert bare._lib.native is None
    monkeypatch.undo()
    tq._lib.load_native()
    theirs = run()
    assert all(torch.equal(a, b) for a, b in zip(mine, theirs)) and tq.kernels.prefill_status(dev) == 0
