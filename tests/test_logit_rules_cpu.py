"""What the logit rules refuse.  CPU only."""
import pytest
import torch

from mllm_b200 import abi, build
from mllm_b200 import runtime as rt


@pytest.fixture(scope="module")
def lib():
    build.build()
    return abi.load()


def _call(lib, logits=4096, bf16=0, stride=1000, B=2, V=1000, hist=None, hist_stride=0, cols=0, lens=None, start=None,
          rep=None, pres=None, freq=None, ids=None, vals=None, b_stride=0, b_cols=0, b_lens=None, allowed=None, a_stride=0,
          out=4096, out_stride=1000):
    return lib.mllm_logit_rules(logits, bf16, stride, B, V, hist, hist_stride, cols, lens, start, rep, pres, freq, ids, vals,
                                b_stride, b_cols, b_lens, allowed, a_stride, out, out_stride, None)


def test_library_refusals(lib):
    assert _call(lib, V=0) == 1 and _call(lib, B=-1) == 1 and _call(lib, B=70000) == 2
    assert _call(lib, stride=999) == 1 and _call(lib, out_stride=999) == 1
    assert _call(lib, hist=4096) == 1 and _call(lib, lens=4096) == 1
    assert _call(lib, hist=4096, lens=4096, cols=5, hist_stride=4) == 1 and _call(lib, hist=4096, lens=4096, cols=-1) == 1
    for name in ("rep", "pres", "freq", "start"):
        assert _call(lib, **{name: 4096}) == 1 and b"history" in lib.mllm_attn_last_error()
    assert _call(lib, ids=4096) == 1 and _call(lib, ids=4096, vals=4096) == 1
    assert _call(lib, ids=4096, vals=4096, b_lens=4096, b_cols=9, b_stride=8) == 1
    assert _call(lib, ids=4096, vals=4096, b_lens=4096, b_cols=1025, b_stride=1025) == 2
    assert _call(lib, allowed=4096, a_stride=31) == 1 and b"allowed_stride" in lib.mllm_attn_last_error()
    assert _call(lib, logits=None) == 1 and _call(lib, out=None) == 1
    assert _call(lib, logits=4098) == 1 and _call(lib, bf16=1, out=4097) == 1
    assert _call(lib, B=0) == 0


def test_library_refuses_long_histories_and_misaligned_lists(lib):
    full = dict(hist=4096, lens=4096, cols=5, hist_stride=5, ids=4096, vals=4096, b_lens=4096, b_cols=5, b_stride=5)
    assert _call(lib, **{**full, "cols": 1 << 30, "hist_stride": 1 << 30}) == 2
    for name, at in (("hist", 4100), ("lens", 4098), ("ids", 4100), ("vals", 4097), ("b_lens", 4098), ("rep", 4098),
                     ("pres", 4098), ("freq", 4098), ("start", 4098)):
        assert _call(lib, **{**full, name: at}) == 1 and b"misaligned" in lib.mllm_attn_last_error()


def test_python_refuses_host_tensors():
    with pytest.raises(RuntimeError, match="CUDA"):
        rt.apply_logit_rules(torch.zeros(1, 5))
