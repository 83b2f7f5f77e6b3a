"""Logits and output in overlapping memory: other rows than the logits' own are refused.  CPU only."""
import pytest

from mllm_b200 import abi, build


@pytest.mark.parametrize("bf16", [0, 1])
def test_overlapping_rows_are_refused(bf16):
    build.build()
    lib = abi.load()
    es, V = (2 if bf16 else 4), 100

    def refused(at, stride=V, out_stride=V, B=3):
        """With out `at` elements behind the logits."""
        st = lib.mllm_logit_rules(1 << 20, bf16, stride, B, V, None, 0, 0, None, None, None, None, None, None, None, 0, 0,
                                  None, None, 0, (1 << 20) + at * es, out_stride, None)
        return st == 1 and b"overlaps" in lib.mllm_attn_last_error()
    assert not refused(0) and not refused(0, stride=150, out_stride=150)                  # in place
    assert refused(1) and refused(-1) and refused(V) and refused(-V) and refused(2 * V) and refused(3 * V - 1)
    assert not refused(3 * V) and not refused(-3 * V)                                     # behind, in front
    assert not refused(V, 200, 200) and not refused(-V, 200, 200)                         # side by side in one tensor
    assert refused(V - 1, 200, 200) and refused(V + 1, 200, 200) and refused(-V - 1, 200, 200)
    assert refused(0, 100, 150) and refused(0, 150, 100) and refused(-120, 150, 100)      # the same begin, other strides
    assert not refused(0, 100, 150, B=1) and refused(1, B=1) and not refused(V, B=1) and not refused(-V, B=1)
    assert not refused(100, 300, 400, B=2) and refused(100, 300, 250, B=2)
