"""What a sequence may do with rows that others share (PagedKVCache.fork).  CPU only."""
import pytest
import torch

from mllm_b200 import runtime as rt


@pytest.mark.parametrize("cls", ["PagedKVCache", "PagedKVCache8"])
@pytest.mark.parametrize("through_slot", [False, True])
def test_no_sequence_is_shortened_into_a_shared_block(cls, through_slot):
    """Its next append would write the others' rows; the lengths stay as they were."""
    c = getattr(rt, cls)(12, 1, 64, block_size=128, max_seqs=3, device="cpu")
    c.set_lengths([300])
    c.fork(0, 1, 300)
    c.fork(0, 2, 256)
    c.set_lengths([310, 400, 260])
    v = c.slot(0, 3) if through_slot else c
    for lens in ([255, 400, 260], [310, 0, 260], [310, 400, 128], [311, 401, 255]):
        with pytest.raises(RuntimeError, match="share"):
            v.set_lengths(lens)
        with pytest.raises(RuntimeError, match="share"):
            v.advance([n - m for n, m in zip(lens, [310, 400, 260])], batch=3)
        assert c.host_lengths() == [310, 400, 260] and c.lengths.tolist() == [310, 400, 260]
    v.set_lengths([256, 300, 256])              # blocks of their own: the copies, and those behind
    assert c.lengths.tolist() == [256, 300, 256]
    c.release(0)
    with pytest.raises(RuntimeError, match="share"):
        v.set_lengths([0, 300, 200])
    c.release(1)
    v.set_lengths([0, 0, 5])                    # the last owner does as it likes
    assert c.host_lengths() == [0, 0, 5] and c.free_blocks == 9
