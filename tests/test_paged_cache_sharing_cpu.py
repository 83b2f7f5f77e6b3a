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


@pytest.mark.parametrize("cls", ["PagedKVCache", "PagedKVCache8"])
def test_which_sequences_came_by_their_rows_together(cls):
    """Through forks of forks, moves, releases and shortened sequences; what is not known to be equal is not."""
    c = getattr(rt, cls)(40, 1, 64, block_size=128, max_seqs=6, device="cpu")
    common = c._rows_in_common
    c.set_lengths([300, 300])
    assert common(1, 300) and not common(2, 1)
    c.release(1)
    c.fork(0, 1, 300)
    c.fork(1, 2, 280)
    c.fork(0, 3, 290)
    c.advance([5, 6, 7, 8], batch=4)
    assert common(2, 300) and not common(2, 301) and common(3, 280) and not common(3, 281) and common(4, 280)
    assert not common(5, 1) and c.slot(1, 3)._rows_in_common(3, 280) and not c.slot(3, 2)._rows_in_common(2, 1)
    c.fork(3, 4, 295)                                    # rows 290 .. of sequence 3 are its own
    assert common(2, 290, first=3) and common(2, 295, first=3) and not common(2, 296, first=3) and common(5, 280)
    c.release(0)
    c.move(4, 0)
    assert common(4, 280) and not common(4, 281) and not common(5, 1)
    c.set_lengths([295, 299, 287, 298])                  # sequence 1 shortened below row 300, where its copy begins at 256
    c.set_lengths([299, 305, 287, 298])
    assert common(2, 290) and not common(2, 291)
    c.set_lengths([270])                                 # and sequence 0 further back
    c.set_lengths([300])
    assert common(4, 270) and not common(4, 271)
    for _ in range(50):                                  # nothing is kept for each time
        c.set_lengths([260])
        c.set_lengths([300])
    assert common(4, 260) and not common(4, 261) and all(len(x) < 6 for x in c._lines)
    c.release(2)
    assert not common(4, 1)
    c.fork(3, 2, 0)
    assert not common(4, 1)


@pytest.mark.parametrize("cls", ["PagedKVCache", "PagedKVCache8"])
def test_a_step_reads_the_prefix_once_only_where_it_is_in_common(cls, monkeypatch):
    """A row that was not forked has rows of its own: the step reads each row's."""
    class Stop(Exception):
        pass

    def taken(name):
        def stop(*a, **kw):
            raise Stop(name)
        return stop
    monkeypatch.setattr(rt, "_check_cuda_bf16", lambda *a: None)
    monkeypatch.setattr(rt, "_capturing", lambda: False)
    monkeypatch.setattr(rt, "_epilogue_kv8_batch", lambda *a: None)
    monkeypatch.setattr(rt, "_decode_step_shared", taken("shared"))
    monkeypatch.setattr(rt, "decode_attention_shared", taken("shared"))
    monkeypatch.setattr(rt, "_decode_kv8", taken("own"))
    monkeypatch.setattr(rt.abi, "call", taken("own"))
    monkeypatch.setattr(rt.abi, "stream_handle", lambda: None)
    monkeypatch.setattr(rt, "_SHARED_MIN_BYTES", 0)
    monkeypatch.setattr(rt, "_SHARED_MIN_BYTES8", 0)
    monkeypatch.setattr(rt, "_SHARED_MIN_BATCH8", 1)
    for forked in (True, False):
        c = getattr(rt, cls)(20, 2, 64, block_size=128, max_seqs=3, device="cpu")
        c.shared_prefix = 200
        c.set_lengths([200])
        c.fork(0, 1, 200)
        if forked:
            c.fork(0, 2, 200)
        else:
            c.set_lengths([200, 200, 200])
        q, kv = (torch.zeros(3, h, 1, 64, dtype=torch.bfloat16) for h in (4, 2))
        with pytest.raises(Stop, match="shared" if forked else "own"):
            rt.decode_step(q, kv, kv, c, torch.tensor([200]), 1e4, 2)


def test_reserved_rows_are_in_common_in_full_blocks_only():
    """What is written behind the fork reaches shared blocks, not the copy of the last one."""
    c = rt.PagedKVCache(9, 1, 64, block_size=128, max_seqs=3, device="cpu")
    c.reserve(0, 300)
    c.fork(0, 1, 300)
    c.fork(1, 2, 100)                                    # sequence 1 has 300 rows: what it copies is there
    assert c._rows_in_common(2, 256) and not c._rows_in_common(2, 257)
    assert c._rows_in_common(2, 100, first=1) and c._rows_in_common(3, 100) and not c._rows_in_common(3, 101)
