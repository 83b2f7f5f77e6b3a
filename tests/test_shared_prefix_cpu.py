"""Sharing blocks between sequences, and what the shared-prefix decode refuses.  CPU only."""
import ctypes as C

import pytest
import torch

from mllm_b200 import abi, build
from mllm_b200 import runtime as rt


@pytest.mark.parametrize("cls", ["PagedKVCache", "PagedKVCache8"])
def test_fork_shares_full_blocks_and_copies_the_last(cls):
    c = getattr(rt, cls)(8, 1, 64, block_size=128, max_seqs=4, device="cpu")
    c.set_lengths([300])
    raw = c.k_pool.view(torch.uint8) if cls.endswith("8") else c.k_pool
    for i, blk in enumerate(c.blocks_of(0)):
        raw[blk] = i + 1
    c.fork(0, 1, 300)
    c.fork(0, 2, 256)
    a, b, d = (c.blocks_of(i) for i in range(3))
    assert b[:2] == a[:2] and b[2] != a[2] and d == a[:2]
    assert (raw[b[2], :, :44] == 3).all() and (raw[b[2], :, 44:] == 0).all()
    assert c.host_lengths()[:3] == [300, 300, 256] and c.lengths[:3].tolist() == [300, 300, 256]
    assert c.block_table[1, :3].tolist() == b and c.free_blocks == 4
    c.advance([1, 1, 1], batch=3)                       # appends go to blocks of the sequence's own
    assert len(c.blocks_of(2)) == 3 and len(set(c.blocks_of(2)) & set(a + b)) == 2
    c.release(0)                                        # the shared blocks stay, with their rows
    assert c.free_blocks == 4 and (raw[b[0]] == 1).all() and (raw[a[2]] == 0).all()
    c.move(1, 0)
    c.release(0)
    assert c.free_blocks == 5 and (raw[d[0]] == 1).all()
    c.release(2)
    assert c.free_blocks == 8 and (raw == 0).all()
    assert sorted(c._free) == list(range(8))


def test_fork_refusals():
    c = rt.PagedKVCache(3, 1, 64, block_size=128, max_seqs=4, device="cpu")
    c.set_lengths([200, 5])
    for src, dst, rows in ((0, 1, 100), (0, 0, 100), (0, 2, 257), (0, 2, -1), (3, 2, 1)):
        with pytest.raises(RuntimeError, match="fork"):
            c.fork(src, dst, rows)
    with pytest.raises(RuntimeError, match="out of blocks"):
        c.fork(0, 2, 200)
    assert c.free_blocks == 0 and c.blocks_of(2) == [] and c.host_lengths() == [200, 5, 0, 0]
    c.fork(0, 2, 128)
    c.slot(2, 2).fork(0, 1, 128)
    assert c.blocks_of(3) == c.blocks_of(0)[:1]


def test_library_refusals():
    build.build()
    lib = abi.load()
    size = lib.mllm_decode_attention_shared_workspace_size

    def call(B=2, H=8, Hkv=2, D=128, P=100, L=300, scale=0.1, q=4096, lens=4096, ws=4096, nb=1 << 40, **over):
        d = dict(k_pool=4096, v_pool=4096, block_stride=2 * 128 * 128, head_stride=128 * 128, row_stride=128,
                 num_blocks=4, block_size=128, block_table=4096, table_stride=4, max_blocks_per_seq=4)
        d.update(over)
        return lib.mllm_decode_attention_shared_paged_bf16(q, C.byref(abi.PagedKV(**d)), lens, P, B, H, Hkv, D, L, scale,
                                                           4096, ws, nb, None)
    assert call(P=-1) == 1 and call(P=301) == 1 and b"prefix_len" in lib.mllm_attn_last_error()
    assert call(H=7) == 1 and call(D=96) == 2 and call(H=18) == 2 and call(L=513, P=10) == 1
    assert call(scale=-1.0) == 1 and call(q=None) == 1 and call(lens=None) == 1
    assert call(q=4104) == 1 and b"misaligned" in lib.mllm_attn_last_error()
    assert call(k_pool=None) == 1 and call(block_size=64) == 1 and call(B=70000) == 2
    long = dict(max_blocks_per_seq=1 << 24, table_stride=1 << 24, L=0x7fffff01)
    assert call(**long) == 2 and b"max_kv_len" in lib.mllm_attn_last_error() and call(**{**long, "L": 1 << 30}, ws=None) == 4
    assert call(ws=None) == 4 and call(ws=4104) == 4
    assert call(nb=size(2, 8, 2, 128, 100) - 1) == 4
    assert call(B=0) == 0
    assert size(2, 8, 2, 128, -1) == 0 and size(2, 7, 2, 128, 5) == 0
    assert size(2, 8, 2, 128, 0) < size(2, 8, 2, 128, 1) <= size(2, 8, 2, 128, 5000)


def test_library_refusals_of_an_8bit_cache():
    build.build()
    lib = abi.load()
    size = lib.mllm_decode_attention_shared_workspace_size

    def call(B=2, H=8, Hkv=2, D=128, P=100, L=300, scale=0.1, q=4096, lens=4096, ws=4096, nb=1 << 40, **over):
        d = dict(k_pool=4096, v_pool=4096, block_stride=2 * 128 * 128, head_stride=128 * 128, row_stride=128, k_exp=4096,
                 v_exp=4096, exp_block_stride=256, exp_head_stride=128, num_blocks=4, block_size=128, block_table=4096,
                 table_stride=4, max_blocks_per_seq=4)
        d.update(over)
        return lib.mllm_decode_attention_shared_paged_kv8(q, C.byref(abi.PagedKV8(**d)), lens, P, B, H, Hkv, D, L, scale,
                                                          4096, ws, nb, None)
    assert call(P=-1) == 1 and call(P=301) == 1 and b"prefix_len" in lib.mllm_attn_last_error()
    assert call(H=7) == 1 and call(D=96) == 2 and call(H=18) == 2 and call(L=513, P=10) == 1
    assert call(scale=-1.0) == 1 and call(q=None) == 1 and call(lens=None) == 1 and call(q=4104) == 1
    assert call(k_exp=None) == 1 and call(k_pool=4104) == 1 and call(row_stride=130) == 1 and call(exp_head_stride=8) == 1
    assert call(block_size=64) == 1 and call(B=70000) == 2
    assert call(ws=None) == 4 and call(ws=4104) == 4 and call(nb=size(2, 8, 2, 128, 100) - 1) == 4
    assert call(B=0) == 0


def test_when_reading_the_prefix_once_pays():
    pays = rt._shared_pays
    for kv8 in (False, True):
        assert not pays(1, 1 << 20, 8, 128, kv8) and not pays(32, 0, 8, 128, kv8) and not pays(32, 128, 8, 128, kv8)
        assert pays(32, 8192, 8, 128, kv8) and pays(64, 32768, 8, 128, kv8)
    assert pays(3, 8192, 8, 128) and not pays(3, 8192, 8, 128, True) and not pays(4, 32768, 8, 128, True)
