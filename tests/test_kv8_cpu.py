"""The 8-bit KV cache's host side: bookkeeping, layout, and what the calls refuse.  CPU only."""
import ctypes as C

import pytest
import torch

from mllm_b200 import abi, build
from mllm_b200 import runtime as rt


@pytest.fixture(scope="module")
def lib():
    build.build()
    return abi.load()


def test_blocks_and_slots_like_the_bf16_cache():
    c = rt.PagedKVCache8(6, 2, 64, block_size=128, max_seqs=4, max_blocks_per_seq=3, device="cpu")
    assert c.k_pool.shape == (6, 2, 128, 64) and c.k_exp.shape == (6, 2, 128) and c.k_pool.dtype == rt.FP8
    c.set_lengths([200, 5])
    s = c.slot(2, 2)
    assert isinstance(s, rt.PagedKVCache8)
    s.reserve(0, 300)
    assert c.blocks_of(2) == s.blocks_of(0) and c.free_blocks == 0
    c.k_exp.fill_(9)
    c.k_pool.view(torch.uint8).fill_(9)
    blocks = c.blocks_of(0)
    c.release(0)
    assert (c.k_exp[blocks] == 0).all() and (c.k_pool.view(torch.uint8)[blocks] == 0).all()
    assert (c.k_exp[c.blocks_of(2)] == 9).all()
    c.move(2, 0)
    assert c.blocks_of(2) == [] and len(c.blocks_of(0)) == 3
    d = c.descriptor()
    assert (d.block_stride, d.head_stride, d.row_stride) == (2 * 128 * 64, 128 * 64, 64)
    assert (d.exp_block_stride, d.exp_head_stride, d.num_blocks, d.block_size) == (256, 128, 6, 128)


def test_gather_gives_value_times_scale():
    c = rt.PagedKVCache8(2, 1, 64, block_size=128, max_seqs=1, device="cpu")
    c.set_lengths([130])
    c.k_pool[c.blocks_of(0)[1], 0, 1] = torch.full((64,), 1.75).to(rt.FP8)
    c.k_exp[c.blocks_of(0)[1], 0, 1] = 127 - 3
    k, v = c.gather(0, 130)
    assert (k[0, 129] == 1.75 / 8).all() and (k[0, :129] == 0).all() and (v == 0).all()


def _desc(**over):
    d = dict(k_pool=4096, v_pool=4096, block_stride=2 * 128 * 128, head_stride=128 * 128, row_stride=128, k_exp=4096,
             v_exp=4096, exp_block_stride=256, exp_head_stride=128, num_blocks=4, block_size=128, block_table=4096,
             table_stride=4, max_blocks_per_seq=4)
    d.update(over)
    return abi.PagedKV8(**d)


BAD_DESCRIPTORS = [
    (dict(k_pool=None), b"pools"), (dict(v_exp=None), b"pools"), (dict(block_table=None), b"pools"),
    (dict(block_size=100), b"128"), (dict(block_size=0), b"128"), (dict(num_blocks=0), b"num_blocks"),
    (dict(table_stride=3), b"table_stride"), (dict(row_stride=120), b"strides"), (dict(head_stride=128 * 128 + 8), b"strides"),
    (dict(exp_head_stride=8), b"exponent"), (dict(exp_block_stride=250), b"exponent"), (dict(k_pool=4100), b"aligned"),
    (dict(v_exp=4097), b"aligned"),
]


def _decode(lib, kv, B=1, H=8, Hkv=2, D=128, L=300, scale=0.1, q=4096, lens=4096, ws=4096, ws_bytes=1 << 30):
    return lib.mllm_decode_attention_paged_kv8(q, C.byref(kv) if kv else None, lens, B, H, Hkv, D, L, scale, 4096, ws,
                                               ws_bytes, None)


def _read(lib, kv, n=1, Hkv=2, D=128, rows=10, out=4096, strides=(2560, 1280, 128)):
    return lib.mllm_kv8_read_bf16(C.byref(kv) if kv else None, None, 4096, n, Hkv, D, rows, out, out, *strides, None)


def _append(lib, kv, T=4, H=8, Hkv=2, D=128, pos=4096, theta=1e4, cos=None, sin=None, qn=None, kn=None, q=4096, out=4096,
            o_st=1024, cu=4096, n=1, start=4096):
    return lib.mllm_qkv_epilogue_varlen_paged_kv8(q, 1536, 128, 4096, 1536, 128, 4096, 1536, 128, T, H, Hkv, D, pos, theta,
                                                  cos, sin, qn, kn, 1e-6, out, o_st, 128,
                                                  C.byref(kv) if kv else None, cu, n, start, None)


@pytest.mark.parametrize("over,text", BAD_DESCRIPTORS)
def test_bad_descriptors_are_refused(lib, over, text):
    for call in (_decode, _read, _append):
        assert call(lib, _desc(**over)) == 1
        assert text in lib.mllm_attn_last_error()


def test_bad_arguments_are_refused(lib):
    kv = _desc()
    for call in (_decode, _read, _append):
        assert call(lib, None) == 1 and b"NULL" in lib.mllm_attn_last_error()
        assert call(lib, kv, D=96) == 2
    assert _decode(lib, kv, H=7) == 1 and b"divisible" in lib.mllm_attn_last_error()
    assert _decode(lib, kv, H=18) == 2 and b"larger than 8" in lib.mllm_attn_last_error()
    assert _decode(lib, kv, L=513) == 1 and b"rows exceed" in lib.mllm_attn_last_error()
    assert _decode(lib, kv, L=0) == 1 and _decode(lib, kv, B=-1) == 1
    assert _decode(lib, kv, scale=0.0) == 1 and _decode(lib, kv, scale=float("nan")) == 1
    assert _decode(lib, kv, q=None) == 1 and _decode(lib, kv, lens=None) == 1
    assert _decode(lib, kv, q=4100) == 1 and b"misaligned" in lib.mllm_attn_last_error()
    assert _decode(lib, kv, ws=None) == 4 and _decode(lib, kv, ws=4097) == 4 and _decode(lib, kv, ws_bytes=100) == 4
    assert _decode(lib, kv, B=0) == 0
    assert _read(lib, kv, rows=-1) == 1 and _read(lib, kv, out=None) == 1
    assert _read(lib, kv, strides=(2560, 1280, 129)) == 1 and _read(lib, kv, strides=(2560, 1280, 64)) == 1
    assert _read(lib, kv, n=40000) == 2
    assert _read(lib, kv, rows=0) == 0 and _read(lib, kv, n=0) == 0
    assert _append(lib, kv, H=7) == 1 and _append(lib, kv, T=-1) == 1
    assert _append(lib, kv, pos=None) == 1 and b"positions" in lib.mllm_attn_last_error()
    assert _append(lib, kv, theta=0.0) == 1 and _append(lib, kv, cos=4096) == 1 and _append(lib, kv, qn=4096) == 1
    assert _append(lib, kv, q=None) == 1 and _append(lib, kv, cu=None) == 1 and _append(lib, kv, start=None) == 1
    assert _append(lib, kv, out=4100) == 1 and _append(lib, kv, o_st=1022) == 1
    assert _append(lib, kv, T=0) == 0 and _append(lib, kv, n=0) == 0


def test_workspace_does_not_depend_on_lengths(lib):
    size = lib.mllm_decode_attention_kv8_workspace_size
    assert size(1, 32, 8, 128) >= 2 * 2 * 148 * 4 * (128 + 1) * 4 and size(64, 32, 8, 128) % 256 == 0
    assert size(4, 8, 3, 128) == 0 and size(4, 0, 8, 128) == 0 and size(0, 32, 8, 128) == 0


def test_python_checks():
    c = rt.PagedKVCache8(2, 1, 64, block_size=128, max_seqs=1, device="cpu")
    x = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        rt.qkv_epilogue_kv8(x, x, x, c, i, i)
    with pytest.raises(RuntimeError, match="PagedKVCache8"):
        rt.kv8_read(rt.PagedKVCache(1, 1, 64, 128, 1, device="cpu"), i, 3)
    with pytest.raises(RuntimeError, match="negative rows"):
        rt.kv8_read(c, i, -1)
    with pytest.raises(RuntimeError, match="lens"):
        rt.kv8_read(c, i.long(), 3)


def test_a_launch_for_another_device_makes_it_current_around_the_call(monkeypatch):
    current = [0]
    seen = []

    class Device:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            self.before, current[0] = current[0], self.dev

        def __exit__(self, *exc):
            current[0] = self.before
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda dev: 100 + dev, raising=False)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(rt.abi, "stream_handle", lambda: 100 + current[0])
    monkeypatch.setattr(rt.abi, "call", lambda name, *args: seen.append((current[0], name, args)))
    rt._launch(0, "f", 1)
    rt._launch(3, "g", 2)
    assert seen == [(0, "f", (1, 100)), (3, "g", (2, 103))] and current == [0]
