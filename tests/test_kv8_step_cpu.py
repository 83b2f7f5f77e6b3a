"""What decode_step and the prompts' epilogue refuse over an 8-bit cache, before they have appended anything.  CPU only."""
import pytest
import torch

from mllm_b200 import runtime as rt


@pytest.mark.parametrize("bad", [dict(H=18), dict(Hkv=1), dict(Hkv=4, H=8), dict(kv=4), dict(B=4), dict(D=128), dict(pos=[1, 2]),
                                 dict(rows=2)])
@pytest.mark.parametrize("cls,prefix", [("PagedKVCache8", 0), ("PagedKVCache8", 100), ("PagedKVCache", 100)])
def test_refused_before_anything_changes(cls, prefix, bad, monkeypatch):
    monkeypatch.setattr(rt, "_check_cuda_bf16", lambda *a: None)
    monkeypatch.setattr(rt, "_capturing", lambda: False)
    for name in ("_epilogue_kv8_batch", "_launch"):
        monkeypatch.setattr(rt, name, lambda *a: pytest.fail("launched"))
    monkeypatch.setattr(rt.abi, "call", lambda *a: pytest.fail("launched"))
    c = getattr(rt, cls)(9, 2, 64, block_size=128, max_seqs=3, device="cpu")
    c.shared_prefix = prefix
    c.set_lengths([128])
    c.fork(0, 1, 128)
    c.fork(0, 2, 128)
    free = c.free_blocks
    a = {**dict(B=3, H=8, Hkv=2, D=64, kv=2, pos=[128]), **bad}
    q, kv = (torch.zeros(a["B"], h, 1, a["D"], dtype=torch.bfloat16) for h in (a["H"], a["kv"]))
    table = (torch.zeros(a["rows"], a["D"]),) * 2 if "rows" in a else None
    with pytest.raises(RuntimeError):
        rt.decode_step(q, kv, kv, c, torch.tensor(a["pos"]), 1e4, a["Hkv"], rope_table=table)
    assert c.host_lengths() == [128] * 3 and c.lengths.tolist() == [128] * 3 and c.free_blocks == free


@pytest.mark.parametrize("bad", [dict(kv=4), dict(D=128), dict(norm=(64, 32)), dict(pos=[0, 1, 2, 3])])
def test_packed_prompts_refused_before_the_lengths_advance(bad, monkeypatch):
    monkeypatch.setattr(rt, "_check_cuda_bf16", lambda *a: None)
    monkeypatch.setattr(rt, "_launch", lambda *a: pytest.fail("launched"))
    c = rt.PagedKVCache8(9, 2, 64, block_size=128, max_seqs=3, device="cpu")
    c.set_lengths([5, 6, 7])
    a = {**dict(kv=2, D=64, norm=None), **bad}
    q, kv = (torch.zeros(5, h, a["D"], dtype=torch.bfloat16) for h in (8, a["kv"]))
    norm = [torch.ones(n) for n in a["norm"]] if a["norm"] else [None, None]
    pos = torch.tensor(a["pos"]) if "pos" in a else None                  # four positions for five tokens
    with pytest.raises(RuntimeError):
        rt.qkv_epilogue_packed(q, kv, kv, c, [3, 2], 1e4, positions=pos, q_norm_weight=norm[0], k_norm_weight=norm[1])
    assert c.host_lengths() == [5, 6, 7] and c.lengths.tolist() == [5, 6, 7]
