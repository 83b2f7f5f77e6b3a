"""Decode attention for a batch that shares a prefix, against 64-bit attention over each sequence's rows.  Needs a
B200.

Tolerance (from the formats): the output is rounded to bf16 (2^-8 of the value at most), P to bf16 (2^-8 of each
weight, so 2^-8 of the weighted mean of |v|), fp32 score sums 2^-18 of sum |q k|, twice, as weight error."""
import math
import random

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def rt(cuda_device):
    from mllm_b200 import build
    build.build()
    from mllm_b200 import runtime
    return runtime


def _status_ok():
    from mllm_b200 import abi
    abi.call("mllm_attn_device_status", None)


def _shared_cache(rt, prefix, suffix, Hkv, D, block, seed):
    """A cache of len(suffix) sequences forked from one prefix, rows random, finite numbers behind the ends."""
    B = len(suffix)
    lens = [prefix + s for s in suffix]
    per = -(-(prefix + max(suffix)) // block)
    c = rt.PagedKVCache(num_blocks=per * B + 3, num_kv_heads=Hkv, head_dim=D, block_size=block, max_seqs=B,
                        max_blocks_per_seq=per + 1)
    random.Random(seed).shuffle(c._free)
    g = torch.Generator(device="cuda").manual_seed(seed)
    c.k_pool.normal_(generator=g)
    c.v_pool.normal_(generator=g)
    c.reserve(0, prefix)
    for b in range(1, B):
        c.fork(0, b, prefix)
    c.set_lengths(lens)
    return c, lens


def _check(c, q, got, lens, Hkv):
    B, H, D = q.shape
    for b, L in enumerate(lens):
        o = got[b, 0].view(Hkv, H // Hkv, D).double()
        if L == 0:
            assert (o == 0).all()
            continue
        k, v = (x.double() for x in c.gather(b, L))
        qq = q[b].view(Hkv, H // Hkv, D).double()
        s = torch.einsum("grd,gtd->grt", qq, k) / math.sqrt(D)
        w = torch.softmax(s, -1)
        ref = torch.einsum("grt,gtd->grd", w, v)
        mean_abs = torch.einsum("grt,gtd->grd", w, v.abs())
        ds = 2.0 ** -18 * torch.einsum("grd,gtd->grt", qq.abs(), k.abs()).amax(-1, keepdim=True) / math.sqrt(D)
        tol = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2 * ds + 2.0 ** -18) * mean_abs
        assert ((o - ref).abs() <= tol).all(), (b, L, ((o - ref).abs() / tol).max())


CASES = [
    # H, Hkv, D, prefix, rows behind it, block, factor on q
    (8, 2, 128, 1, [1], 128, 1.0),
    (32, 8, 128, 127, [1, 2, 3], 128, 1.5),
    (32, 8, 128, 128, [0, 5, 64, 65], 128, 1.5),
    (32, 8, 128, 129, [0, 0], 256, 1.5),
    (32, 4, 64, 512, [1, 64, 17, 128, 0, 33, 2, 90], 128, 1.0),
    (32, 8, 128, 2000, [s % 200 for s in range(32)], 256, 1.5),        # one tile of query rows, full
    (32, 8, 128, 2000, [s % 7 for s in range(33)], 384, 1.5),          # a second tile with one sequence
    (40, 8, 128, 5000, [s * 3 for s in range(64)], 256, 1.0),          # groups of 5: three tiles, the pair not full
    (10, 2, 128, 700, [300] * 130, 128, 2.0),                          # two blocks of query rows
    (4, 4, 64, 300, [s % 3 for s in range(300)], 128, 1.0),            # groups of one
    (7, 1, 64, 40000, [9, 1], 128, 1.0),                               # many stretches
    (8, 1, 128, 1000, [1] * 40, 128, 300.0),                           # one weight close to 1
]


@pytest.mark.parametrize("H,Hkv,D,prefix,suffix,block,qf", CASES)
def test_against_64_bit_attention(rt, H, Hkv, D, prefix, suffix, block, qf):
    c, lens = _shared_cache(rt, prefix, suffix, Hkv, D, block, seed=3)
    g = torch.Generator(device="cuda").manual_seed(5)
    q = (qf * torch.randn(len(lens), H, D, device="cuda", generator=g)).bfloat16()
    got = rt.decode_attention_shared(q, c, Hkv, prefix)
    _status_ok()
    _check(c, q, got, lens, Hkv)
    assert torch.equal(got, rt.decode_attention_shared(q, c, Hkv, prefix, max_kv_len=c.capacity))


@pytest.mark.parametrize("H,Hkv,D,B", [(32, 8, 128, 13), (32, 8, 128, 40), (32, 4, 64, 9), (4, 4, 64, 1)])
def test_one_call_after_another_at_many_prefix_lengths(rt, H, Hkv, D, B):
    """Every number of tiles per stretch, odd and even, so that the two softmax groups of a CTA end at different times in
    both orders; calls follow one another without a wait between them, in memory that held NaN."""
    g = torch.Generator(device="cuda").manual_seed(21)
    q = (1.5 * torch.randn(B, H, D, device="cuda", generator=g)).bfloat16()
    for prefix in (200, 700, 1261, 1800, 2900, 4100, 6200, 8700, 10167, 13627):
        c, lens = _shared_cache(rt, prefix, [1 + s % 9 for s in range(B)], Hkv, D, 384, seed=prefix)
        held = torch.full((1 << 24,), float("nan"), device="cuda")   # what the workspaces lie in next
        del held
        got = [rt.decode_attention_shared(q, c, Hkv, prefix) for _ in range(10)]
        _status_ok()
        _check(c, q, got[0], lens, Hkv)
        for x in got[1:]:
            assert torch.equal(got[0], x)


def test_any_part_of_the_common_rows_gives_the_same_answer(rt):
    """The prefix length is the caller's choice: 0 .. all rows in common, inside tiles and blocks."""
    c, lens = _shared_cache(rt, 600, [1, 50, 200], 2, 128, 256, seed=7)
    q = torch.randn(3, 8, 128, device="cuda").bfloat16()
    for prefix in (0, 1, 63, 64, 65, 255, 256, 257, 511, 600):
        got = rt.decode_attention_shared(q, c, 2, prefix)
        _status_ok()
        _check(c, q, got, lens, 2)


def test_rows_behind_the_prefix_do_not_reach_other_sequences(rt):
    """What lies behind the prefix in its last block, and behind each sequence's end, may be anything."""
    c, lens = _shared_cache(rt, 200, [0, 30, 5], 2, 64, 128, seed=9)
    q = torch.randn(3, 8, 64, device="cuda").bfloat16()
    want = rt.decode_attention_shared(q, c, 2, 200)
    for b, L in enumerate(lens):
        blk = c.blocks_of(b)[L // 128]
        c.k_pool[blk, :, L % 128:] = float("nan")
        c.v_pool[blk, :, L % 128:] = float("inf")
    got = rt.decode_attention_shared(q, c, 2, 200)
    _status_ok()
    assert torch.equal(want, got)


def test_infinities_among_the_prefix_rows(rt):
    """An infinite V element in the tile where the prefix ends and the own rows begin counts once, as the prefix's."""
    c, lens = _shared_cache(rt, 200, [9, 0, 30, 5], 2, 64, 128, seed=9)
    q = torch.randn(4, 8, 64, device="cuda").bfloat16()
    want = rt.decode_attention_shared(q, c, 2, 200)
    for b in range(4):
        c.v_pool[c.blocks_of(b)[1], :, 195 % 128, 3] = float("inf")
    got = rt.decode_attention_shared(q, c, 2, 200).view(4, 8, 64)
    _status_ok()
    assert (got[..., 3] == float("inf")).all()
    got[..., 3] = want.view(4, 8, 64)[..., 3]
    assert torch.equal(got, want.view(4, 8, 64))


@pytest.mark.parametrize("B", [3, 40])
def test_tiles_whose_scores_are_all_minus_infinity(rt, B):
    """Of four tiles of 128 prefix rows three have scores of -inf only, and the others lie near -500 (log2): no tile
    may set a maximum that those underflow against."""
    prefix, Hkv, D = 40 * 128, 8, 128
    c, lens = _shared_cache(rt, prefix, [0] * B, Hkv, D, 128, seed=2)
    for t, blk in enumerate(c.blocks_of(0)):
        c.k_pool[blk, :, :, 0] = 0.0 if t % 4 == 2 else -float("inf")
        c.k_pool[blk, :, :, 1] = -500.0
    q = torch.zeros(B, 32, D, device="cuda", dtype=torch.bfloat16)
    q[..., 0], q[..., 1] = 1.0, 8.0
    got = rt.decode_attention_shared(q, c, Hkv, prefix)
    _status_ok()
    k, v = c.gather(0, prefix)
    rows = (k[0, :, 0] == 0).nonzero().flatten()
    ref = v[:, rows].double().mean(1)
    tol = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -17) * v[:, rows].double().abs().mean(1)
    o = got.view(B, Hkv, 4, D).double()
    assert ((o - ref[None, :, None]).abs() <= tol[None, :, None]).all()


def test_captured_and_replayed_with_other_lengths(rt):
    c, lens = _shared_cache(rt, 300, [1, 100, 40], 2, 128, 128, seed=4)
    for b in range(3):
        c.reserve(b, 500)
    q = torch.randn(3, 8, 128, device="cuda").bfloat16()
    graphs = []
    for _ in range(2):          # two graphs, replayed in turn, do not share their workspaces
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = rt.decode_attention_shared(q, c, 2, 300, max_kv_len=500)
        graphs.append((graph, out))
    for step in range(3):
        c.set_lengths([300 + 10 * step, 350 + step, 301])
        want = rt.decode_attention_shared(q, c, 2, 300)
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
    _status_ok()


def test_lengths_shorter_than_the_prefix(rt):
    from mllm_b200 import abi
    c, lens = _shared_cache(rt, 300, [10, 20, 30], 2, 128, 128, seed=4)
    q = torch.randn(3, 8, 128, device="cuda").bfloat16()
    c.lengths[1] = 0            # an empty row of a padded batch: zeros, no error
    got = rt.decode_attention_shared(q, c, 2, 300)
    _status_ok()
    _check(c, q, got, [310, 0, 330], 2)
    for bad in (299, -4, 331):
        c.lengths[1] = bad
        rt.decode_attention_shared(q, c, 2, 300)
        with pytest.raises(abi.MllmError) as e:
            _status_ok()
        assert e.value.status == 7


def test_refusals(rt):
    c, lens = _shared_cache(rt, 100, [1, 2], 2, 128, 128, seed=4)
    q = torch.randn(2, 8, 128, device="cuda").bfloat16()
    for bad in (-1, 103):
        with pytest.raises(RuntimeError, match="prefix_len|workspace"):
            rt.decode_attention_shared(q, c, 2, bad)
    with pytest.raises(RuntimeError, match="kv heads"):
        rt.decode_attention_shared(q, c, 4, 100)
    with pytest.raises(RuntimeError, match="PagedKVCache"):
        rt.decode_attention_shared(q, rt.KVCache(2, 2, 128, 16), 2, 0)
    with pytest.raises(RuntimeError, match="bfloat16"):
        rt.decode_attention_shared(q.float(), c, 2, 100)


def test_a_padded_batch_may_begin_with_empty_rows(rt):
    """Empty rows (length 0, tables full of anything) anywhere in the batch: zeros for them, the prefix from a row that
    has it; a batch of nothing but empty rows is all zeros."""
    c, lens = _shared_cache(rt, 300, [5, 6, 7, 8], 2, 128, 128, seed=4)
    q = torch.randn(4, 8, 128, device="cuda").bfloat16()
    keep = c.block_table.clone()
    for empty in ([0], [0, 1, 3], [2], [0, 1, 2, 3]):
        c.block_table.copy_(keep)
        c.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        for b in empty:
            c.lengths[b] = 0
            c.block_table[b] = -7
        got = rt.decode_attention_shared(q, c, 2, 300)
        _status_ok()
        _check(c, q, got, [0 if b in empty else n for b, n in enumerate(lens)], 2)


def test_on_side_streams_at_once(rt):
    """Two streams over one cache at the same time, each call with its own workspace."""
    c, lens = _shared_cache(rt, 3000, [100, 1, 700, 30], 8, 128, 256, seed=6)
    qs = [torch.randn(4, 32, 128, device="cuda").bfloat16() for _ in range(8)]
    want = [rt.decode_attention_shared(q, c, 8, 3000) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 2]):
            got.append(rt.decode_attention_shared(q, c, 8, 3000))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_a_step_refuses_what_does_not_fit_the_cache(rt):
    c, lens = _shared_cache(rt, 200, [1, 2], 2, 64, 128, seed=9)
    c.shared_prefix = 200
    ok = dict(B=2, H=8, Hkv=2, D=64, kv=2, pos=[201])
    for bad in (dict(B=3), dict(D=128), dict(Hkv=4, kv=4), dict(kv=4), dict(pos=[1, 2, 3]), dict(rows=3)):
        a = {**ok, **bad}
        q = torch.zeros(a["B"], a["H"], 1, a["D"], device="cuda", dtype=torch.bfloat16)
        kv = torch.zeros(a["B"], a["kv"], 1, a["D"], device="cuda", dtype=torch.bfloat16)
        table = tuple(torch.zeros(a["rows"], a["D"], device="cuda") for _ in range(2)) if "rows" in a else None
        with pytest.raises(RuntimeError):
            rt.decode_step(q, kv, kv, c, torch.tensor(a["pos"], device="cuda"), 1e4, a["Hkv"], rope_table=table)
        assert c.host_lengths() == lens and c.lengths.tolist() == lens
