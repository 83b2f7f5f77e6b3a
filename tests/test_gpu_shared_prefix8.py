"""Decode attention over an 8-bit cache for a batch that shares a prefix: its prefix part bit for bit against the bf16
kernel over the rows read back, the whole against 64-bit attention, and through decode_step.  Needs a B200.

Tolerance (from the formats): the output is rounded to bf16 (2^-8 of the value at most), the prefix's P to bf16 (2^-8
of each weight, so 2^-8 of the weighted mean of |v|), the own rows' P to a half (less; but 2^-25 absolute below 2^-14,
against the largest weight times scale: 2^-25 of the largest |v| for each row), fp32 score sums 2^-18 of sum |q k|,
twice, as weight error."""
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


def _pools(c):
    return [c.k_pool.view(torch.uint8), c.v_pool.view(torch.uint8), c.k_exp, c.v_exp]


def _random_bytes(t, lo, hi, g):
    t.copy_(torch.randint(lo, hi, t.shape, device="cuda", generator=g, dtype=torch.int32).to(torch.uint8))


def _cache(rt, prefix, suffix, Hkv, D, block, seed, exps=((114, 118), (119, 123)), nan=False):
    """A cache of len(suffix) sequences forked from one prefix: every byte random (NaN only where asked for), the scales'
    exponent bytes from exps (K's, V's)."""
    B = len(suffix)
    lens = [prefix + s for s in suffix]
    per = -(-(prefix + max(suffix)) // block)
    c = rt.PagedKVCache8(num_blocks=per * B + 3, num_kv_heads=Hkv, head_dim=D, block_size=block, max_seqs=B,
                         max_blocks_per_seq=per + 1)
    random.Random(seed).shuffle(c._free)
    g = torch.Generator(device="cuda").manual_seed(seed)
    for pool in _pools(c)[:2]:
        _random_bytes(pool, 0, 256, g)
        if not nan:
            pool.sub_(((pool & 127) == 127).to(torch.uint8))
    _random_bytes(c.k_exp, *exps[0], g)
    _random_bytes(c.v_exp, *exps[1], g)
    c.reserve(0, prefix)
    for b in range(1, B):
        c.fork(0, b, prefix)
    c.set_lengths(lens)
    return c, lens


def _read_back(rt, c, prefix, lens):
    """A bf16 cache of the same sequences with the same prefix rows."""
    Hkv, D, block = c.k_pool.shape[1], c.k_pool.shape[3], c.block_size
    d = rt.PagedKVCache(num_blocks=c.num_blocks, num_kv_heads=Hkv, head_dim=D, block_size=block, max_seqs=len(lens),
                        max_blocks_per_seq=c.max_blocks_per_seq)
    d.reserve(0, prefix)
    rows = rt.kv8_read(c, torch.tensor([prefix], dtype=torch.int32, device="cuda"), len(d.blocks_of(0)) * block)
    for pool, r in zip((d.k_pool, d.v_pool), rows):
        for i, blk in enumerate(d.blocks_of(0)):
            pool[blk] = r[0, :, i * block:(i + 1) * block]
    for b in range(1, len(lens)):
        d.fork(0, b, prefix)
    d.set_lengths(lens)
    return d


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
        tol = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2 * ds + 2.0 ** -18) * mean_abs + L * 2.0 ** -25 * v.abs().max()
        assert ((o - ref).abs() <= tol).all(), (b, L, ((o - ref).abs() / tol).max())


SHAPES = [
    # H, Hkv, D, sequences, prefix (one tile: both kernels cut it alike), block
    (8, 2, 128, 1, 1, 128),
    (8, 2, 128, 3, 77, 128),
    (32, 8, 128, 32, 128, 256),        # one tile of query rows, full
    (32, 4, 64, 8, 120, 384),
    (40, 8, 128, 64, 128, 256),        # a pair and a single tile
    (4, 4, 64, 300, 65, 128),
    (7, 1, 64, 2, 128, 128),
]


@pytest.mark.parametrize("kind", ["usual", "large", "tiny", "nan"])
@pytest.mark.parametrize("H,Hkv,D,B,prefix,block", SHAPES)
def test_the_prefix_part_has_the_bits_of_the_bf16_kernel(rt, H, Hkv, D, B, prefix, block, kind):
    """A row of the cache stands for bf16 values exactly, and both kernels do the same with those (all 256 bytes, scales
    small and large, NaN): with no rows behind the prefix the results are equal bit for bit (where NaN, both are)."""
    exps = {"large": ((114, 118), (130, 141)), "tiny": ((27, 60), (27, 60))}.get(kind, ((114, 118), (119, 123)))
    c, lens = _cache(rt, prefix, [0] * B, Hkv, D, block, seed=3, exps=exps)
    if kind == "nan":   # in V of kv head 0, before the other sequences copy the block
        blk = c.blocks_of(0)[0]
        c.v_pool.view(torch.uint8)[blk, 0, 0, 5] = 0x7F
        c.v_pool.view(torch.uint8)[blk, 0, prefix - 1, D - 2] = 0xFF
        for b in range(1, B):
            if c.blocks_of(b)[0] != blk:
                c._copy_rows(blk, c.blocks_of(b)[0], prefix)
    d = _read_back(rt, c, prefix, lens)
    q = torch.randn(B, H, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    got = rt.decode_attention_shared(q, c, Hkv, prefix)
    want = rt.decode_attention_shared(q, d, Hkv, prefix)
    _status_ok()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.isnan(got).any() == (kind == "nan")
    assert torch.equal(got.nan_to_num(), want.nan_to_num())


CASES = [
    # H, Hkv, D, prefix, rows behind it, block, factor on q
    (8, 2, 128, 1, [1], 128, 1.0),
    (32, 8, 128, 127, [1, 2, 3], 128, 1.5),
    (32, 8, 128, 129, [0, 5, 64, 65], 256, 1.5),
    (32, 4, 64, 512, [1, 64, 17, 128, 0, 33, 2, 190], 128, 1.0),
    (32, 8, 128, 2000, [s % 200 for s in range(33)], 384, 1.5),
    (40, 8, 128, 5000, [s * 3 for s in range(64)], 256, 1.0),
    (10, 2, 128, 700, [300] * 130, 128, 2.0),
    (4, 4, 64, 300, [s % 3 for s in range(300)], 128, 1.0),
    (7, 1, 64, 40000, [9, 1], 128, 1.0),
]


@pytest.mark.parametrize("v_exps", [(119, 123), (90, 140)])
@pytest.mark.parametrize("H,Hkv,D,prefix,suffix,block,qf", CASES)
def test_against_64_bit_attention(rt, H, Hkv, D, prefix, suffix, block, qf, v_exps):
    c, lens = _cache(rt, prefix, suffix, Hkv, D, block, seed=5, exps=((114, 118), v_exps))
    q = (qf * torch.randn(len(lens), H, D, device="cuda",
                          generator=torch.Generator(device="cuda").manual_seed(6))).bfloat16()
    got = rt.decode_attention_shared(q, c, Hkv, prefix)
    _status_ok()
    _check(c, q, got, lens, Hkv)
    assert torch.equal(got, rt.decode_attention_shared(q, c, Hkv, prefix, max_kv_len=c.capacity))


@pytest.mark.parametrize("H,Hkv,D,B", [(32, 8, 128, 13), (32, 8, 128, 40), (32, 4, 64, 9), (4, 4, 64, 1)])
def test_one_call_after_another_at_many_prefix_lengths(rt, H, Hkv, D, B):
    q = torch.randn(B, H, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).bfloat16()
    for prefix in (200, 700, 1261, 1800, 2900, 4100, 6200, 8700, 10167, 13627):
        c, lens = _cache(rt, prefix, [1 + s % 9 for s in range(B)], Hkv, D, 384, seed=prefix)
        held = torch.full((1 << 24,), float("nan"), device="cuda")   # what the workspaces lie in next
        del held
        got = [rt.decode_attention_shared(q, c, Hkv, prefix) for _ in range(10)]
        _status_ok()
        _check(c, q, got[0], lens, Hkv)
        for x in got[1:]:
            assert torch.equal(got[0], x)


def test_any_part_of_the_common_rows_gives_the_same_answer(rt):
    c, lens = _cache(rt, 600, [1, 50, 200], 2, 128, 256, seed=7)
    q = torch.randn(3, 8, 128, device="cuda").bfloat16()
    for prefix in (0, 1, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 600):
        got = rt.decode_attention_shared(q, c, 2, prefix)
        _status_ok()
        _check(c, q, got, lens, 2)
    assert torch.equal(rt.decode_attention_shared(q, c, 2, 0), rt.decode_attention(q, c, 2))


def test_rows_behind_the_prefix_do_not_reach_other_sequences(rt):
    c, lens = _cache(rt, 200, [0, 30, 5], 2, 64, 128, seed=9)
    q = torch.randn(3, 8, 64, device="cuda").bfloat16()
    want = rt.decode_attention_shared(q, c, 2, 200)
    for b, L in enumerate(lens):
        blk = c.blocks_of(b)[L // 128]
        for t in _pools(c):
            t[blk, :, L % 128:] = 255
    got = rt.decode_attention_shared(q, c, 2, 200)
    _status_ok()
    assert torch.equal(want, got)


def test_a_padded_batch_short_lengths_and_bad_blocks(rt):
    from mllm_b200 import abi
    c, lens = _cache(rt, 300, [5, 6, 7, 8], 2, 128, 128, seed=4)
    q = torch.randn(4, 8, 128, device="cuda").bfloat16()
    full = rt.decode_attention_shared(q, c, 2, 300)
    keep = c.block_table.clone()
    for empty in ([0], [0, 1, 3], [2], [0, 1, 2, 3]):
        c.block_table.copy_(keep)
        for b in empty:
            c.block_table[b] = -7
        c.lengths.copy_(torch.tensor([0 if b in empty else n for b, n in enumerate(lens)], dtype=torch.int32))
        got = rt.decode_attention_shared(q, c, 2, 300, max_kv_len=308)
        _status_ok()
        for b in range(4):
            assert (got[b] == 0).all() if b in empty else torch.allclose(got[b], full[b], rtol=2.0 ** -6, atol=1e-2)
    c.block_table.copy_(keep)
    for bad in (-1, 299, 309):
        c.lengths.copy_(torch.tensor([305, bad, 307, 308], dtype=torch.int32))
        rt.decode_attention_shared(q, c, 2, 300, max_kv_len=308)
        with pytest.raises(abi.MllmError) as e:
            _status_ok()
        assert e.value.status == 7
    c.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
    c.block_table[0, 1] = c.num_blocks
    rt.decode_attention_shared(q, c, 2, 300, max_kv_len=308)
    with pytest.raises(abi.MllmError):
        _status_ok()
    c.block_table.copy_(keep)
    assert torch.equal(rt.decode_attention_shared(q, c, 2, 300, max_kv_len=308), full)
    _status_ok()


def test_captured_on_a_side_stream_and_two_at_once(rt):
    cases = []
    for seed, (H, Hkv, D, B, P) in enumerate([(32, 8, 128, 20, 3000), (8, 2, 64, 50, 900)]):
        c, lens = _cache(rt, P, [1 + 3 * s for s in range(B)], Hkv, D, 256, seed=seed)
        q = torch.randn(B, H, D, device="cuda").bfloat16()
        cases.append((c, q, Hkv, P, rt.decode_attention_shared(q, c, Hkv, P)))
    graphs = []
    for c, q, Hkv, P, _ in cases:
        s = torch.cuda.Stream()
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            out = rt.decode_attention_shared(q, c, Hkv, P, max_kv_len=c.capacity)
        graphs.append((g, out, s))
    for _ in range(20):
        for g, _, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
        for (c, q, Hkv, P, want), (_, _, s) in zip(cases, graphs):
            with torch.cuda.stream(s):
                assert torch.equal(rt.decode_attention_shared(q, c, Hkv, P), want)
    torch.cuda.synchronize()
    _status_ok()
    for (*_, want), (_, out, _) in zip(cases, graphs):
        assert torch.equal(out, want)


@pytest.mark.parametrize("B,prefix,used", [(8, 8192, True), (1, 8192, False), (8, 512, False)])
def test_a_step_reads_the_prefix_once_where_that_pays(rt, B, prefix, used, monkeypatch):
    """decode_step on an 8-bit cache with shared_prefix set against the step without it: outputs of two orders of
    summation with P rounded to bf16 or to a half, |v| <= 1: twice 2^-8 of the value and of 1."""
    H, Hkv, D = 32, 8, 128
    calls = []
    shared = rt.decode_attention_shared
    monkeypatch.setattr(rt, "decode_attention_shared", lambda *a: calls.append(a[3]) or shared(*a))
    c, lens = _cache(rt, prefix, [0] * B, Hkv, D, 256, seed=1, exps=((114, 118), (115, 119)))
    g = torch.Generator(device="cuda").manual_seed(B)
    q, k, v = (torch.randn(B, h, 1, D, device="cuda", generator=g).bfloat16() for h in (H, Hkv, Hkv))
    v.clamp_(-1, 1)
    got = []
    for shared_rows in (prefix, 0):
        c.shared_prefix = shared_rows
        c.set_lengths([prefix] * B)
        got.append(rt.decode_step(q, k, v, c, torch.tensor([prefix], device="cuda"), 1e6, Hkv).double())
    _status_ok()
    assert calls == ([prefix] if used else [])
    assert ((got[0] - got[1]).abs() <= 2 * 2.0 ** -8 * (1.75 + got[1].abs())).all()


@pytest.mark.parametrize("kv8", [True, False])
@pytest.mark.parametrize("H,Hkv,D,B,prefix", [(8, 2, 128, 3, 300), (32, 4, 64, 40, 700), (4, 4, 64, 1, 64)])
def test_queries_that_the_kernel_before_has_just_written(rt, H, Hkv, D, B, prefix, kv8):
    """The epilogue writes new queries into the same memory again and again, the decode reads them behind it: launches that
    all start early and wait for one another.  Every result is the one with a wait for the device before each call."""
    N = 40
    c, lens = _cache(rt, prefix, [1 + s % 9 for s in range(B)], Hkv, D, 128, seed=3)
    if not kv8:
        c = _read_back(rt, c, prefix, lens)
    appends = rt.PagedKVCache8(num_blocks=B, num_kv_heads=Hkv, head_dim=D, block_size=128, max_seqs=B)   # not looked at
    for b in range(B):
        appends.reserve(b, 1)
    cu = torch.arange(B + 1, dtype=torch.int32, device="cuda")
    start = torch.zeros(B, dtype=torch.int32, device="cuda")
    pos = torch.arange(B, device="cuda")
    x = torch.randn(N, B, H + 2 * Hkv, D, device="cuda").bfloat16()
    q = torch.empty(B, H, D, device="cuda", dtype=torch.bfloat16)

    def step(i):
        rt.qkv_epilogue_kv8(x[i, :, :H], x[i, :, H:H + Hkv], x[i, :, H + Hkv:], appends, cu, start, pos, 1e4, out=q)
        return rt.decode_attention_shared(q, c, Hkv, prefix, max_kv_len=max(lens))
    want = []
    for i in range(N):
        torch.cuda.synchronize()
        want.append(step(i).clone())
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        recorded = [step(i) for i in range(N)]
    for _ in range(5):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(recorded, want))
        again = [step(i) for i in range(N)]
        assert all(torch.equal(a, b) for a, b in zip(again, want))
    _status_ok()
