"""The 8-bit paged KV cache: the quantising epilogue, the read-back and the decode attention against plain
64-bit arithmetic, and attention through the framework's functions on it.  Needs a B200.

Tolerances (fixed from the formats, not from runs).  A rounding is off by at most half a step: 2^-8 of the value
for bf16, 2^-4 for e4m3 (2^-10 of the row's scale below its smallest normal), 2^-11 for a half (2^-25 absolute
below 2^-14).  fp32 steps are given 2^-18 of the norm of what they sum: sums of D <= 128 products, each step
2^-24, and the approximate exp2 (2^-22)."""
import math
import random

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

BF16_HALF, E4M3_HALF, F16_HALF, F32 = 2.0 ** -8, 2.0 ** -4, 2.0 ** -11, 2.0 ** -18


@pytest.fixture(scope="module")
def rt(cuda_device):
    from mllm_b200 import build
    build.build()
    from mllm_b200 import runtime
    return runtime


def _status_ok():
    from mllm_b200 import abi
    abi.call("mllm_attn_device_status", None)


def _cache(rt, n, Hkv, D, rows, block=128, seed=0, extra=2):
    c = rt.PagedKVCache8(num_blocks=n * (-(-rows // block)) + extra, num_kv_heads=Hkv, head_dim=D, block_size=block,
                         max_seqs=max(n, 1))
    random.Random(seed).shuffle(c._free)
    return c


def _fill_garbage(c, g):
    """Every byte of the pools random (NaN bytes among them), as freed memory may be."""
    for t in (c.k_pool.view(torch.uint8), c.v_pool.view(torch.uint8), c.k_exp, c.v_exp):
        t.copy_(torch.randint(0, 256, t.shape, device="cuda", generator=g, dtype=torch.int32).to(torch.uint8))


def _bytes(c):
    return [t.clone() for t in (c.k_pool.view(torch.uint8), c.v_pool.view(torch.uint8), c.k_exp, c.v_exp)]


def _quantise64(y):
    """The format's definition in 64 bits, of finite rows: (values as stored, 2^e)."""
    scale = torch.exp2(torch.ceil(torch.log2(y.abs().amax(-1, keepdim=True).clamp_min(1e-300) / 448)).clamp(-100, 120))
    x = y / scale
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(1e-300))).clamp_min(-6) - 3)
    return torch.round(x / step) * step * scale, scale


def _norm_rope64(x, w, cos, sin, eps):
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    lo, hi = x.chunk(2, -1)
    c, s = cos.double()[:, None], sin.double()[:, None]
    h = lo.shape[-1]
    return torch.cat([lo * c[..., :h] - hi * s[..., :h], hi * c[..., h:] + lo * s[..., h:]], -1)


EPILOGUE = [
    # H, Hkv, D, tokens per sequence, rows before them, tokens behind the last sequence, norm, offset of the views
    (32, 8, 128, [1] * 5, [4096, 0, 127, 128, 1], 0, True, 0),
    (8, 2, 128, [37, 1, 300, 0, 129], [0, 5, 0, 3, 200], 0, True, 0),
    (10, 2, 128, [77, 200], [51, 0], 3, False, 0),
    (32, 4, 64, [256, 3, 40], [0, 128, 1], 1, True, 0),
    (4, 4, 64, [1, 1, 0, 2], [10, 300, 7, 0], 0, False, 4),
    (5, 1, 128, [33], [95], 2, True, 1),             # rows that start on no 8-byte boundary
    (40, 8, 128, [2] * 40, list(range(40)), 0, True, 0),   # more sequences than one ballot
    # enough tokens for the form that streams them (some SMs' warps get one more than others)
    (8, 2, 128, [3000, 1, 0, 777, 1500], [0, 130, 9, 5, 100], 5, True, 0),
    (5, 1, 64, [1] * 50 + [4999], [3] * 51, 0, False, 0),
    (10, 2, 64, [2500, 2499], [0, 1], 700, True, 8),
]


@pytest.mark.parametrize("H,Hkv,D,tokens,start,behind,norm,off", EPILOGUE)
def test_epilogue_and_read_against_the_formula(rt, H, Hkv, D, tokens, start, behind, norm, off):
    g = torch.Generator(device="cuda").manual_seed(1)
    n, T = len(tokens), sum(tokens) + behind
    c = _cache(rt, n, Hkv, D, max(s + t for s, t in zip(start, tokens)) + 1, seed=3)
    for b in range(n):
        c.reserve(b, start[b] + tokens[b])
    _fill_garbage(c, g)
    before = _bytes(c)
    W = (H + 2 * Hkv) * D + (off and 1)
    flat = torch.randn(T * W + off, device="cuda", generator=g).bfloat16()[off:].view(T, W)
    q = flat[:, : H * D].view(T, H, D)
    k = flat[:, H * D:(H + Hkv) * D].view(T, Hkv, D)
    v = flat[:, (H + Hkv) * D:(H + 2 * Hkv) * D].view(T, Hkv, D)
    ang = torch.rand(T, D // 2, device="cuda", generator=g, dtype=torch.float64) * 6.3
    cos, sin = torch.cat([ang, ang], 1).cos().float(), torch.cat([ang, ang], 1).sin().float()
    wq = (1 + 0.1 * torch.randn(D, device="cuda", generator=g)).bfloat16() if norm else None
    wk = (1 + 0.1 * torch.randn(D, device="cuda", generator=g)).bfloat16() if norm else None
    cu = torch.tensor([sum(tokens[:b]) for b in range(n + 1)], dtype=torch.int32, device="cuda")
    st = torch.tensor(start, dtype=torch.int32, device="cuda")
    out = torch.full((T, H, D), 7.0, dtype=torch.bfloat16, device="cuda")
    got = rt.qkv_epilogue_kv8(q, k, v, c, cu, st, rope_table=(cos, sin), q_norm_weight=wq, k_norm_weight=wk, eps=1e-6,
                              out=out)
    _status_ok()
    own = T - behind
    q64 = _norm_rope64(q, wq, cos, sin, 1e-6)[:own]
    tol = BF16_HALF * q64.abs() + F32 * q64.norm(dim=-1, keepdim=True)
    assert ((got[:own].double() - q64).abs() <= tol).all()
    assert (got[own:] == 7.0).all()                       # tokens behind the last sequence: left as they were

    rows = max(tokens + [1])
    lens = torch.tensor([s + t for s, t in zip(start, tokens)], dtype=torch.int32, device="cuda")
    kr, vr = rt.kv8_read(c, lens, rows, first=st)
    _status_ok()
    k64 = _norm_rope64(k, wk, cos, sin, 1e-6)
    v64, _ = _quantise64(v.double())
    written = set()
    for b in range(n):
        t0, t1 = sum(tokens[:b]), sum(tokens[:b + 1])
        gk, gv = kr[b, :, : t1 - t0].double().transpose(0, 1), vr[b, :, : t1 - t0].double().transpose(0, 1)
        ref = k64[t0:t1]
        scale = _quantise64(ref)[1]
        noise = F32 * ref.norm(dim=-1, keepdim=True)
        assert ((gk - ref).abs() <= E4M3_HALF * ref.abs() + 2.0 ** -10 * scale + noise).all()
        assert (gv == v64[t0:t1]).all()                   # V comes from bf16: no fp32 step before its rounding
        assert (kr[b, :, t1 - t0:] == 0).all() and (vr[b, :, t1 - t0:] == 0).all()
        for r in range(start[b], start[b] + tokens[b]):
            written.add((c.blocks_of(b)[r // c.block_size], r % c.block_size))
    keep = torch.ones(c.num_blocks, c.block_size, dtype=torch.bool)
    for blk, r in written:
        keep[blk, r] = False
    keep = keep.cuda()
    for x, y in zip(before, _bytes(c)):                   # nothing else in the pools changed
        same = (x == y).flatten(3).all(-1) if x.dim() == 4 else x == y
        assert same.transpose(1, 2)[keep].all()


def test_tokens_in_front_of_the_first_sequence(rt):
    """Tokens before cu_seqlens[0] belong to no sequence: enough of them that a warp of the streaming form begins
    with such tokens and goes on to owned ones.  The owned rows are those of a call on the owned tokens alone."""
    H, Hkv, D, lead, tokens = 4, 1, 64, 4000, [1500, 2500]
    g = torch.Generator(device="cuda").manual_seed(8)
    T = lead + sum(tokens)
    q, k, v = (torch.randn(T, h, D, device="cuda", generator=g).bfloat16() for h in (H, Hkv, Hkv))
    pos = torch.arange(T, device="cuda")
    st = torch.zeros(2, dtype=torch.int32, device="cuda")
    got = []
    for first in (lead, 0):
        c = _cache(rt, 2, Hkv, D, max(tokens))
        for b in range(2):
            c.reserve(b, tokens[b])
        cu = torch.tensor([first, first + tokens[0], first + sum(tokens)], dtype=torch.int32, device="cuda")
        skip = lead - first
        out = torch.full((T - skip, H, D), 7.0, dtype=torch.bfloat16, device="cuda")
        rt.qkv_epilogue_kv8(q[skip:], k[skip:], v[skip:], c, cu, st, pos[skip:].contiguous(), 1e4, out=out)
        _status_ok()
        assert (out[:first] == 7).all()
        got.append([out[first:]] + [c.gather(b, tokens[b]) for b in range(2)])
    assert torch.equal(got[0][0], got[1][0])
    for x, y in zip(got[0][1:], got[1][1:]):
        assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1]) and x[0].abs().max() > 1


def test_epilogue_from_positions_equals_the_table(rt):
    """Angles from positions are those of the framework's RoPE table."""
    g = torch.Generator(device="cuda").manual_seed(2)
    H, Hkv, D, T = 8, 2, 128, 50
    x = torch.randn(T, H + 2 * Hkv, D, device="cuda", generator=g).bfloat16()
    pos = torch.randint(0, 40000, (T,), device="cuda", generator=g)
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    res = []
    for table in (None, rt.RoPE.build_cos_sin(pos, D, 1e6)):
        c = _cache(rt, 1, Hkv, D, T)
        c.reserve(0, T)
        q = rt.qkv_epilogue_kv8(x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:], c, cu, st, pos, 1e6, table)
        res.append([q.view(torch.int16)] + _bytes(c))
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_rows_out_of_the_ordinary(rt):
    """Zero rows, rows of very small and very large numbers, and non-finite elements (stored as NaN, the others of
    the row as if they were not there)."""
    D, T = 64, 6
    v = torch.zeros(T, 1, D)
    v[1] = torch.linspace(-1, 1, D) * 2.0 ** -125         # below the smallest scale: zero
    v[2] = torch.linspace(-1, 1, D) * 2.0 ** 126
    v[3] = torch.linspace(-3, 3, D)
    v[3, 0, 5], v[3, 0, 6], v[3, 0, 7] = float("inf"), float("-inf"), float("nan")
    v[4, 0, 9] = 448.0 * 2.0 ** 7
    v[5, 0, 9] = 449.0 * 2.0 ** 7
    v = v.bfloat16().cuda()
    q = torch.zeros(T, 1, D, dtype=torch.bfloat16, device="cuda")
    c = _cache(rt, 1, 1, D, T)
    c.reserve(0, T)
    cu, st = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, T], [0]))
    rt.qkv_epilogue_kv8(q, q, v, c, cu, st, torch.zeros(T, dtype=torch.int64, device="cuda"))
    _, got = rt.kv8_read(c, torch.tensor([T], dtype=torch.int32, device="cuda"), T)
    got = got[0, 0].double()
    ref = v[:, 0].double()
    bad = ~torch.isfinite(ref)
    assert torch.isnan(got[bad]).all() and torch.isfinite(got[~bad]).all()
    clean = torch.where(bad, 0.0, ref)
    want = _quantise64(clean)[0]
    assert (got[~bad] == want[~bad]).all()
    assert (got[0] == 0).all() and (got[1] == 0).all()


def _attention64(q, k, v):
    """q [Hkv, R, D], k/v [Hkv, L, D]: 64-bit attention, and its normalised weights."""
    s = torch.einsum("grd,gtd->grt", q, k) / math.sqrt(q.shape[-1])
    w = torch.softmax(s, -1)
    return torch.einsum("grt,gtd->grd", w, v), w


def _check_decode(rt, c, q, got, lens, Hkv):
    B, H, D = q.shape
    for b, L in enumerate(lens):
        o = got[b, 0].view(Hkv, H // Hkv, D).double()
        if L == 0:
            assert (o == 0).all()
            continue
        k, v = (x.double() for x in c.gather(b, L))
        idx = torch.tensor(c.blocks_of(b), device="cuda")
        ev = torch.exp2(c.v_exp[idx].double() - 127).transpose(0, 1).flatten(1, 2)[:, :L]     # [Hkv, L]
        qq = q[b].view(Hkv, H // Hkv, D).double()
        ref, w = _attention64(qq, k, v)
        ws = w * ev[:, None]
        mean_abs = torch.einsum("grt,gtd->grd", w, v.abs())
        # scores: fp32 sums of products, 2^-18 of sum |q k|, change the weights by that much relative
        ds = F32 * torch.einsum("grd,gtd->grt", qq.abs(), k.abs()).amax(-1, keepdim=True) / math.sqrt(D)
        small = 2.0 ** -25 * ws.amax(-1, keepdim=True) * (v.abs() / ev[..., None]).sum(1)[:, None]
        tol = BF16_HALF * ref.abs() + (F16_HALF + 2 * ds + F32) * mean_abs + small + 1e-37
        assert ((o - ref).abs() <= tol).all(), (b, L, ((o - ref).abs() / tol).max())


def _random_cache(rt, lens, Hkv, D, block, spread, seed):
    """A cache of random rows, whatever lies behind their ends random bytes."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = _cache(rt, len(lens), Hkv, D, max(lens + [1]), block, seed)
    c.set_lengths(list(lens))
    _fill_garbage(c, g)
    for b, L in enumerate(lens):
        for i, blk in enumerate(c.blocks_of(b)):
            r = min(block, L - i * block)
            for pool, exps in ((c.k_pool, c.k_exp), (c.v_pool, c.v_exp)):
                pool.view(torch.uint8)[blk, :, :r] = \
                    (torch.randn(Hkv, r, D, device="cuda", generator=g) * 110).clamp(-448, 448).to(rt.FP8).view(torch.uint8)
                e = torch.randint(-spread, spread + 1, (Hkv, r), device="cuda", generator=g)
                exps[blk, :, :r] = (120 + e).to(torch.uint8)
    return c


DECODE = [
    # H, Hkv, D, lengths, block, spread of the rows' exponents, factor on q
    (32, 8, 128, [4096, 4097, 1, 0, 127, 128, 129, 63, 64, 65], 256, 1, 1.5),
    (40, 8, 128, [513, 33, 16, 15, 17, 31, 32, 300], 128, 2, 1.0),
    (32, 4, 64, [513], 128, 1, 1.0),
    (8, 8, 128, [200, 0, 0, 777], 384, 0, 2.0),
    (7, 1, 64, [1000, 5, 130], 128, 1, 1.0),
    (2, 2, 64, [1], 128, 1, 1.0),
    (10, 2, 128, [0, 0, 0], 128, 1, 1.0),
    (10, 2, 128, [700, 91], 128, 20, 1e-4),      # rows of very different size
    (10, 2, 128, [700, 91], 128, 1, 300.0),      # one weight close to 1
    (16, 2, 64, [40] * 70 + [0] * 3 + [129] * 30, 128, 1, 1.0),   # more sequences than three warps of lengths
    (8, 2, 128, [768, 0, 5], 128, 1, 1.0),       # the longest that is not cut, and one row more
    (8, 2, 128, [769, 0, 5], 128, 1, 1.0),
    (4, 4, 64, [300] * 75, 128, 1, 1.0),         # short, but more pairs than CTAs
]


@pytest.mark.parametrize("H,Hkv,D,lens,block,spread,qf", DECODE)
def test_decode_against_64_bit_attention(rt, H, Hkv, D, lens, block, spread, qf):
    c = _random_cache(rt, lens, Hkv, D, block, spread, seed=11)
    g = torch.Generator(device="cuda").manual_seed(5)
    q = (torch.randn(len(lens), H, D, device="cuda", generator=g) * qf).bfloat16()
    got = rt.decode_attention(q, c, Hkv, max_kv_len=max(lens + [1]))
    _status_ok()
    _check_decode(rt, c, q, got, lens, Hkv)
    # a larger bound on the lengths changes nothing, nor does a second call
    again = rt.decode_attention(q, c, Hkv, max_kv_len=c.capacity)
    assert torch.equal(got, again)


def test_decode_of_queries_and_rows_that_are_not_numbers(rt):
    """A NaN in a query reaches that head's output only; a NaN row the heads of its kv head only."""
    c = _random_cache(rt, [300, 200], 2, 64, 128, 1, seed=3)
    q = torch.randn(2, 8, 64, device="cuda").bfloat16()
    clean = rt.decode_attention(q, c, 2, max_kv_len=300)
    bad = q.clone()
    bad[0, 5, 3] = float("nan")
    got = rt.decode_attention(bad, c, 2, max_kv_len=300).view(2, 8, 64)
    assert torch.isnan(got[0, 5]).all()
    got[0, 5] = clean.view(2, 8, 64)[0, 5]
    assert torch.equal(got, clean.view(2, 8, 64))
    c.v_pool.view(torch.uint8)[c.blocks_of(1)[0], 1, 17, 9] = 0x7F
    got = rt.decode_attention(q, c, 2, max_kv_len=300).view(2, 8, 64)
    assert torch.isnan(got[1, 4:, 9]).all() and torch.equal(got[0], clean.view(2, 8, 64)[0])
    assert torch.equal(got[1, :4], clean.view(2, 8, 64)[1, :4])


def test_decode_on_a_side_stream_and_two_at_once(rt):
    lens = [2000, 1500, 3, 900]
    c = _random_cache(rt, lens, 8, 128, 256, 1, seed=8)
    qs = [torch.randn(4, 32, 128, device="cuda").bfloat16() for _ in range(8)]
    want = [rt.decode_attention(q, c, 8, max_kv_len=2000) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 2]):
            got.append(rt.decode_attention(q, c, 8, max_kv_len=2000))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_bad_lengths_and_blocks_are_recorded(rt):
    from mllm_b200 import abi
    c = _random_cache(rt, [300, 40], 2, 128, 128, 1, seed=9)
    q = torch.randn(2, 8, 128, device="cuda").bfloat16()
    for bad in (-1, 301):
        c.lengths[1] = bad
        rt.decode_attention(q, c, 2, max_kv_len=300)
        with pytest.raises(abi.MllmError) as e:
            _status_ok()
        assert e.value.status == 7
    c.lengths[1] = 40
    keep = c.block_table.clone()
    c.block_table[1, 0] = c.num_blocks
    x = torch.zeros(2, 12, 128, dtype=torch.bfloat16, device="cuda")
    before = _bytes(c)
    rt.qkv_epilogue_kv8(x[:, :8], x[:, 8:10], x[:, 10:], c, torch.tensor([0, 0, 2], dtype=torch.int32, device="cuda"),
                        torch.tensor([0, 3], dtype=torch.int32, device="cuda"),
                        torch.zeros(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(abi.MllmError):
        _status_ok()
    assert all(torch.equal(a, b) for a, b in zip(before, _bytes(c)))
    kr, _ = rt.kv8_read(c, c.lengths[:2], 300)
    with pytest.raises(abi.MllmError):
        _status_ok()
    assert (kr[1] == 0).all()
    c.block_table.copy_(keep)
    rt.decode_attention(q, c, 2, max_kv_len=300)
    _status_ok()


def test_a_step_at_one_position_for_all(rt):
    """positions [1] stands for every sequence's, as on the other caches."""
    got = []
    for pos in ([300], [300] * 3, [[300]] * 3):
        c = _random_cache(rt, [300] * 3, 2, 128, 128, 1, seed=9)
        q, k, v = (torch.randn(3, h, 1, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(h)).bfloat16()
                   for h in (8, 2, 2))
        got.append(rt.decode_step(q, k, v, c, torch.tensor(pos, device="cuda"), 1e4, 2))
    _status_ok()
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_a_negative_first_row_reads_nothing(rt):
    from mllm_b200 import abi
    c = _random_cache(rt, [300, 40], 2, 128, 128, 1, seed=9)
    for first in (-1, -200, -(2 ** 31)):
        f = torch.tensor([first, 7], dtype=torch.int32, device="cuda")
        kr, vr = rt.kv8_read(c, c.lengths[:2], 256, first=f)
        with pytest.raises(abi.MllmError) as e:
            _status_ok()
        assert e.value.status == 7
        assert (kr[0] == 0).all() and (vr[0] == 0).all() and (kr[1, :, 33:] == 0).all()
        assert torch.equal(kr[1, :, :33].float(), c.gather(1, 40)[0][:, 7:])


@pytest.mark.parametrize("H,Hkv,D,norm", [(8, 2, 128, True), (8, 4, 64, False)])
def test_prompts_then_steps_through_the_framework(rt, H, Hkv, D, norm):
    """Packed prompts, a second chunk of one of them, then decode steps (eager and from a captured graph): every
    output against 64-bit attention over what the cache holds, and chunked the same as at once."""
    g = torch.Generator(device="cuda").manual_seed(4)
    wq = (1 + 0.1 * torch.randn(D, device="cuda", generator=g)).bfloat16() if norm else None
    wk = (1 + 0.1 * torch.randn(D, device="cuda", generator=g)).bfloat16() if norm else None
    lens = [150, 7, 260]
    T = sum(lens)
    x = torch.randn(T, (H + 2 * Hkv), D, device="cuda", generator=g).bfloat16()

    def packed(c, rows, q_lens):
        q = rt.qkv_epilogue_packed(rows[:, :H], rows[:, H:H + Hkv], rows[:, H + Hkv:], c, q_lens, 1e4,
                                   q_norm_weight=wq, k_norm_weight=wk)
        return q, rt.prefill_attention_packed(q, c, q_lens, Hkv)
    c = _cache(rt, 3, Hkv, D, 400)
    q, out = packed(c, x, lens)
    c2 = _cache(rt, 3, Hkv, D, 400, seed=5)
    packed(c2, x[:157 + 200], [150, 7, 200])
    _, out2 = packed(c2, x[157 + 200:], [0, 0, 60])
    _status_ok()
    assert torch.equal(out2, out[157 + 200:])
    t = 0
    for b, L in enumerate(lens):
        k, v = (y.double() for y in c.gather(b, L))
        qq = q[:, t:t + L].double().view(Hkv, H // Hkv, L, D)
        s = torch.einsum("grsd,gtd->grst", qq, k) / math.sqrt(D)
        s = s.masked_fill(torch.ones(L, L, dtype=torch.bool, device="cuda").triu(1), float("-inf"))
        w = torch.softmax(s, -1)
        ref = torch.einsum("grst,gtd->sgrd", w, v).reshape(L, H * D)
        mean = torch.einsum("grst,gtd->sgrd", w, v.abs()).reshape(L, H * D)
        # P is rounded to bf16 by the prefill kernel
        assert ((out[t:t + L].double() - ref).abs() <= BF16_HALF * ref.abs() + (BF16_HALF + 2.0 ** -12) * mean).all()
        t += L

    def step(c, x):
        pos = c.lengths[:3].long()
        return rt.decode_step(x[:, :H, None], x[:, H:H + Hkv, None], x[:, H + Hkv:, None], c, pos, 1e4, Hkv, wq, wk)
    xs = [torch.randn(3, H + 2 * Hkv, D, device="cuda", generator=g).bfloat16() for _ in range(4)]
    eager = [step(c, y) for y in xs]
    _status_ok()
    assert c.host_lengths() == [n + 4 for n in lens]
    buf = xs[0].clone()
    c2.set_lengths(lens)
    for b in range(3):
        c2.reserve(b, 400)
    c2.capture_max_len = 400
    graph = torch.cuda.CUDAGraph()
    scratch = rt.GraphScratch()
    with rt.graph_scratch(scratch), torch.cuda.graph(graph):
        o = step(c2, buf)
    c2.capture_max_len = None
    c2.set_lengths(lens)
    for i, y in enumerate(xs):
        buf.copy_(y)
        graph.replay()
        c2.advance_host(1, 3)
        assert torch.equal(o, eager[i])
    assert c2.lengths.tolist() == c.lengths.tolist()
    _status_ok()
    # [B, H, S, D] calls on equal lengths do the same as packed ones
    c3, c4 = _cache(rt, 2, Hkv, D, 200), _cache(rt, 2, Hkv, D, 200, seed=2)
    y = x[:140]
    q4, o4 = packed(c4, y, [70, 70])
    b4 = y.view(2, 70, H + 2 * Hkv, D).transpose(1, 2)
    q3 = rt.qkv_epilogue(b4[:, :H], b4[:, H:H + Hkv], b4[:, H + Hkv:], c3, torch.arange(70, device="cuda"), 1e4, wq, wk)
    assert torch.equal(q3.transpose(0, 1).reshape(H, 140, D), q4)
    assert torch.equal(rt.prefill_attention(q3, c3, Hkv).view(140, H * D), o4)
