"""The serving operators on memory whose offsets pass 32 bits: the same rows at the front and at the far end of large
buffers give the same bits.  Needs a B200 (about 30 GB of it)."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

FAR = 2 ** 31 + 4096            # elements: beyond 2^32 bytes of 2-byte numbers, beyond a signed 32-bit index


@pytest.fixture(scope="module")
def rt(cuda_device):
    from mllm_b200 import build
    build.build()
    from mllm_b200 import runtime
    return runtime


@pytest.fixture(autouse=True)
def _free(cuda_device):
    yield
    torch.cuda.empty_cache()


def _status_ok():
    from mllm_b200 import abi
    abi.call("mllm_attn_device_status", None)


def _ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def test_8bit_cache_with_blocks_far_apart(rt):
    H, Hkv, D = 8, 2, 128
    T, blocks = 200, 2 ** 33 // (Hkv * 128 * D) // 2 + 70   # a pool of 4.3 GB, twice
    near = rt.PagedKVCache8(4, Hkv, D, 128, 1)
    far = rt.PagedKVCache8(blocks, Hkv, D, 128, 1, max_blocks_per_seq=4)
    assert far.k_pool.numel() > 2 ** 32
    far._free.reverse()                                     # the last blocks first
    x = torch.randn(T, H + 2 * Hkv, D, device="cuda").bfloat16()
    big = torch.empty(FAR + T * (H + 2 * Hkv) * D, dtype=torch.bfloat16, device="cuda")
    y = big[FAR:].view(T, H + 2 * Hkv, D)
    y.copy_(x)
    res = []
    for c, src in ((near, x), (far, y)):
        c.reserve(0, T)
        q = rt.qkv_epilogue_kv8(src[:, :H], src[:, H:H + Hkv], src[:, H + Hkv:], c, _ints(0, T), _ints(0),
                                torch.arange(T, device="cuda"), 1e4)
        c.set_lengths([T])
        k, v = rt.kv8_read(c, c.lengths[:1], T)
        res.append((q, k, v, rt.decode_attention(q[-1:].contiguous(), c, Hkv)))
    _status_ok()
    assert max(far.blocks_of(0)) * Hkv * 128 * D > 2 ** 32 - 2 ** 22
    for a, b in zip(*res):
        assert torch.equal(a, b)


def test_token_rows_far_apart(rt):
    """Two tokens whose projections lie more than 2^31 elements apart, and an output of the same layout."""
    H, Hkv, D = 4, 2, 64
    W = (H + 2 * Hkv) * D
    big = torch.zeros(FAR + W, dtype=torch.bfloat16, device="cuda")
    rows = big.as_strided((2, H + 2 * Hkv, D), (FAR, D, 1))
    rows.copy_(torch.randn(2, H + 2 * Hkv, D, device="cuda"))
    out = torch.zeros(FAR + H * D, dtype=torch.bfloat16, device="cuda").as_strided((2, H, D), (FAR, D, 1))
    dense = rows.contiguous()
    res = []
    for src, o in ((rows, out), (dense, None)):
        c = rt.PagedKVCache8(2, Hkv, D, 128, 1)
        c.reserve(0, 2)
        q = rt.qkv_epilogue_kv8(src[:, :H], src[:, H:H + Hkv], src[:, H + Hkv:], c, _ints(0, 2), _ints(0),
                                torch.arange(2, device="cuda"), 1e4, out=o)
        res.append((q.contiguous(), *rt.kv8_read(c, _ints(2), 2)))
    _status_ok()
    for a, b in zip(*res):
        assert torch.equal(a, b)


def test_shared_prefix_with_blocks_far_apart(rt):
    H, Hkv, D, P = 8, 2, 128, 300
    blocks = 2 ** 33 // (Hkv * 128 * D * 2) // 2 + 70
    near = rt.PagedKVCache(12, Hkv, D, 128, 3, max_blocks_per_seq=4)
    far = rt.PagedKVCache(blocks, Hkv, D, 128, 3, max_blocks_per_seq=4)
    assert far.k_pool.numel() * 2 > 2 ** 32
    far._free.reverse()
    near.k_pool.normal_()
    near.v_pool.normal_()
    for c in (near, far):
        c.reserve(0, P)
        for b in (1, 2):
            c.fork(0, b, P)
        c.set_lengths([P + 3, P + 100, P])
    for b in range(3):
        for i, j in zip(near.blocks_of(b), far.blocks_of(b)):
            far.k_pool[j], far.v_pool[j] = near.k_pool[i], near.v_pool[i]
    q = torch.randn(3, H, D, device="cuda").bfloat16()
    assert torch.equal(rt.decode_attention_shared(q, near, Hkv, P), rt.decode_attention_shared(q, far, Hkv, P))
    _status_ok()


def test_shared_prefix_of_8bit_blocks_far_apart(rt):
    H, Hkv, D, P = 8, 2, 128, 300
    near = rt.PagedKVCache8(12, Hkv, D, 128, 3, max_blocks_per_seq=4)
    far = rt.PagedKVCache8(2 ** 33 // (Hkv * 128 * D) // 2 + 70, Hkv, D, 128, 3, max_blocks_per_seq=4)
    assert far.k_pool.numel() > 2 ** 32
    far._free.reverse()
    pools = [[c.k_pool.view(torch.uint8), c.v_pool.view(torch.uint8), c.k_exp, c.v_exp] for c in (near, far)]
    for t, lo, hi in zip(pools[0], (0, 0, 114, 119), (127, 127, 118, 123)):
        t.copy_(torch.randint(lo, hi, t.shape, device="cuda").to(torch.uint8))
    for c in (near, far):
        c.reserve(0, P)
        for b in (1, 2):
            c.fork(0, b, P)
        c.set_lengths([P + 3, P + 100, P])
    for b in range(3):
        for i, j in zip(near.blocks_of(b), far.blocks_of(b)):
            for a, z in zip(*pools):
                z[j] = a[i]
    q = torch.randn(3, H, D, device="cuda").bfloat16()
    assert torch.equal(rt.decode_attention_shared(q, near, Hkv, P), rt.decode_attention_shared(q, far, Hkv, P))
    _status_ok()


def test_logit_rows_far_apart(rt):
    V = 5000
    big = torch.zeros(FAR + V, dtype=torch.bfloat16, device="cuda")
    x = big.as_strided((2, V), (FAR, 1))
    x.copy_(torch.randn(2, V, device="cuda"))
    hist = torch.randint(0, V, (2, 50), device="cuda")
    kw = dict(history=hist, history_lens=_ints(50, 30), repetition=torch.full((2,), 1.5, device="cuda"),
              frequency=torch.full((2,), 0.5, device="cuda"))
    want = rt.apply_logit_rules(x.contiguous(), **kw)
    assert torch.equal(rt.apply_logit_rules(x, **kw), want)
    rt.apply_logit_rules(x, **kw, out=x)
    assert torch.equal(x, want)
    _status_ok()
