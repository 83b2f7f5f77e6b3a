"""How the shared-prefix decode is ordered behind the kernels before it: its two grids run side by side, the second
behind the ticket that the first publishes in the workspace.  Needs a B200."""
import ctypes as C
import math

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


def _cache(rt, kv8, prefix, B, Hkv, D, room=40):
    """B sequences that begin with the same `prefix` rows, and one row each behind it."""
    cls = rt.PagedKVCache8 if kv8 else rt.PagedKVCache
    per = -(-(prefix + room) // 128)
    c = cls(num_blocks=per * B, num_kv_heads=Hkv, head_dim=D, block_size=128, max_seqs=B, max_blocks_per_seq=per)
    g = torch.Generator(device="cuda").manual_seed(prefix)
    if kv8:
        for pool in (c.k_pool, c.v_pool):
            pool.copy_((torch.randn(pool.shape, device="cuda", generator=g) * 110).clamp(-448, 448).to(rt.FP8))
        c.k_exp.fill_(127 - 7)
        c.v_exp.fill_(127 - 7)
    else:
        c.k_pool.normal_(generator=g)
        c.v_pool.normal_(generator=g)
    c.set_lengths([prefix])
    for b in range(1, B):
        c.fork(0, b, prefix)
    c.set_lengths([prefix + 1] * B)
    return c


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("H,Hkv,D,B,prefix", [(32, 8, 128, 40, 3000), (8, 2, 64, 3, 130)])
def test_whatever_a_workspace_holds(rt, H, Hkv, D, B, prefix, kv8):
    """Calls in one workspace whose bytes are anything before the first and what the last one left before the others; a
    call leaves no ticket behind, so that a replay of it waits for its own."""
    from mllm_b200 import abi
    c = _cache(rt, kv8, prefix, B, Hkv, D)
    q = torch.randn(B, H, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    want = rt.decode_attention_shared(q, c, Hkv, prefix)
    n = abi.load().mllm_decode_attention_shared_workspace_size(B, H, Hkv, D, prefix)
    out = torch.empty_like(want)
    name = "mllm_decode_attention_shared_paged_" + ("kv8" if kv8 else "bf16")
    desc = c.descriptor()

    def call(ws):
        abi.call(name, q.data_ptr(), C.byref(desc), c.lengths.data_ptr(), prefix, B, H, Hkv, D, prefix + 1,
                 1 / math.sqrt(D), out.data_ptr(), ws.data_ptr(), n, abi.stream_handle())
    for fill in (0, 255, 127):
        ws = torch.full((n,), fill, dtype=torch.uint8, device="cuda")
        for _ in range(3):
            out.fill_(float("nan"))
            call(ws)
            assert torch.equal(out, want)
            assert (ws[:8] == 0).all()
    graph = torch.cuda.CUDAGraph()
    ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    with torch.cuda.graph(graph):
        call(ws)
    for _ in range(3):
        out.fill_(float("nan"))
        graph.replay()
        assert torch.equal(out, want)
        assert (ws[:8] == 0).all()
    _status_ok()


@pytest.mark.parametrize("H,Hkv,D,B,prefix", [(8, 2, 128, 3, 300), (32, 4, 64, 40, 700)])
def test_rows_that_the_kernel_before_has_just_appended(rt, H, Hkv, D, B, prefix):
    """An append and the decode that reads it, again and again into the same cache rows: launches that all start early.
    Every result is the one with a wait for the device before each call."""
    N = 30
    c = _cache(rt, True, prefix, B, Hkv, D)
    cu = torch.arange(B + 1, dtype=torch.int32, device="cuda")
    start = torch.full((B,), prefix, dtype=torch.int32, device="cuda")
    pos = torch.full((B,), prefix, dtype=torch.int64, device="cuda")
    x = torch.randn(N, B, H + 2 * Hkv, D, device="cuda").bfloat16()
    q = torch.empty(B, H, D, device="cuda", dtype=torch.bfloat16)

    def step(i):
        rt.qkv_epilogue_kv8(x[i, :, :H], x[i, :, H:H + Hkv], x[i, :, H + Hkv:], c, cu, start, pos, 1e4, out=q)
        return rt.decode_attention_shared(q, c, Hkv, prefix, max_kv_len=prefix + 1)
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
