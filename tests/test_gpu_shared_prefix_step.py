"""decode_step on a cache with shared_prefix set whose sequences have not all come by the prefix together.  Needs a
B200."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def rt(cuda_device):
    from mllm_b200 import build
    build.build()
    from mllm_b200 import runtime
    return runtime


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("how", ["own rows", "shortened", "fewer rows"])
def test_every_sequence_reads_its_own_rows(rt, kv8, how):
    """The step is the one without shared_prefix, bit for bit; with the prefix read once from the first sequence the odd
    one's output would be another's."""
    from mllm_b200 import abi
    B, H, Hkv, D, P = 8, 32, 8, 128, 8192
    assert rt._shared_pays(B, P, Hkv, D, kv8)
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(B, h, 1, D, device="cuda", generator=g).bfloat16() for h in (H, Hkv, Hkv))
    pos = torch.tensor([P], device="cuda")
    out = []
    for prefix in (P, 0):
        c = (rt.PagedKVCache8 if kv8 else rt.PagedKVCache)(num_blocks=3 * P // 256 + 2 * B, num_kv_heads=Hkv, head_dim=D,
                                                           block_size=256, max_seqs=B, max_blocks_per_seq=P // 256 + 1)
        gp = torch.Generator(device="cuda").manual_seed(2)
        for pool in (c.k_pool, c.v_pool):
            pool.copy_(torch.randn(pool.shape, device="cuda", generator=gp))
        if kv8:
            c.k_exp.fill_(127)
            c.v_exp.fill_(127)
        c.set_lengths([P])
        for b in range(1, B):
            if b != 5 or how == "shortened":
                c.fork(0, b, P)
            elif how == "fewer rows":
                c.fork(0, b, P - 10)
        c.set_lengths([P] * B)
        if how == "shortened":
            c.release(5)
            c.fork(0, 5, P - 1)                          # its last block is its own ...
            c.set_lengths([P] * 5 + [P - 200] + [P] * 2)
            c.set_lengths([P] * B)                       # ... and what follows row P - 200 may be anything
        c.k_pool.view(torch.uint8 if kv8 else torch.bfloat16)[c.blocks_of(5)[-1], :, 60:] = 48
        c.shared_prefix = prefix
        out.append(rt.decode_step(q, k, v, c, pos, 1e6, Hkv))
    abi.call("mllm_attn_device_status", None)
    assert torch.equal(out[0], out[1])
