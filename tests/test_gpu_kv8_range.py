"""The 8-bit cache at the ends of its formats' ranges: weights far below the largest, in sums over very many rows, and
elements at the top of bf16's range.  Needs a B200.

Tolerances as in test_gpu_kv8.py; but a weight times scale is rounded to a half with the largest at 2^15, so one below
2^-29 of the largest (2^-14 as a half) is off by 2^-25 / 2^15 = 2^-40 of the largest at most.  A warp sums at most L / 4
rows in fp32, one product of 16 rows after another: L / 64 steps, each off by one unit in the last place of the sum of
magnitudes at most (2^-23; how the tensor cores round is not specified), and the weights in L / 32 additions a thread, each
rounded (2^-24): (L / 64) 2^-23 + (L / 32) 2^-24 = L 2^-28 of the mean magnitude."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

BF16_HALF, F16_HALF, F32 = 2.0 ** -8, 2.0 ** -11, 2.0 ** -18


@pytest.fixture(scope="module")
def rt(cuda_device):
    from mllm_b200 import build
    build.build()
    from mllm_b200 import runtime
    return runtime


def _status_ok():
    from mllm_b200 import abi
    abi.call("mllm_attn_device_status", None)


@pytest.mark.parametrize("L,B,top_exp", [(1 << 20, 300, 0), (1 << 18, 300, 8), (5000, 1, 8), (300, 1, 0)])
def test_one_dominant_row_among_many(rt, L, B, top_exp):
    """Each of the others has 2^-18 to 2^-29 of the dominant row's weight (and 2^-8 of its scale); together they are
    up to several times as much.  Enough sequences that a warp goes through most of one's rows behind that row."""
    H, D, at = 8, 64, 5
    c = rt.PagedKVCache8(num_blocks=-(-L // 1024), num_kv_heads=1, head_dim=D, block_size=1024, max_seqs=B)
    c.set_lengths([L])
    one = torch.zeros(D, device="cuda")
    one[0] = -1.0
    v = 1.0 + 0.5 * (torch.arange(D, device="cuda") % 5)
    c.k_pool.copy_(one.to(rt.FP8))
    c.v_pool.copy_(v.to(rt.FP8))
    c.k_exp.fill_(127)
    c.v_exp.fill_(127)
    blk, row = c.blocks_of(0)[at // 1024], at % 1024
    c.k_pool.view(torch.uint8)[blk, 0, row] = 0
    c.v_pool.view(torch.uint8)[blk, 0, row] = torch.full((D,), -(2.0 ** -top_exp), device="cuda").to(rt.FP8).view(torch.uint8)
    c.v_exp[blk, 0, row] = 127 + top_exp
    for b in range(1, B):
        c.fork(0, b, L)
    q = torch.zeros(B, H, D, device="cuda", dtype=torch.bfloat16)
    q[:, :, 0] = torch.tensor([100.0, 110, 120, 130, 139, 141, 150, 160])   # over 8: 18 to 28.9 in log2
    got = rt.decode_attention(q, c, 1, max_kv_len=L).view(B, H, D).double()
    _status_ok()
    k, vv = (x[0].double() for x in c.gather(0, L))
    s = q[0].double() @ k.T / math.sqrt(D)
    w = torch.softmax(s, -1)
    ref, mean_abs = w @ vv, w @ vv.abs()
    ev = torch.ones(L, device="cuda", dtype=torch.float64)
    ev[at] = 2.0 ** top_exp
    ds = F32 * (q[0].double().abs() @ k.abs().T).amax(-1, keepdim=True) / math.sqrt(D)
    small = 2.0 ** -40 * (w * ev).amax(-1, keepdim=True) * (vv.abs() / ev[:, None]).sum(0)
    tol = BF16_HALF * ref.abs() + (F16_HALF + 2 * ds + F32 + L * 2.0 ** -28) * mean_abs + small
    assert ((got - ref).abs() <= tol).all(), ((got - ref).abs() / tol).amax((0, 2))


def test_rows_at_the_top_of_the_range(rt):
    """A finite element stays finite: 256 * 2^120 and above are no bf16 numbers, so those that would be rounded there are
    stored as 240 * 2^120, the largest that is one."""
    D = 64
    top = float(torch.finfo(torch.bfloat16).max)
    rows = [top, -top, 1.9375 * 2.0 ** 127, 1.9296875 * 2.0 ** 127, 1.875 * 2.0 ** 127, 1.75 * 2.0 ** 127, 1.7421875 * 2.0 ** 127]
    T = len(rows) + 1
    x = torch.zeros(T, 1, D)
    for i, r in enumerate(rows):
        x[i, 0, 3], x[i, 0, 4], x[i, 0, 40] = r, 2.0 ** 124, -(2.0 ** 126)
    x[T - 1, 0, 3], x[T - 1, 0, 4], x[T - 1, 0, 50] = float("inf"), float("nan"), top
    v = x.bfloat16().cuda()
    want = v.double().clamp(-240 * 2.0 ** 120, 240 * 2.0 ** 120)
    scale = torch.exp2(torch.ceil(torch.log2(want.nan_to_num().abs().amax(-1, keepdim=True) / 448)))
    y = want / scale
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(1e-300))).clamp_min(-6) - 3)
    want = torch.round(y / step) * step * scale
    want[T - 1, 0, 3] = float("nan")
    q = torch.zeros(T, 1, D, dtype=torch.bfloat16, device="cuda")
    c = rt.PagedKVCache8(num_blocks=1, num_kv_heads=1, head_dim=D, block_size=128, max_seqs=1)
    c.reserve(0, T)
    cu, st = (torch.tensor(n, dtype=torch.int32, device="cuda") for n in ([0, T], [0]))
    # position 0 turns nothing and there is no norm: K is stored as it came, as V is, but that sin 0 times an element that
    # is not finite is NaN in the other one of its pair
    rt.qkv_epilogue_kv8(q, v, v, c, cu, st, torch.zeros(T, dtype=torch.int64, device="cuda"))
    k_want = want.clone()
    k_want[T - 1, 0, [3 + D // 2, 4 + D // 2]] = float("nan")
    for got, ref in zip(rt.kv8_read(c, torch.tensor([T], dtype=torch.int32, device="cuda"), T), (k_want, want)):
        got, ref = got[0, 0].double(), ref[:, 0]
        bad = torch.isnan(ref)
        assert torch.equal(torch.isnan(got), bad)
        assert (got[~bad] == ref[~bad]).all()
    _status_ok()


@pytest.mark.parametrize("power", [10, 20, 23, 24, 25, 27, 30, 60])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_of_any_size(rt, power, sign):
    """Scores so large that neighbouring numbers are far apart: one row has all the weight, and its V comes out as it is."""
    L, D = 400, 64
    c = rt.PagedKVCache8(num_blocks=4, num_kv_heads=2, head_dim=D, block_size=128, max_seqs=1)
    c.set_lengths([L])
    g = torch.Generator(device="cuda").manual_seed(power)
    k = torch.zeros(2, 512, D, device="cuda")
    k[:, :, 0] = torch.randint(-6, 6, (2, 512), device="cuda", generator=g) * 16.0
    top = [77, 301]
    for h in range(2):
        k[h, top[h], 0] = 112 * sign                     # the only one: the others are 16 and more below
    v = (torch.randn(2, 512, D, device="cuda", generator=g) * 100).clamp(-448, 448).to(rt.FP8).float()
    for pool, rows in ((c.k_pool, k), (c.v_pool, v)):
        for i, blk in enumerate(c.blocks_of(0)):
            pool[blk] = rows[:, 128 * i:128 * i + 128].to(rt.FP8)
    c.k_exp.fill_(127)
    c.v_exp.copy_(torch.randint(120, 130, c.v_exp.shape, device="cuda", generator=g, dtype=torch.int32).to(torch.uint8))
    q = torch.zeros(1, 8, D, device="cuda", dtype=torch.bfloat16)
    q[:, :, 0] = sign * 2.0 ** power / 8                 # scores of 14 to 2^power, in steps of 2^(power - 2)
    got = rt.decode_attention(q, c, 2, max_kv_len=L)[0, 0].view(2, 4, D).double()
    _status_ok()
    rows = c.gather(0, L)[1].double()
    for h in range(2):
        want = rows[h, top[h]]
        assert ((got[h] - want).abs() <= (BF16_HALF + F32) * want.abs()).all()
