"""The 8-bit cache at the top of bf16's range.  Needs a B200."""
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
