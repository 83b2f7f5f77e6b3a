"""Penalties, biases and masks on logits against the rules computed token by token in 64 bits.  Needs a B200.

Tolerance: every fp32 step is off by at most 2^-24 of its result; six of them (scale, product, two differences, the
sum of biases and its addition) on numbers no larger than the sum of the magnitudes that enter.  Rounding to bf16 adds
2^-8 of the value."""
import numpy as np
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


def _pack(allow):
    B, V = allow.shape
    bits = np.zeros((B, -(-V // 32) * 32), np.uint8)
    bits[:, :V] = allow
    return torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view(np.int32).copy()).cuda()


def _reference(x, rows):
    """(result, magnitude of what entered) in 64 bits."""
    y, mag = x.astype(np.float64), np.abs(x.astype(np.float64))
    for b, r in enumerate(rows):
        V = x.shape[1]
        h = [t for t in r["history"]]
        for v in {t for t in h if 0 <= t < V}:
            y[b, v] = y[b, v] * r["rep"] if y[b, v] < 0 else y[b, v] / r["rep"]
            mag[b, v] = max(mag[b, v], abs(y[b, v]))
            c = sum(1 for t in h[r["start"]:] if t == v)
            y[b, v] -= c * r["freq"] + (c > 0) * r["pres"]
            mag[b, v] += c * abs(r["freq"]) + abs(r["pres"])
        for v, w in r["bias"]:
            if 0 <= v < V:
                y[b, v] += w
                mag[b, v] += abs(w)
        y[b, ~r["allow"]] = -np.inf
    return y, mag


def _tensors(rows, mask):
    B = len(rows)
    n, m = max(len(r["history"]) for r in rows), max(len(r["bias"]) for r in rows)
    hist = torch.full((B, max(n, 1)), 3, dtype=torch.int64)       # what lies behind a row's length is not looked at
    ids, vals = torch.full((B, max(m, 1)), 5, dtype=torch.int64), torch.full((B, max(m, 1)), float("nan"))
    for b, r in enumerate(rows):
        hist[b, :len(r["history"])] = torch.tensor(r["history"], dtype=torch.int64)
        if r["bias"]:
            ids[b, :len(r["bias"])] = torch.tensor([i for i, _ in r["bias"]])
            vals[b, :len(r["bias"])] = torch.tensor([w for _, w in r["bias"]])
    f = lambda k: torch.tensor([r[k] for r in rows], dtype=torch.float32).cuda()
    i = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
    kw = dict(history=hist.cuda(), history_lens=i([len(r["history"]) for r in rows]), output_start=i([r["start"] for r in rows]),
              repetition=f("rep"), presence=f("pres"), frequency=f("freq"), bias_ids=ids.cuda(), bias_values=vals.cuda(),
              bias_lens=i([len(r["bias"]) for r in rows]))
    if mask:
        kw["allowed"] = _pack(np.stack([r["allow"] for r in rows]))
    return kw


def _rows(rng, B, V, n, m, mask):
    rows = []
    f32 = lambda v: float(np.float32(v))
    for b in range(B):
        k = int(rng.integers(0, n + 1)) if b else n
        h = rng.integers(0, V, k)
        h[: k // 2] = rng.integers(0, min(V, 9), k // 2)          # many times the same few
        rng.shuffle(h)
        h = [int(t) for t in h]
        if k > 4:
            h[1], h[2] = -1, V                                    # ids that do not exist
        ids = [int(t) for t in rng.integers(0, V, int(rng.integers(0, m + 1)) if b else m)]
        if len(ids) > 3:
            ids[1], ids[2], ids[3] = ids[0], h[0] if h else 0, V + 7   # twice the same, one seen, one unknown
        allow = rng.random(V) < rng.random() if mask else np.ones(V, bool)
        if mask and b == 1:
            allow[:] = False                                      # a row that allows nothing
        rows.append(dict(history=h, start=int(rng.integers(0, k + 2)), rep=f32(rng.uniform(0.7, 1.6)), pres=f32(rng.uniform(-1, 1)),
                         freq=f32(rng.uniform(-0.5, 0.5)), bias=[(t, f32(rng.normal() * 3)) for t in ids], allow=allow))
    return rows


CASES = [
    # rows, vocabulary, history, biases, mask, dtype, elements between rows beyond the vocabulary
    (1, 1, 3, 2, False, "f32", 0),
    (2, 31, 40, 5, True, "bf16", 0),
    (3, 1000, 200, 20, True, "f32", 5),
    (4, 1025, 0, 30, True, "bf16", 3),
    (4, 4096, 300, 0, False, "f32", 0),
    (70, 5003, 100, 10, True, "bf16", 5),
    (2, 151936, 5000, 300, True, "f32", 0),
    (8, 151936, 20000, 1024, True, "bf16", 0),
    (300, 50001, 50, 4, True, "f32", 3),
]


@pytest.mark.parametrize("B,V,n,m,mask,dn,pad", CASES)
def test_against_the_rules(rt, B, V, n, m, mask, dn, pad):
    rng = np.random.default_rng(B * 1000 + V)
    rows = _rows(rng, B, V, n, m, mask)
    dt = torch.bfloat16 if dn == "bf16" else torch.float32
    full = (torch.randn(B, V + pad, generator=torch.Generator().manual_seed(1)) * 4).to(dt)
    full[:, 0] = float("-inf")
    x = full.cuda()[:, :V]
    y, mag = _reference(full[:, :V].float().numpy(), rows)
    kw = _tensors(rows, mask)
    got = rt.apply_logit_rules(x, **kw)
    _status_ok()
    assert torch.equal(x.cpu(), full[:, :V])
    g = got.float().cpu().numpy().astype(np.float64)
    inf = np.isneginf(y)
    assert (np.isneginf(g) == inf).all()
    tol = 6 * 2.0 ** -24 * mag + (2.0 ** -8 * np.abs(y) if dn == "bf16" else 0)
    assert (np.abs(g - y)[~inf] <= tol[~inf]).all()
    # untouched tokens keep their bits, and the call works in place with the same result
    for b, r in enumerate(rows):
        t = r["allow"].copy()
        t[[v for v in r["history"] if 0 <= v < V]] = False
        t[[v for v, _ in r["bias"] if 0 <= v < V]] = False
        t = torch.from_numpy(t)
        assert torch.equal(got[b].cpu()[t], full[b, :V][t])
    keep = full.cuda()
    view = keep[:, :V]
    assert rt.apply_logit_rules(view, **kw, out=view) is view
    assert torch.equal(view, got) and torch.equal(keep[:, V:].cpu(), full[:, V:])


def test_each_rule_alone_and_none(rt):
    x = torch.randn(3, 2000, device="cuda")
    assert torch.equal(rt.apply_logit_rules(x), x)
    h = torch.tensor([[5, 5, 7], [1, 2, 3], [9, 9, 9]], device="cuda")
    n = torch.tensor([3, 2, 0], dtype=torch.int32, device="cuda")
    assert torch.equal(rt.apply_logit_rules(x, history=h, history_lens=n), x)
    half = torch.full((3,), 0.5, device="cuda")
    got = rt.apply_logit_rules(x, history=h, history_lens=n, frequency=half)
    want = x.clone()
    for b, v, c in ((0, 5, 2), (0, 7, 1), (1, 1, 1), (1, 2, 1)):
        want[b, v] -= 0.5 * c
    assert torch.equal(got, want)
    got = rt.apply_logit_rules(x, history=h, history_lens=n, presence=half,
                               output_start=torch.tensor([2, 0, 0], dtype=torch.int32, device="cuda"))
    want = x.clone()
    for b, v in ((0, 7), (1, 1), (1, 2)):
        want[b, v] -= 0.5
    assert torch.equal(got, want)
    none = torch.zeros(3, 63, dtype=torch.int32, device="cuda")
    assert torch.isneginf(rt.apply_logit_rules(x, allowed=none)).all()
    one = torch.tensor([[1 << 30] + [0] * 62], dtype=torch.int32, device="cuda").expand(3, 63)
    got = rt.apply_logit_rules(x, allowed=one)
    assert torch.equal(got[:, 30], x[:, 30]) and torch.isneginf(got).sum() == 3 * 1999
    empty = torch.zeros(3, 0, dtype=torch.int64, device="cuda")
    zero = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert torch.equal(rt.apply_logit_rules(x, history=empty, history_lens=zero, presence=half, bias_ids=empty,
                                            bias_values=empty.float(), bias_lens=zero), x)


def test_forbidden_numbers_that_are_none(rt):
    """A forbidden token is -inf whatever its logit; an allowed NaN or infinity stays, penalised or not."""
    x = torch.zeros(1, 64, device="cuda")
    x[0, 3], x[0, 4], x[0, 5], x[0, 6] = float("nan"), float("nan"), float("inf"), float("-inf")
    allow = np.ones((1, 64), bool)
    allow[0, 4] = False
    got = rt.apply_logit_rules(x, history=torch.tensor([[3, 4, 5, 6]], device="cuda"),
                               history_lens=torch.tensor([4], dtype=torch.int32, device="cuda"),
                               repetition=torch.tensor([1.2], device="cuda"), allowed=_pack(allow))[0].cpu()
    assert torch.isnan(got[3]) and torch.isneginf(got[4]) and torch.isposinf(got[5]) and torch.isneginf(got[6])


def test_list_lengths_out_of_range_are_recorded(rt):
    from mllm_b200 import abi
    x = torch.randn(2, 500, device="cuda")
    h = torch.tensor([[5, 6], [5, 6]], device="cuda")
    r = torch.full((2,), 2.0, device="cuda")
    for bad in (-1, 3):
        got = rt.apply_logit_rules(x, history=h, history_lens=torch.tensor([bad, 1], dtype=torch.int32, device="cuda"),
                                   repetition=r)
        with pytest.raises(abi.MllmError) as e:
            _status_ok()
        assert e.value.status == 7
        assert torch.equal(got[1, 6:], x[1, 6:]) and got[1, 5] != x[1, 5]
    _status_ok()


def test_then_sampled_and_captured(rt):
    """Rules, then the sampler: only allowed tokens come out; the pair replays from a graph on new logits."""
    rng = np.random.default_rng(0)
    V, B = 5000, 6
    allow = rng.random((B, V)) < 0.02
    mask = _pack(allow)
    rep = torch.full((B,), 1.3, device="cuda")
    hist = torch.from_numpy(np.stack([rng.choice(np.flatnonzero(a), 30) for a in allow])).cuda()
    lens = torch.full((B,), 30, dtype=torch.int32, device="cuda")
    x = torch.randn(B, V, device="cuda") * 3
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rt.apply_logit_rules(x, history=hist, history_lens=lens, repetition=rep, frequency=rep, allowed=mask)
    for seed in range(5):
        x.copy_(torch.randn(B, V, device="cuda") * 3)
        graph.replay()
        want = rt.apply_logit_rules(x, history=hist, history_lens=lens, repetition=rep, frequency=rep, allowed=mask)
        assert torch.equal(y, want)
        greedy = rt.sample(y.clone(), use_greedy=True).tolist()
        drawn = rt.sample(y.clone(), temperature=1.5, top_p=0.9, seed=seed).tolist()
        for b in range(B):
            assert allow[b, greedy[b]] and allow[b, drawn[b]]
            assert greedy[b] == int(y[b].argmax())
    _status_ok()
