"""The serving step with its newer parts in place: a prefix that the batch shares, 8-bit caches and per-request
rules, alone and together, through the continuous batcher.  Needs a B200."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a GPU", allow_module_level=True)

from mllm_b200 import abi  # noqa: E402
from mllm_b200 import runtime as rt  # noqa: E402
from mllm_b200.serving import ContinuousBatcher, DecoderModel, DecoderShape, LogitRules, apply_rules  # noqa: E402
from tests.test_gpu_serving import _solo_logits  # noqa: E402

SHAPE = DecoderShape(vocab=2048, hidden=1024, layers=3, heads=8, kv_heads=2, head_dim=128, intermediate=2048)


def _run(model, prompts, news, **kw):
    bat = ContinuousBatcher(model, max_batch=3, num_blocks=24, block_size=128, record_logits=True, **kw)
    free = bat.caches[0].free_blocks
    ids = [bat.submit(p, n) for p, n in zip(prompts, news)]
    out = bat.run()
    assert all(c.free_blocks == free for c in bat.caches)
    abi.call("mllm_attn_device_status", None)
    return [out[i] for i in ids], [torch.stack(bat.done[i].logits) for i in ids], bat


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("plen", [1, 128, 300])
def test_shared_prefix_matches_solo_runs(plen, graphs):
    """As the batcher without a prefix is tested: against each request alone, prefix and prompt in one contiguous cache,
    within 0.03 of the largest logit (bf16 through three layers), and the greedy token where the margin is clear."""
    model = DecoderModel(SHAPE, seed=3)
    rng = np.random.default_rng(plen)
    prefix = rng.integers(0, SHAPE.vocab, plen).tolist()
    prompts = [rng.integers(0, SHAPE.vocab, n).tolist() for n in (5, 130, 37, 1, 64)]
    toks, logits, bat = _run(model, prompts, [12, 5, 20, 16, 10], prefix=prefix, graphs=graphs)
    assert (bat.graph_steps > 5) == graphs
    agree = total = 0
    for p, t, got in zip(prompts, toks, logits):
        ref = _solo_logits(model, prefix + p, t)
        scale = ref.abs().max().item()
        np.testing.assert_allclose(got.numpy(), ref.numpy(), atol=0.03 * scale, rtol=0)
        top2 = ref.topk(2, dim=-1).values
        clear = (top2[:, 0] - top2[:, 1]) > 0.02 * scale
        agree += int((ref.argmax(-1) == torch.tensor(t))[clear].sum())
        total += int(clear.sum())
    assert total > 0 and agree == total


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("plen", [1, 128, 300])
def test_shared_prefix_read_once_matches_solo_runs(plen, graphs, monkeypatch):
    """The same through decode_attention_shared, which decode_step leaves aside for batches and prefixes this small."""
    calls = []
    shared = rt.decode_attention_shared
    monkeypatch.setattr(rt, "_SHARED_MIN_BYTES", 0)
    monkeypatch.setattr(rt, "decode_attention_shared", lambda *a: calls.append(a[3]) or shared(*a))
    test_shared_prefix_matches_solo_runs(plen, graphs)
    assert calls and set(calls) == {plen}


@pytest.mark.parametrize("B,prefix,used", [(4, 8192, True), (1, 8192, False), (4, 512, False)])
def test_a_step_reads_the_prefix_once_where_that_pays(B, prefix, used, monkeypatch):
    """decode_step on a cache with shared_prefix set against the step without it: bf16 outputs of two summation orders
    (each within 2^-8 of the value and 2^-8 of the mean of |v| < 1, for P), twice."""
    H, Hkv, D = 32, 8, 128
    g = torch.Generator(device="cuda").manual_seed(B)
    calls = []
    shared = rt.decode_attention_shared
    monkeypatch.setattr(rt, "decode_attention_shared", lambda *a: calls.append(a[3]) or shared(*a))
    c = rt.PagedKVCache(num_blocks=prefix // 256 + 2 * B + 1, num_kv_heads=Hkv, head_dim=D, block_size=256, max_seqs=B,
                        max_blocks_per_seq=prefix // 256 + 2)
    c.k_pool.normal_(generator=g)
    c.v_pool.uniform_(-1, 1, generator=g)
    c.set_lengths([prefix])
    for b in range(1, B):
        c.fork(0, b, prefix)
    q, k, v = (torch.randn(B, h, 1, D, device="cuda", generator=g).bfloat16() for h in (H, Hkv, Hkv))
    v.clamp_(-1, 1)
    pos = torch.tensor([prefix], device="cuda")
    got = []
    for shared_rows in (prefix, 0):
        c.shared_prefix = shared_rows
        c.set_lengths([prefix] * B)
        got.append(rt.decode_step(q, k, v, c, pos, 1e6, Hkv).double())
    abi.call("mllm_attn_device_status", None)
    assert calls == ([prefix] if used else [])
    assert ((got[0] - got[1]).abs() <= 2 * 2.0 ** -8 * (1 + got[1].abs())).all()


@pytest.mark.parametrize("prefix_len", [0, 200])
def test_8bit_caches_batched_and_alone(prefix_len):
    """8-bit caches: requests side by side (steps from graphs) against one at a time, eager.  Another order of additions in
    the projections can move a cached element by one e4m3 step, so up to the first token that differs (a near-tie)
    the logits agree to the same 0.03 of the largest."""
    model = DecoderModel(SHAPE, seed=4, kv8=True)
    rng = np.random.default_rng(1)
    prefix = rng.integers(0, SHAPE.vocab, prefix_len).tolist()
    prompts = [rng.integers(0, SHAPE.vocab, n).tolist() for n in (20, 200, 3, 129, 64)]
    news = [20, 15, 25, 12, 18]
    toks, logits, bat = _run(model, prompts, news, prefix=prefix)
    assert bat.graph_steps > 5
    compared = 0
    for p, n, t, got in zip(prompts, news, toks, logits):
        solo_t, solo_l, _ = _run(model, [p], [n], prefix=prefix, graphs=False)
        scale = solo_l[0].abs().max().item()
        for k in range(n):
            np.testing.assert_allclose(got[k].numpy(), solo_l[0][k].numpy(), atol=0.03 * scale, rtol=0)
            compared += 1
            if t[k] != solo_t[0][k]:
                top2 = solo_l[0][k].topk(2).values
                assert float(top2[0] - top2[1]) < 0.03 * scale
                break
    assert compared > 50


def test_8bit_caches_with_the_prefix_read_once(monkeypatch):
    """The same with the prefix read once, which decode_step leaves aside for batches and prefixes this small."""
    calls = []
    shared = rt.decode_attention_shared
    monkeypatch.setattr(rt, "_SHARED_MIN_BYTES8", 0)
    monkeypatch.setattr(rt, "_SHARED_MIN_BATCH8", 1)
    monkeypatch.setattr(rt, "decode_attention_shared", lambda *a: calls.append(a[3]) or shared(*a))
    test_8bit_caches_batched_and_alone(200)
    assert calls and set(calls) == {200}


@pytest.mark.parametrize("kv8,prefix_len", [(False, 0), (True, 150), (False, 150)])
def test_rules_hold_for_their_request_only(kv8, prefix_len):
    """A grammar, penalties and biases on some of the requests: the picked tokens are the greedy ones of the recorded
    logits under the rules computed in 64 bits; requests without rules pick the plain greedy token."""
    model = DecoderModel(SHAPE, seed=6, kv8=kv8)
    rng = np.random.default_rng(2)
    prefix = rng.integers(0, SHAPE.vocab, prefix_len).tolist()

    def even_then_odd(tokens):
        return (np.arange(SHAPE.vocab) + len(tokens)) % 2 == 0
    rules = [None, LogitRules(allowed=even_then_odd), LogitRules(repetition=1.7, presence=0.5, frequency=0.25),
             LogitRules(bias={7: 50.0, 8: -5.0}), LogitRules(repetition=1.2, frequency=1.0, bias={9: 1.0}, allowed=even_then_odd)]
    bat = ContinuousBatcher(model, max_batch=3, num_blocks=24, block_size=128, record_logits=True, prefix=prefix)
    prompts = [rng.integers(0, SHAPE.vocab, n).tolist() for n in (20, 100, 3, 64, 7)]
    ids = [bat.submit(p, 14, rules=r) for p, r in zip(prompts, rules)]
    bat.run()
    abi.call("mllm_attn_device_status", None)
    for i, p, r in zip(ids, prompts, rules):
        req = bat.done[i]
        for k, (t, row) in enumerate(zip(req.tokens, req.logits)):
            x = row.double().numpy().copy()
            if r is not None:
                made = req.tokens[:k]
                for v in set(prefix + p + made):
                    x[v] = x[v] * r.repetition if x[v] < 0 else x[v] / r.repetition
                    x[v] -= made.count(v) * r.frequency + (v in made) * r.presence
                for v, b in r.bias.items():
                    x[v] += b
                if r.allowed:
                    x[~r.allowed(made)] = -np.inf
            # fp32 arithmetic on numbers below 100: six steps of 2^-24
            assert x[t] >= x.max() - 6 * 2.0 ** -24 * 100, (i, k)
    assert bat.done[ids[3]].tokens == [7] * 14


def test_apply_rules_on_rows_without_any():
    x = torch.randn(2, 100, device="cuda")
    assert torch.equal(apply_rules(x, [None, LogitRules()], [[], [1]], [[], []]), x)
