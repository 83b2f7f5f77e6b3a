"""Requests whose rules fail, and steps that raise, in the continuous batcher.  On CPU with a stand-in model and the
rules' device call stood in for by the same on the host."""
import numpy as np
import pytest
import torch

from mllm_b200 import runtime as rt
from mllm_b200.serving import ContinuousBatcher, LogitRules
from tests.test_serving_cpu import CountingModel, PackedCountingModel


class PackedBehindPrefix(PackedCountingModel):
    def forward_packed(self, ids, q_lens, caches):
        lens = caches[0].host_lengths()
        for c in caches:
            c.advance(list(q_lens), batch=len(q_lens))
        assert all(c.host_lengths() == [a + b for a, b in zip(lens, q_lens)] for c in caches)
        last = torch.tensor([sum(q_lens[:b + 1]) - 1 for b in range(len(q_lens))])
        logits = torch.zeros(len(q_lens), self.vocab)
        logits[torch.arange(len(q_lens)), (ids[last] + 1) % self.vocab] = 1.0
        return logits


@pytest.fixture
def host_rules(monkeypatch):
    """Masks and biases of apply_logit_rules on the host."""
    def rules(logits, allowed=None, bias_ids=None, bias_values=None, bias_lens=None, **_):
        out = logits.clone()
        if bias_ids is not None:
            for b in range(len(out)):
                for j in range(int(bias_lens[b])):
                    out[b, int(bias_ids[b, j])] += bias_values[b, j]
        if allowed is not None:
            v = torch.arange(logits.shape[1])
            out[((allowed[:, v // 32] >> (v % 32)) & 1) == 0] = float("-inf")
        return out
    monkeypatch.setattr(rt, "apply_logit_rules", rules)


def _everything(tokens):
    return np.ones(CountingModel.vocab, dtype=bool)


def _run(specs, model=None, **kw):
    """specs: (prompt, new tokens, rules); the batcher after a run in which every row and block came back."""
    bat = ContinuousBatcher(model or CountingModel(), max_batch=2, num_blocks=10, block_size=128, **kw)
    free = bat.caches[0].free_blocks
    lens = bat.caches[0].host_lengths()
    ids = [bat.submit(p, n, rules=r) for p, n, r in specs]
    out = bat.run()
    assert not bat.live and not bat.waiting and sorted(out) == ids
    assert all(c.free_blocks == free and c.host_lengths() == lens for c in bat.caches)
    return [bat.done[i] for i in ids]


def _counted(p, n):
    return [(p[-1] + k) % CountingModel.vocab for k in range(1, n + 1)]


def _raises(after):
    def allowed(tokens):
        if len(tokens) == after:
            raise KeyError("no such state")
        return _everything(tokens)
    return allowed


def _wrong_shape(after):
    return lambda tokens: [True] * 5 if len(tokens) == after else _everything(tokens)


@pytest.mark.parametrize("model", [CountingModel, PackedBehindPrefix])
@pytest.mark.parametrize("prefix", [[], [3] * 300])
@pytest.mark.parametrize("after", [0, 2])
@pytest.mark.parametrize("failing,error", [(_raises, KeyError), (_wrong_shape, ValueError)])
def test_rules_that_fail_end_their_request_only(host_rules, failing, error, after, prefix, model):
    """At the first token (the prompt's) and in the middle of the answer; beside, before and behind others."""
    good = LogitRules(allowed=_everything)
    specs = [([5, 6, 7], 4, None), ([100] * 90, 6, LogitRules(allowed=failing(after))), ([40], 9, good),
             ([9] * 129, 3, LogitRules(allowed=failing(after))), ([1, 2], 1, None)]
    done = _run(specs, model(), prefix=prefix)
    for r, (p, n, rules) in zip(done, specs):
        fails = rules is not None and rules is not good
        assert r.tokens == _counted(p, after if fails else n)
        assert type(r.error) is error if fails else r.error is None


@pytest.mark.parametrize("at", ["prefill", "decode", "rules"])
@pytest.mark.parametrize("prefix", [[], [3] * 130])
def test_a_step_that_raises_can_be_taken_again(host_rules, monkeypatch, at, prefix):
    """Whatever else raises in a step (here once, in every place in turn) leaves rows, blocks and requests as they were."""
    class Failing(CountingModel):
        left = 0

        def forward(self, ids, positions, caches):
            if self.left and (at == "decode") == (ids.shape[1] == 1) and at != "rules":
                self.left -= 1
                caches[0].advance(ids.shape[1], batch=ids.shape[0])    # some of the layers were through
                raise MemoryError("device memory")
            return super().forward(ids, positions, caches)
    m = Failing()
    host = rt.apply_logit_rules

    def rules(*a, **kw):
        if at == "rules" and m.left:
            m.left -= 1
            raise MemoryError("device memory")
        return host(*a, **kw)
    monkeypatch.setattr(rt, "apply_logit_rules", rules)
    bat = ContinuousBatcher(m, max_batch=2, num_blocks=10, block_size=128, prefix=prefix)
    free = bat.caches[0].free_blocks
    specs = [([5, 6, 7], 4), ([100] * 90, 3), ([40, 41], 6), ([9] * 129, 2)]
    ids = [bat.submit(p, n, rules=LogitRules(allowed=_everything)) for p, n in specs]
    raised = 0
    while bat.waiting or bat.live:
        m.left = 1
        try:
            bat.step()
        except MemoryError:
            raised += 1
            for i, r in enumerate(bat.live):
                assert all(c.host_lengths()[i] == len(prefix) + len(r.prompt) + len(r.tokens) - 1 for c in bat.caches)
        m.left = 0
        bat.step()
    assert raised >= 2
    for i, (p, n) in zip(ids, specs):
        assert bat.done[i].tokens == _counted(p, n) and bat.done[i].error is None
    assert all(c.free_blocks == free for c in bat.caches)


def _nothing(after):
    return lambda tokens: _everything(tokens) & (len(tokens) != after)


@pytest.mark.parametrize("after", [0, 2])
def test_a_request_whose_rules_leave_no_token_ends(host_rules, after):
    """An empty mask, or biases of -inf on all that the mask allows: nothing may be picked, token 0 no more than others."""
    few = np.zeros(CountingModel.vocab, dtype=bool)
    few[[0, 7, 300]] = True
    banned = LogitRules(bias={0: -np.inf, 7: -np.inf, 300: -np.inf, 5: 1.0},
                        allowed=lambda tokens: few if len(tokens) == after else _everything(tokens))
    specs = [([40], 5, None), ([5, 6, 7], 4, LogitRules(allowed=_nothing(after))), ([100] * 90, 3, LogitRules(allowed=_everything)),
             ([600], 4, banned), ([60], 4, LogitRules(bias={61: -np.inf}))]
    done = _run(specs)
    for r, (p, n, _) in list(zip(done, specs))[:3:2]:
        assert r.tokens == _counted(p, n) and r.error is None
    for r, tokens in ((done[1], _counted([7], after)), (done[3], [5] * after)):   # 5: a tie with the model's choice, and lower
        assert r.tokens == tokens and type(r.error) is ValueError and "no token" in str(r.error)
    assert done[4].error is None and len(done[4].tokens) == 4 and 61 not in done[4].tokens   # a ban that leaves others


def test_a_bias_is_a_number():
    with pytest.raises(ValueError, match="bias"):
        LogitRules(bias={3: float("nan")})
    LogitRules(bias={3: -float("inf"), 4: float("inf")})
