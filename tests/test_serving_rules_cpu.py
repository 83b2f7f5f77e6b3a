"""A shared prefix and per-request rules in the continuous batcher: bookkeeping and checks, on CPU with a stand-in
model."""
import numpy as np
import pytest
import torch

from mllm_b200.serving import ContinuousBatcher, LogitRules, _pack_mask
from tests.test_serving_cpu import CountingModel


def test_requests_share_the_prefix_blocks():
    m = CountingModel()
    prefix = [3] * 300                                   # 2 full blocks and 44 rows
    bat = ContinuousBatcher(m, max_batch=2, num_blocks=9, block_size=128, prefix=prefix)
    assert m.calls == [(1, 300)] and bat.caches[0].free_blocks == 6
    specs = [([5, 6, 7], 4), ([100] * 90, 3), ([40], 130), ([9] * 129, 2), ([1, 2], 1)]
    ids = [bat.submit(p, n) for p, n in specs]
    while bat.waiting or bat.live:
        bat.step()
        lens = bat.caches[0].host_lengths()
        table = bat.caches[0].blocks_of(2)
        assert lens[2] == 300 and len(table) == 3
        for i, r in enumerate(bat.live):
            assert lens[i] == 300 + len(r.prompt) + len(r.tokens) - 1
            mine = bat.caches[0].blocks_of(i)
            assert mine[:2] == table[:2] and mine[2] != table[2]
    for rid, (p, n) in zip(ids, specs):
        assert bat.done[rid].tokens == [(p[-1] + k) % m.vocab for k in range(1, n + 1)]
    assert all(c.free_blocks == 6 and c.host_lengths() == [0, 0, 300] for c in bat.caches)


def test_a_request_must_fit_beside_the_prefix():
    bat = ContinuousBatcher(CountingModel(), max_batch=1, num_blocks=4, block_size=128, max_blocks_per_seq=4,
                            prefix=[1] * 250)            # holds 2 blocks, one of them shared
    bat.submit([2] * 100, 30)                            # rows 250 .. 379: a copy of block 1 and one more
    with pytest.raises(ValueError, match="longer"):
        bat.submit([2] * 200, 100)
    bat.run()
    assert bat.caches[0].free_blocks == 2


def test_rules_are_checked():
    for bad in (dict(repetition=0.0), dict(repetition=float("nan")), dict(presence=float("inf")),
                dict(bias={i: 1.0 for i in range(1025)})):
        with pytest.raises(ValueError):
            LogitRules(**bad)
    words = _pack_mask([v % 3 == 0 for v in range(70)], 70)
    assert words.dtype == np.int32 and words.shape == (3,)
    bits = [(int(words[v // 32]) >> (v % 32)) & 1 for v in range(96)]
    assert bits == [int(v % 3 == 0 and v < 70) for v in range(96)]
    with pytest.raises(ValueError, match="truth value per token"):
        _pack_mask([True] * 5, 6)
    bat = ContinuousBatcher(CountingModel(), max_batch=1, num_blocks=2, block_size=128)
    bat.submit([1], 2, rules=LogitRules(presence=1.0))
    with pytest.raises(RuntimeError, match="CUDA"):      # the rules run on the device only
        bat.run()
