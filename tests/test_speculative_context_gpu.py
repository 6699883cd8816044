"""Speculative decoding up to a model's context and not past it."""
import numpy as np
import pytest
import torch

import charlotte_b200 as cb
from charlotte_b200 import model as M
from charlotte_b200 import speculative as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["qwen3", "gemma3"])
@pytest.mark.parametrize("cache", [cb.CACHE_F16, cb.CACHE_Q8])
def test_the_last_positions_are_the_models_own(cuda, kind, cache):
    """Tokens up to the context's end, plain and with drafts that would pass it; one token more is refused."""
    context = 64
    m = M.synthesize(M.tiny(kind, context=context), seed=3)
    rng = np.random.default_rng(4)
    prompts = [[int(x) for x in rng.integers(0, 1000, n)] for n in (30, 5)]
    count = context - 30 + 1   # the longer prompt's last step stands at the last position
    plain = S.SpeculativeDecoder(m, 2, 1, cache)
    want, _ = plain.generate(prompts, count, drafter=lambda told, rows: ([], []))
    assert plain.lengths.tolist() == [context, 5 + count - 1]
    if cache == cb.CACHE_F16:
        d = M.Decoder(m)
        for p, w in zip(prompts, want):
            first = d.prefill(p)
            rest, _ = d.generate(count - 1)
            assert [int(first[0]), *map(int, rest)] == w
        d.close()
    told_all = [p + w + [1] * 40 for p, w in zip(prompts, want)]

    def deep(told, rows):   # what comes, then more
        known = next(t for t in told_all if t[:len(told)] == told)[len(told):][:rows - 1]
        return known, list(range(len(known)))
    for nodes in (6, 33):
        fast = S.SpeculativeDecoder(m, 2, nodes, cache)
        got, _ = fast.generate(prompts, count, drafter=deep)
        assert [g[:count] for g in got] == [w[:count] for w in want]
        assert int(fast.lengths.max()) <= context
        with pytest.raises(ValueError, match="past the context of 64"):
            fast.generate(prompts, count + 1, drafter=deep)


def test_steps_past_the_context_are_refused(cuda):
    m = M.synthesize(M.tiny("qwen3", context=32), seed=5)
    d = S.SpeculativeDecoder(m, 2, 8)
    with pytest.raises(ValueError, match="past the context of 32"):
        d.prefill([[1] * 34, [2, 3]])
    assert d.lengths.tolist() == [0, 0]
    d.prefill([[1] * 31, [2, 3]])          # entries 0 .. 29 of the first
    step = [([7, 8, 9], [-1, 0, 0]), ([3], [-1])]
    assert all(d.step(step))               # its rows at 30 and 31, two of them at 31
    d.lengths.copy_(torch.tensor([30, 2], dtype=torch.int32))
    before = d.lengths.tolist()
    with pytest.raises(ValueError, match="past the context of 32"):
        d.step([([7, 8, 9], [-1, 0, 1]), ([3], [-1])])
    assert d.lengths.tolist() == before
    d.lengths.copy_(torch.tensor([32, 2], dtype=torch.int32))
    with pytest.raises(ValueError, match="past the context of 32"):
        d.step([([7], [-1]), ([3], [-1])])
    new = d.step([([], []), ([3], [-1])])   # the full sequence takes no part
    assert new[0] == [] and len(new[1]) == 1


def test_trees_are_cut_at_a_depth():
    tokens, parents = [5, 6, 7, 8, 9], [-1, 0, 1, 0, 3]
    assert S.less_deep(tokens, parents, 3) == (tokens, parents)
    assert S.less_deep(tokens, parents, 2) == ([5, 6, 8], [-1, 0, 0])
    assert S.less_deep(tokens, parents, 1) == ([5], [-1])
    with pytest.raises(ValueError):
        S.less_deep([1, 2], [-1, 5], 3)
