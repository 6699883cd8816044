"""The draw's settings of a speculative step: what a caller leaves out, and
the uniform numbers that a target with a temperature needs."""
import pytest
import torch

from charlotte_b200 import model as M
from charlotte_b200 import speculative as S

pytestmark = pytest.mark.gpu

FULL = dict(temperature=0.8, top_k=64, top_p=1.0, min_p=0.0)


def decoder():
    d = S.SpeculativeDecoder(M.synthesize(M.tiny("qwen3"), seed=5), 2, 3)
    d.prefill([[1, 2, 3, 4], [9, 8, 7]])
    return d


def test_settings_left_out_change_nothing(cuda):
    """A temperature alone is the whole list's draw at it."""
    step = [([4, 5, 6], [-1, 0, 0]), ([7], [-1])]
    drawn = set()
    for x in (0.02, 0.4, 0.7, 0.93, 0.999):
        u = torch.full((2, 3), x)
        want = decoder().step(step, FULL, u)
        assert decoder().step(step, dict(temperature=0.8), u) == want
        assert decoder().step(step, FULL | dict(min_p=0.0), u) == want
        drawn.add(want[1][-1])
    assert len(drawn) > 1   # the numbers do choose
    # a drafting model's settings likewise
    d = decoder()
    d.step([([4], [-1]), ([7], [-1])], FULL, torch.full((2, 3), 0.4))
    lists = d.candidates.view(2, 3, 64, 2).clone()
    u = torch.tensor([[0.3, 0.6, 0.9], [0.2, 0.5, 0.8]])
    want = decoder().step(step, FULL, u, lists, dict(FULL, temperature=0.5))
    assert decoder().step(step, FULL, u, lists, dict(temperature=0.5)) == want


def test_no_settings_are_greedy(cuda):
    step = [([4], [-1]), ([7], [-1])]
    want = decoder().step(step)
    assert decoder().step(step, {}) == want
    assert decoder().step(step, dict(temperature=0.0, top_p=0.3)) == want


def test_a_temperature_needs_uniform_numbers(cuda):
    d = decoder()
    before = d.lengths.tolist()
    with pytest.raises(ValueError, match="uniform"):
        d.step([([4], [-1]), ([7], [-1])], FULL)
    assert d.lengths.tolist() == before
