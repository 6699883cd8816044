"""Tokens that are not the model's, in speculative decoding."""
import pytest
import torch

from charlotte_b200 import model as M
from charlotte_b200 import speculative as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("token", [1000, 5000, -1])
def test_a_sequence_holds_the_models_tokens(cuda, token):
    d = S.SpeculativeDecoder(M.synthesize(M.tiny("qwen3"), seed=5), 2, 4)   # a vocabulary of 1,000
    with pytest.raises(ValueError, match="vocabulary"):
        d.prefill([[1, token, 3], [2, 3]])
    with pytest.raises(ValueError, match="vocabulary"):
        d.prefill([[1, 2, token], [2, 3]])
    assert d.lengths.tolist() == [0, 0]
    d.prefill([[1, 2, 3], [2, 3]])
    with pytest.raises(ValueError, match="vocabulary"):
        d.step([([3], [-1]), ([token], [-1])])
    assert d.lengths.tolist() == [2, 1]


def test_a_drafted_one_is_refused_and_its_siblings_are_not(cuda):
    """A drafting model may have more tokens than the target."""
    m = M.synthesize(M.tiny("qwen3"), seed=5)
    d, plain = (S.SpeculativeDecoder(m, 1, 4) for _ in range(2))
    d.prefill([[1, 2, 3]])
    plain.prefill([[1, 2, 3]])
    first = plain.step([([3], [-1])])[0][0]
    second = plain.step([([first], [-1])])[0][0]
    assert d.step([([3, 4095, first, 7], [-1, 0, 0, 1])])[0] == [first, second]
