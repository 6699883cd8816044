"""A speculative step whose kernels' waits ran out fails, commits nothing, and
can be taken again. The waits are made to run out by cb_debug_spin_limit(0),
as in test_failure_gpu: nothing faults or hangs, and every copy lands."""
import numpy as np
import pytest
import torch

import charlotte_b200 as cb
from charlotte_b200 import model as M
from charlotte_b200 import speculative as S

pytestmark = pytest.mark.gpu


@pytest.fixture
def short_waits():
    cb.check(cb.lib().cb_fault_check(None))
    yield lambda polls: cb.check(cb.lib().cb_debug_spin_limit(polls))
    cb.lib().cb_debug_spin_limit(-1)
    cb.lib().cb_fault_check(None)


def test_a_failed_step_is_an_error_and_commits_nothing(cuda, short_waits):
    """One row a step over a vocabulary whose head streams from HBM, so that some product's first wait does run out."""
    m = M.synthesize(M.qwen3_0_6b(context=64), seed=3)
    d, same = (S.SpeculativeDecoder(m, 1, 1) for _ in range(2))
    prompt = [int(x) for x in np.random.default_rng(4).integers(0, 1000, 12)]
    d.prefill([prompt])
    same.prefill([prompt])
    short_waits(0)
    with pytest.raises(cb.CharlotteError) as e:
        d.step([([prompt[-1]], [-1])])
    assert e.value.status == cb.ERROR_STEP and "bounded wait" in str(e.value)
    short_waits(-1)
    assert d.lengths.tolist() == [11]
    a, b = prompt[-1], prompt[-1]
    for _ in range(5):
        a, b = d.step([([a], [-1])])[0][-1], same.step([([b], [-1])])[0][-1]
        assert a == b
    assert d.lengths.tolist() == [16]


def test_a_failed_prompt_is_an_error_and_commits_nothing(cuda, short_waits):
    m = M.synthesize(M.qwen3_0_6b(context=64), seed=3)
    d = S.SpeculativeDecoder(m, 1, 1)
    d.prefill([[5, 6, 7]])
    short_waits(0)
    with pytest.raises(cb.CharlotteError):
        d.prefill([list(range(1, 12))])
    short_waits(-1)
    assert d.lengths.tolist() == [2]
    cb.check(cb.lib().cb_fault_check(None))


def test_logits_that_are_not_finite_are_an_error(cuda):
    """As the exact decoder's record says of its draw; the step is not committed, and others go on."""
    m = M.synthesize(M.tiny("qwen3"), seed=3)
    d = S.SpeculativeDecoder(m, 2, 3)
    d.prefill([[5, 6, 7], [8, 9]])
    step = [([7, 1], [-1, 0]), ([9], [-1])]
    gain = d.output_norm.clone()
    d.output_norm.fill_(float("nan"))
    with pytest.raises(cb.CharlotteError, match="not finite") as e:
        d.step(step)
    assert e.value.status == cb.ERROR_STEP
    assert d.lengths.tolist() == [2, 1]
    d.output_norm.copy_(gain)
    assert all(d.step(step))
