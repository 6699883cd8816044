"""Tree attention whose waits run out (cb_debug_spin_limit): the tcgen05 form
reports it in the fault word, returns, and leaves its workspace ready: the same
call then gives the right results. Nothing faults or hangs: copies on their
way land before the kernel leaves."""
import ctypes

import numpy as np
import pytest
import torch

import charlotte_b200 as cb
import test_tree_attention_gpu as T

pytestmark = pytest.mark.gpu


@pytest.fixture
def short_waits():
    cb.check(cb.lib().cb_fault_check(None))
    yield lambda polls: cb.check(cb.lib().cb_debug_spin_limit(polls))
    cb.lib().cb_debug_spin_limit(-1)
    cb.lib().cb_fault_check(None)


@pytest.mark.parametrize("fmt", [T.F16, T.Q8])
@pytest.mark.parametrize("heads,kv_heads,dim,tokens", [(8, 2, 64, 10), (4, 2, 128, 20), (4, 2, 256, 9)])
@pytest.mark.parametrize("polls", [0, 1, 5])
def test_a_wait_that_runs_out_is_reported(cuda, short_waits, fmt, heads, kv_heads, dim, tokens, polls):
    rng = np.random.default_rng(dim)
    T.Form.flags = cb.RUN_TENSOR
    try:
        lengths = [3000, 700, 129, 5000]   # whole and divided tiles, pairs within a CTA's share and over several
        call, out, _, want = T.run_case(rng, fmt, heads, kv_heads, dim, lengths, None, tokens, None, 5100)
    finally:
        T.Form.flags = 0
    T.near(out, want)
    cb.check(cb.lib().cb_fault_check(None))
    first = out.clone()
    short_waits(polls)
    call(flags=cb.RUN_TENSOR)
    torch.cuda.synchronize()
    bits = ctypes.c_uint(0)
    status = cb.lib().cb_fault_check(ctypes.byref(bits))
    if polls == 0:   # with a poll or more every wait may yet have been met
        assert status == cb.ERROR_STEP and bits.value & 1 and "bounded wait" in cb.last_error()
    short_waits(-1)
    for _ in range(2):
        out.fill_(float("nan"))
        call(flags=cb.RUN_TENSOR)
        torch.cuda.synchronize()
        assert torch.equal(out, first)
    cb.check(cb.lib().cb_fault_check(None))
