"""The loaders of tree attention's tcgen05 form over an 8-bit cache: short
stretches of tiles that come by one copy and piece by piece in every order (a
first tile that a ring's wrap divides, a last one that is part of a tile), so
that a slot of the codes' ring takes one kind after the other. Two hundred
pairs and more, so that the CTAs' shares hold whole pairs. Tolerance as in
test_tree_attention_gpu."""
import numpy as np
import pytest
import torch

import charlotte_b200 as cb
import test_tree_attention_gpu as T

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("slots", [320, 384, 520])
@pytest.mark.parametrize("tokens", [3, 20])
def test_whole_and_divided_tiles_take_turns(cuda, dim, slots, tokens):
    rng = np.random.default_rng(slots + dim + tokens)
    sequences, kv_heads = 36, 6
    # full rings begin anywhere (the wrap falls into any tile); short ones end inside their first to last tile
    lengths = [int(x) for x in rng.integers(slots, 4 * slots, 24)] + [int(x) for x in rng.integers(0, slots - tokens, sequences - 24)]
    T.Form.flags = cb.RUN_TENSOR
    try:
        call, out, _, want = T.run_case(rng, T.Q8, 2 * kv_heads, kv_heads, dim, lengths, None, tokens, None, slots)
        T.near(out, want)
        first = out.clone()
        for _ in range(20):
            out.fill_(float("nan"))
            call(flags=cb.RUN_TENSOR)
            torch.cuda.synchronize()
            assert torch.equal(out, first)
    finally:
        T.Form.flags = 0
    cb.check(cb.lib().cb_fault_check(None))
