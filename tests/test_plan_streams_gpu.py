"""A plan's own workspace on streams other than the one it was made on."""
import math

import numpy as np
import pytest
import torch

import charlotte_b200 as cb
import speculative_reference as R
import test_tree_attention_gpu as T

pytestmark = pytest.mark.gpu

CYCLES = 200_000_000   # about a tenth of a second


def step(rng):
    """A long step whose parts meet in the workspace: its fields and its results."""
    fields, k, v = T.make_cache(rng, T.Q8, 1, 6001, 2, 128)
    q = rng.standard_normal((1, 1, 4, 128)).astype(np.float32)
    scale = float(np.float32(0.12))
    want = R.attention(q[0].astype(np.float64), k[0], v[0], R.visible(R.chain(1), 6000, 1, 6001, 0, 6001), 6001, scale / math.log2(math.e))
    out = torch.full((1, 1, 4, 128), float("nan"), device="cuda")
    return dict(cache=fields, query=torch.from_numpy(q).cuda(), out=out, lengths=T.u32([6000]), sequences=1, tokens=1,
                query_heads=4, max_keys=6001, scale_log2e=scale), want


def used_memory(need):
    """Leaves the allocator a block of that size which does not hold zeros."""
    block = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    del block


def test_a_first_call_on_another_stream(cuda):
    """The workspace is zeroed before any stream's first call, however long the plan's own stream has work."""
    fields, want = step(np.random.default_rng(1))
    need = cb.plan("tree_attention", **fields).workspace.numel()
    side = torch.cuda.Stream()
    used_memory(need)
    torch.cuda._sleep(CYCLES)
    call = cb.plan("tree_attention", **fields)
    call(stream=side)
    side.synchronize()
    T.near(fields["out"][0], want)
    torch.cuda.synchronize()
    call()
    torch.cuda.synchronize()
    T.near(fields["out"][0], want)


def test_a_plan_dropped_before_its_call_has_run(cuda):
    """Its workspace is not handed out again while another stream still works in it."""
    fields, want = step(np.random.default_rng(2))
    need = cb.plan("tree_attention", **fields).workspace.numel()
    side = torch.cuda.Stream()
    for as_current in (False, True):
        fields["out"].fill_(float("nan"))
        torch.cuda.synchronize()
        call = cb.plan("tree_attention", **fields)
        with torch.cuda.stream(side):
            torch.cuda._sleep(CYCLES)
            if as_current:
                call()
        if not as_current:
            call(stream=side)
        del call
        others = [torch.full((need,), 255, dtype=torch.uint8, device="cuda") for _ in range(3)]
        torch.cuda.synchronize()
        T.near(fields["out"][0], want)
        del others
