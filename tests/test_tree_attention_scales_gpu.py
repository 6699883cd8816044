"""Tree attention over an 8-bit cache whose value scales differ by many orders
of magnitude: a visible key that has no weight in a row costs that row no
accuracy, however large its values, and a row in which it has all the weight
is as accurate beside it. Rows are compared one by one, each norm-wise at
the 5e-6 that test_tree_attention_gpu derives: operands keep 22 bits relative
to a row's largest weight times scale."""
import math

import numpy as np
import pytest
import torch

import charlotte_b200 as cb
import speculative_reference as R
import test_tree_attention_gpu as T

pytestmark = pytest.mark.gpu


def case(rng, heads, kv_heads, dim, length, tokens, ratio, at, favour, flags):
    """One sequence with a key at entry `at` whose values are `ratio` times the others'. Its score is 30 + log2(ratio) below
    the others' range in rows of favour[row] < 0, so that it weighs 2^-30 there, and as much above it in the others."""
    slots = length + tokens
    fields, k, v = T.make_cache(rng, T.Q8, 1, slots, kv_heads, dim)
    scale_log2e = float(np.float32(math.log2(math.e) / math.sqrt(dim)))
    signs = rng.choice([-1, 1], (kv_heads, dim))
    q = rng.standard_normal((tokens, heads, dim))
    group = heads // kv_heads
    along = np.repeat(signs, group, 0) / math.sqrt(dim)
    q -= (q * along).sum(-1, keepdims=True) * along
    q += np.asarray(favour).reshape(tokens, heads)[..., None] * 4.0 * along
    q = q.astype(np.float32)
    others = np.abs(np.einsum("thd,ehd->teh", q[:, ::group].astype(np.float64), k[0])).max() * scale_log2e * 1.5
    gap = 30.0 + math.log2(ratio) + others
    # a key of codes ±127 along the signs: its product with a row is favour · 4 · size
    size = gap / (4.0 * scale_log2e)
    key_scale = np.float32(size / (127 * math.sqrt(dim)))
    for h in range(kv_heads):
        fields["key"][0, at, h] = torch.from_numpy((128 + 127 * signs[h]).astype(np.uint8)).cuda()
        fields["key_scale"][0, h, at] = float(key_scale)
        k[0, at, h] = 127.0 * signs[h] * float(key_scale)
        big = np.float32(float(fields["value_scale"][0, h, at]) * ratio)
        v[0, at, h] *= float(big) / float(fields["value_scale"][0, h, at])
        fields["value_scale"][0, h, at] = float(big)
    out = torch.full((1, tokens, heads, dim), float("nan"), device="cuda")
    cb.plan("tree_attention", cache=fields, query=torch.from_numpy(q).cuda(), out=out, lengths=T.u32([length]), sequences=1,
            tokens=tokens, query_heads=heads, max_keys=slots, scale_log2e=scale_log2e)(flags=flags)
    torch.cuda.synchronize()
    want = R.attention(q.astype(np.float64), k[0], v[0], R.visible(R.chain(tokens), length, tokens, slots, 0, slots), slots,
                       scale_log2e / math.log2(math.e))
    got = out[0].double().cpu().numpy()
    error = np.linalg.norm(got - want, axis=-1) / np.linalg.norm(want, axis=-1)
    assert np.isfinite(got).all()
    return error


@pytest.mark.parametrize("flags", [0, cb.RUN_TENSOR])
@pytest.mark.parametrize("heads,kv_heads,dim,tokens", [(8, 2, 128, 1), (16, 4, 64, 12), (16, 8, 128, 32), (8, 2, 256, 8)])
@pytest.mark.parametrize("ratio", [1.0, 1e3, 1e5, 1e9, 1e20, 1e30])
@pytest.mark.parametrize("at", [3, 700, 2500])
def test_a_weightless_key_of_large_values(cuda, flags, heads, kv_heads, dim, tokens, ratio, at):
    rng = np.random.default_rng(int(math.log2(ratio)) + at)
    error = case(rng, heads, kv_heads, dim, 2600, tokens, ratio, at, -np.ones((tokens, heads)), flags)
    assert error.max() <= 5e-6, error.max()


@pytest.mark.parametrize("flags", [0, cb.RUN_TENSOR])
@pytest.mark.parametrize("heads,kv_heads,dim,tokens", [(8, 2, 128, 1), (16, 4, 64, 12), (16, 8, 128, 32), (8, 2, 256, 8)])
@pytest.mark.parametrize("ratio", [1.0, 1e3, 1e9, 1e30])
@pytest.mark.parametrize("at", [3, 700, 2500])
def test_some_rows_have_nothing_else(cuda, flags, heads, kv_heads, dim, tokens, ratio, at):
    """The key has all the weight in a third of the rows and none in their neighbours."""
    rng = np.random.default_rng(int(math.log2(ratio)) + at + 1)
    favour = np.where(rng.random((tokens, heads)) < 1 / 3, 1.0, -1.0)
    favour[0, 0] = 1.0
    error = case(rng, heads, kv_heads, dim, 2600, tokens, ratio, at, favour, flags)
    assert error.max() <= 5e-6, error.max()
