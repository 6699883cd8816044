"""Verification (cb_verify_run) of drafts that are sure of a token: a draft
whose first candidate's probability rounds to one leaves its siblings a mass
of 1e-6 to 1e-13, by which theirs are normalized once it is refused.

The 64-bit statement here takes that mass as the sum of what is left, never
as one less what is gone. Whole numbers are equal except where a decision lies
within 1e-5 of falling the other way, as in test_verify_gpu: the kernel's
probabilities carry f32's rounding, relative to themselves."""
import numpy as np
import pytest
import torch

import charlotte_b200 as cb
import speculative_reference as R
import test_verify_gpu as V

pytestmark = pytest.mark.gpu


def peaked(rng, tokens, gap, temperature):
    """A draft's list over `tokens` in their order: the first's logit `gap` (after the temperature) above the others'."""
    logits = np.zeros(64)
    logits[1:] = -(gap + np.concatenate([[0.0], np.cumsum(rng.exponential(0.15, 62))]))
    return np.stack([(logits * temperature).astype(np.float32).view(np.uint32), tokens.astype(np.uint32)], -1)


def walk(candidates, draft, ids, u, masks, target, draft_settings):
    """One sequence: (path, sampled token, margin)."""
    parent = [-1] + [(int(m) & ((1 << i) - 1)).bit_length() - 1 for i, m in enumerate(masks) if i]
    at, path, margin = 0, [0], 1.0
    while True:
        tokens, q_tokens = candidates[at, :, 1], draft[at, :, 1]
        r = R.distribution(candidates[at, :, 0], tokens, **target)
        q = R.distribution(draft[at, :, 0], q_tokens, **draft_settings)
        nxt = None
        for i in (i for i in range(1, len(ids)) if parent[i] == at):
            given = q[q_tokens == ids[i]].sum()
            if not given > 0:
                continue
            left = q.sum()   # the mass of the tokens not refused
            p = r[tokens == ids[i]].sum()
            margin = min(margin, abs(u[i] * given / left - p))
            if u[i] * given / left < p:
                nxt = i
                break
            rest = np.maximum(r - np.array([q[q_tokens == t].sum() for t in tokens]) / left, 0.0)
            if rest.sum() > 0:
                margin = min(margin, rest.sum())
                r = rest / rest.sum()
            q = np.where(q_tokens == ids[i], 0.0, q)
        if nxt is None:
            break
        at = nxt
        path.append(at)
    running = np.cumsum(r)
    goal = u[0] * running[-1]
    margin = min(margin, np.abs(running[r > 0] - goal).min())
    return path, int(tokens[int(np.argmax((running > goal) & (r > 0)))]), margin


@pytest.mark.parametrize("gap", [3.0, 11.0, 14.0, 17.5, 18.0, 22.0, 30.0, 60.0])
@pytest.mark.parametrize("temperature", [1.0, 0.6, 0.25])
def test_siblings_of_a_sure_token(cuda, gap, temperature):
    """A root and its four children, then the second's two: the first drafts the token that the draft is sure of, the
    others what it gives next to nothing."""
    rng = np.random.default_rng(int(gap * 10) + int(temperature * 100))
    s, tokens = 256, 7
    masks = np.tile(np.array([1, 3, 5, 9, 17, 0b100101, 0b1000101], np.uint64), (s, 1))
    parent = [0, 0, 0, 0, 0, 2, 2]
    candidates = V.lists(rng, (s, tokens), spread=0.6)
    draft, ids = np.empty_like(candidates), np.zeros((s, tokens), np.uint32)
    for b in range(s):
        for i in range(tokens):
            order = np.concatenate([rng.permutation(6), 6 + rng.permutation(58)])   # sure of one of the likely tokens
            draft[b, i] = peaked(rng, candidates[b, i, order, 1], gap, temperature)
        ids[b, 1:5] = draft[b, 0, [0, 1, 2, 3], 1]
        ids[b, 5:7] = draft[b, 2, [0, 1], 1]
    u = rng.random((s, tokens)).astype(np.float32)
    target, ds = V.settings(0.9, top_k=40), V.settings(temperature)
    path, kept, sampled = V.run(candidates, draft, ids, u, masks, None, target, ds)
    sure = 0
    for b in range(s):
        want, token, margin = walk(candidates[b], draft[b], ids[b], u[b].astype(np.float64), masks[b], target, ds)
        if margin < 1e-5:
            continue
        sure += 1
        assert path[b].tolist() == want + [R.ABSENT] * (tokens - len(want)), b
        assert kept[b] == len(want) and sampled[b, 0] == token and sampled[b, 1] == 0, b
    assert sure >= 0.9 * s


@pytest.mark.parametrize("gap", [14.0, 18.0, 25.0, 30.0])
@pytest.mark.parametrize("temperature", [0.6, 0.9])
def test_emitted_tokens_are_the_targets_own_draws(cuda, gap, temperature):
    """Three siblings drawn without replacement from a draft that is sure of its first: each candidate's count within five
    deviations of p, those of which fewer than 25 are expected counted together (with the next likely where all of
    those are fewer)."""
    rng = np.random.default_rng(int(gap))
    s, tokens = 200_000, 4
    one = V.lists(rng, (1, tokens), spread=0.5)
    draft_one = one.copy()
    draft_one[0, 0] = peaked(rng, one[0, 0, :, 1], gap, temperature)
    masks = np.tile(np.array([1, 3, 5, 9], np.uint64), (s, 1))
    target, ds = V.settings(0.9, top_k=30), V.settings(temperature)
    p = R.distribution(one[0, 0, :, 0], one[0, 0, :, 1], **target)
    q = R.distribution(draft_one[0, 0, :, 0], draft_one[0, 0, :, 1], **ds)
    ranked = np.argsort(-(np.log(q) + rng.gumbel(size=(s, 64))), -1)[:, :3]
    ids = np.concatenate([np.zeros((s, 1)), draft_one[0, 0, :, 1][ranked]], 1)
    path, kept, sampled = V.run(np.tile(one, (s, 1, 1, 1)), np.tile(draft_one, (s, 1, 1, 1)), ids.astype(np.uint32),
                                rng.random((s, tokens)), masks, None, target, ds)
    first = np.where(kept > 1, np.take_along_axis(ids, np.minimum(path[:, 1:2], 3).astype(np.int64), 1)[:, 0], sampled[:, 0])
    counts = np.array([(first == one[0, 0, j, 1]).sum() for j in range(64)])
    order = np.argsort(p)
    rare = np.zeros(64, bool)   # the least likely, until 25 are expected of them together
    rare[order[:max(int((s * p < 25).sum()), int(np.searchsorted(s * np.cumsum(p[order]), 25)) + 1)]] = True
    for count, share in [*zip(counts[~rare], p[~rare]), (counts[rare].sum(), p[rare].sum())]:
        assert abs(count - s * share) <= 5 * np.sqrt(s * share * (1 - share)), (count, s * share)
    assert counts.sum() == s and not counts[p == 0].any()


def test_a_mass_below_normal_numbers_stays_finite(cuda):
    """Siblings of 1e-40 each (their quotients keep few bits): refused or kept, the draw after them is of the target's
    candidates."""
    rng = np.random.default_rng(9)
    s, tokens = 200, 4
    masks = np.tile(np.array([1, 3, 5, 9], np.uint64), (s, 1))
    candidates = V.lists(rng, (s, tokens), spread=0.6)
    draft = candidates.copy()
    for b in range(s):
        draft[b, 0] = peaked(rng, candidates[b, 0, :, 1], 92.0, 1.0)
    ids = np.concatenate([np.zeros((s, 1)), draft[:, 0, :3, 1]], 1)
    u = rng.random((s, tokens)).astype(np.float32)
    path, kept, sampled = V.run(candidates, draft, ids, u, masks, None, V.settings(top_k=20), V.settings())
    assert (sampled[:, 1] == 0).all()
    for b in range(s):
        at = path[b, kept[b] - 1]
        assert sampled[b, 0] in candidates[b, at, :20, 1], b
        if kept[b] == 1 and u[b, 0] > 0.5:   # the first was refused: nothing of it is left to draw
            assert sampled[b, 0] != ids[b, 1], b
