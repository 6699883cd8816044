"""Sampled speculative steps of a whole decoder: the token after a prompt is
distributed as the target model's own draw, with drafts as without."""
import numpy as np
import pytest
import torch

import charlotte_b200 as cb
import speculative_reference as R
from charlotte_b200 import model as M
from charlotte_b200 import speculative as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", [cb.CACHE_F16, cb.CACHE_Q8])
@pytest.mark.parametrize("drafted", [0, 3])
def test_the_next_token_is_the_targets_draw(cuda, cache, drafted):
    """64 sequences of one prompt, 100 steps from the same place: each candidate's count within five deviations of its
    probability, the least likely counted together until 25 are expected of them."""
    sequences, rounds, prompt = 64, 100, [5, 6, 7, 8]
    m = M.synthesize(M.tiny("qwen3"), seed=7)
    settings = dict(temperature=2.0, top_k=20, top_p=0.95, min_p=0.0)
    d = S.SpeculativeDecoder(m, sequences, 1 + drafted, cache)
    d.prefill([prompt] * sequences)
    start = d.lengths.clone()
    rng = np.random.default_rng(8)
    d.step([([prompt[-1]], [-1])] * sequences)
    candidates = d.candidates.view(sequences, 1 + drafted, 64, 2)[0, 0].cpu().numpy().view(np.uint32)
    p = R.distribution(candidates[:, 0], candidates[:, 1], **settings)
    # siblings: a likely token, an unlikely one, and one that the target's draw never gives
    tree = ([prompt[-1], *(int(candidates[i, 1]) for i in (1, 6, 40)[:drafted])], [-1] + [0] * drafted)
    counts = np.zeros(64)
    for _ in range(rounds):
        d.lengths.copy_(start)
        u = torch.from_numpy(rng.random((sequences, 1 + drafted), np.float32))
        for new in d.step([tree] * sequences, settings, u):
            counts[int(np.nonzero(candidates[:, 1] == new[0])[0][0])] += 1
    n = sequences * rounds
    order = np.argsort(p)
    rare = np.zeros(64, bool)
    rare[order[:max(int((n * p < 25).sum()), int(np.searchsorted(n * np.cumsum(p[order]), 25)) + 1)]] = True
    assert (~rare).sum() >= 5 and not counts[p == 0].any()
    for count, share in [*zip(counts[~rare], p[~rare]), (counts[rare].sum(), p[rare].sum())]:
        assert abs(count - n * share) <= 5 * np.sqrt(n * share * (1 - share)), (count, n * share)
