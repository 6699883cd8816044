"""A draw's distribution keeps its first candidate whatever top_p is, in
verification (cb_verify_run) as in the selection (cb_select_run)."""
import numpy as np
import pytest
import torch

import charlotte_b200 as cb
import speculative_reference as R
import test_verify_gpu as V

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("top_p", [0.0, 1e-30, 1e-6])
@pytest.mark.parametrize("temperature", [0.0, 0.7])
def test_one_row_is_the_selections_first(cuda, top_p, temperature):
    rng = np.random.default_rng(6)
    rows, vocab = 100, 3000
    logits = torch.from_numpy((rng.standard_normal((rows, vocab)) * 2.5).astype(np.float32)).cuda()
    tiles, tickets = cb.lib().cb_select_tiles(vocab), cb.lib().cb_select_tickets(vocab)
    candidates = torch.zeros(rows, 64, 2, dtype=torch.int32, device="cuda")
    record = torch.zeros(rows, 4, dtype=torch.int32, device="cuda")
    cb.run("select", logits=logits, count=vocab, partials=torch.zeros(rows * tiles * 128, dtype=torch.int32, device="cuda"),
           ticket=torch.zeros(rows * tickets, dtype=torch.int32, device="cuda"), candidates=candidates, sampled=record,
           position0=5, tokens=1, seed0=3, seed1=4, top_k=40, temperature=temperature, top_p=top_p, min_p=0.0,
           log_min_p=0.0, rows=rows, logits_stride=vocab)
    u = record[:, 2].contiguous().view(torch.float32).cpu().numpy()[:, None]
    _, kept, sampled = V.run(candidates.cpu().numpy().view(np.uint32), None, np.zeros((rows, 1), np.uint32), u, None, None,
                             V.settings(temperature, 40, top_p))
    assert (kept == 1).all()
    assert (sampled == record.cpu().numpy().view(np.uint32)).all()
    assert (sampled[:, 0] == logits.argmax(-1).cpu().numpy()).all()


@pytest.mark.parametrize("have_draft", [True, False])
@pytest.mark.parametrize("top_p", [0.0, 1e-6])
def test_a_chain_of_the_first_candidates_is_kept(cuda, have_draft, top_p):
    """Target and draft of their first candidates alone: a draft of them is kept whole, any other refused."""
    rng = np.random.default_rng(7)
    candidates = V.lists(rng, (3, 4))
    ids = np.zeros((3, 4), np.uint32)
    ids[:, 1:] = candidates[:, :3, 0, 1]
    ids[1, 2] = candidates[1, 1, 1, 1]   # the second most likely
    u = np.full((3, 4), 0.999)
    path, kept, sampled = V.run(candidates, candidates if have_draft else None, ids, u, None, None, V.settings(0.8, top_p=top_p),
                                V.settings(1.0, top_p=top_p))
    assert kept.tolist() == [4, 2, 4]
    assert sampled[:, 0].tolist() == [candidates[0, 3, 0, 1], candidates[1, 1, 0, 1], candidates[2, 3, 0, 1]]
    assert path[0].tolist() == [0, 1, 2, 3] and path[1].tolist() == [0, 1, R.ABSENT, R.ABSENT]
