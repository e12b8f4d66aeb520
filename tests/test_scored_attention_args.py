"""scored_attention's refusals (CPU)."""
import pytest
import torch

from tests.helpers import small_case
from tokenfactory_amd import scored_attention
from tokenfactory_amd.scored_attention import check_scores


def wl():
    return small_case([9, 9], [1, 1], d=64, dtype=torch.bfloat16)


def test_runs_on_devices_only():
    w = wl()
    scores = torch.zeros(w.batch.req_to_token.shape)
    with pytest.raises(RuntimeError, match="ROCm"):
        scored_attention(w.q, w.k_pool, w.v_pool, w.batch, scores)


@pytest.mark.parametrize("which", ["q", "scores"])
def test_gradients_are_refused(which):
    w = wl()
    scores = torch.zeros(w.batch.req_to_token.shape)
    (w.q if which == "q" else scores).requires_grad_()
    with pytest.raises(NotImplementedError, match="gradient"):
        scored_attention(w.q, w.k_pool, w.v_pool, w.batch, scores)


@pytest.mark.parametrize("scores", [
    torch.zeros((8, 32), dtype=torch.float64), torch.zeros((7, 32)), torch.zeros((8, 31)),
    torch.zeros((8, 64))[:, ::2], torch.zeros(8 * 32), torch.zeros((1, 32)).expand(8, 32)])
def test_scores_must_fit_the_table(scores):
    with pytest.raises(ValueError, match="scores"):
        check_scores("f", scores, torch.zeros((8, 32), dtype=torch.int64))


@pytest.mark.parametrize("scores", [torch.zeros((8, 32)), torch.zeros((9, 40)),
                                    torch.zeros((8, 50))[:, 3:40]])
def test_scores_that_fit(scores):
    check_scores("f", scores, torch.zeros((8, 32), dtype=torch.int64))
