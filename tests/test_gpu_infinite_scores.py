"""Rows whose visible keys all score minus infinity: NaN, as the softmax over them is, and
not the zeros of rows that see no key; rows that see other keys beside those leave them out."""
import dataclasses

import pytest
import torch

from tests.part_oracle import assert_attention, attention64, score_error
from tests.test_gpu_shared_prefix import call, shared_case
from tokenfactory_amd import SharedPrefixes, scored_attention

pytestmark = pytest.mark.gpu

LAYOUTS = [([50, 0], [4, 7, 5, 9], [0, 0, 0, 1]),            # few keys
           ([1700, 0], [40, 300, 5, 129], [0, 0, 0, 1])]     # several pieces and tiles


def case(layout, ext, d):
    """(workload, groups, the workload with finite keys): request 1's keys and, with them, the
    shared ones score -inf for every query; the others' own are finite."""
    prefixes, own, groups = layout
    wl, members = shared_case(prefixes, own, groups, ext=ext, d=d, seed=70)
    wl.q[..., 0] = -1
    finite = dataclasses.replace(wl, k_pool=wl.k_pool.clone())
    slots = wl.batch.req_to_token[wl.rows[1], :wl.seq_lens[1]]
    wl.k_pool[slots, :, 0] = float("inf")
    return wl, members, finite


def check(got, want, spread, finite, what):
    odd = want.isnan()
    assert odd.any() and not odd.all()
    assert torch.equal(got.isnan().cpu(), odd), what
    rows = ~odd.flatten(1).any(dim=1)
    assert_attention(got[rows.to(got.device)], want[rows], spread[rows], finite, what)


@pytest.mark.parametrize("ext", [[1] * 4, [2, 1, 3, 2]])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("d", [256, 128, 192])
def test_shared(gpu, d, layout, ext):
    wl, members, finite = case(layout, ext, d)
    print(f"[shared] D={d} {layout} {ext}", flush=True)
    want, spread, _ = attention64(wl)
    check(call(wl, SharedPrefixes(members)), want, spread, finite, f"{d} {layout}")


def test_padding_stays_zero(gpu):
    wl, members, finite = case(LAYOUTS[0], [1] * 4, 256)
    wl.batch.seq_lens[2] = 0
    want, spread, _ = attention64(wl, seq_lens=wl.batch.seq_lens.tolist())
    got = call(wl, SharedPrefixes(members))
    check(got, want, spread, finite, "padding")
    assert (got[2] == 0).all()


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("d", [256, 128, 192])
def test_scored_decodes(gpu, d, layout):
    """Output, and the weights: NaN for a request with such a row, the others' as ever."""
    wl, members, finite = case(layout, [1] * 4, d)
    print(f"[scored] D={d} {layout}", flush=True)
    want, spread, weights = attention64(wl)
    scores = torch.zeros(wl.batch.req_to_token.shape, device=gpu)
    got = scored_attention(wl.q, wl.k_pool, wl.v_pool, wl.batch, scores, scaling=wl.scale)
    check(got, want, spread, finite, f"{d} {layout}")
    check_weights(wl, finite, scores, weights)


@pytest.mark.parametrize("d", [256, 64])
def test_scored_prompts(gpu, d):
    wl, members, finite = case(LAYOUTS[0], [2, 1, 3, 9], d)
    _, _, weights = attention64(wl)
    scores = torch.zeros(wl.batch.req_to_token.shape, device=gpu)
    scored_attention(wl.q, wl.k_pool, wl.v_pool, wl.batch, scores, scaling=wl.scale)
    check_weights(wl, finite, scores, weights)


def check_weights(wl, finite, scores, weights):
    for row, n, w in zip(wl.rows, wl.seq_lens, weights):
        got = scores[row, :n].double().cpu()
        assert torch.equal(got.isnan(), w.isnan()), row
        if not w.isnan().any():   # (the bound of tests/test_gpu_scored_attention.py)
            terms = wl.num_q_heads * 32
            rel = 2 * score_error(finite) + (n / 32 + 64) * 2.0 ** -22 + terms * 2.0 ** -24
            assert ((got - w).abs() <= w * rel * 1.01 + 2.0 ** -100).all(), row
        assert (scores[row, n:] == 0).all()
