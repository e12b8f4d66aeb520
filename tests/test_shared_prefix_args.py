"""shared_prefix_attention's and SharedPrefixes' refusals, and the lists of a plan (CPU)."""
import numpy as np
import pytest
import torch

from tests.helpers import small_case
from tokenfactory_amd import SharedPrefixes, shared_prefix_attention
from tokenfactory_amd.shared_prefix import MAX_LAYOUTS, MIN_STEPS, _Plan, cut_units


@pytest.mark.parametrize("groups", [[([0, 0], 5)], [([0, 1], 5), ([1, 2], 5)], [([0, -1], 5)],
                                    [([0, 1], -1)], [([0, 1], 1 << 31)]])
def test_bad_groups(groups):
    with pytest.raises(ValueError):
        SharedPrefixes(groups)


def test_runs_on_devices_only():
    wl = small_case([9, 9], [1, 1], d=64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="ROCm"):
        shared_prefix_attention(wl.q, wl.k_pool, wl.v_pool, wl.batch, SharedPrefixes([([0, 1], 4)]))


def test_gradients_are_refused():
    wl = small_case([9, 9], [1, 1], d=64, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError, match="gradient"):
        shared_prefix_attention(wl.q.requires_grad_(), wl.k_pool, wl.v_pool, wl.batch,
                                SharedPrefixes([([0, 1], 4)]))


def test_groups_must_fit_the_batch():
    wl = small_case([9, 9], [1, 1], d=64, dtype=torch.bfloat16)
    dev = torch.device("cpu")
    with pytest.raises(ValueError, match="batch of 2"):
        SharedPrefixes([([0, 2], 4)])._plan(wl.batch, 2, 4, 1, 64, 0, dev)
    with pytest.raises(ValueError, match="width"):
        SharedPrefixes([([0, 1], 400)])._plan(wl.batch, 2, 4, 1, 64, 0, dev)


def lists(plan):
    """(items, work, pieces, tokens, units) of a plan's host copy."""
    cuts = [at // 4 for at in plan._offsets] + [len(plan._host)]
    parts = [plan._host[a:b] for a, b in zip(cuts, cuts[1:])]
    return [x.reshape(-1, n) for x, n in zip(parts, (8, 8, 8, 4, 2))]


EXT = [1, 4, 2, 1, 70, 1] + [1] * 60
GROUPS = [([0, 1, 5] + list(range(6, 60)), 2000), ([2, 4, 62], 50)]


@pytest.mark.parametrize("head_dim,fp8,pieces", [(256, False, True), (256, True, True),
                                                 (128, False, True), (128, True, False),
                                                 (8, False, True), (136, False, False)])
def test_what_takes_the_shared_parts(head_dim, fp8, pieces):
    plan = _Plan([([0, 1], 1000)], [1, 1], 24, 4, head_dim, torch.device("cpu"), 256, 1100, fp8)
    assert (plan.n_pieces > 0) == pieces and (plan.n_shared > 0) != pieces
    assert (plan.n_stream > 0) == pieces and plan.row_groups == 1


@pytest.mark.parametrize("head_dim", [256, 128, 192])
@pytest.mark.parametrize("groups", [[], [([1, 2], 60)]])
def test_steps_that_share_nothing(head_dim, groups):
    """No group, or (at 256 dims) one whose other member is a long prompt."""
    ext = [1, 1, 100]
    plan = _Plan(groups, ext, 24, 4, head_dim, torch.device("cpu"), 256, 1100, False)
    assert plan.shares == (bool(groups) and head_dim != 256)


@pytest.mark.parametrize("head_dim,new,beside", [(256, 9, True), (128, 10, True),
                                                 (128, 11, False)])
def test_rows_too_many_to_stream_beside(head_dim, new, beside):
    plan = _Plan([([0, 1], 1000)], [1, new], 24, 4, head_dim, torch.device("cpu"), 256, 1100, 0)
    assert plan.n_pieces and (plan.n_stream > 0) == beside
    assert plan.row_groups == (1 if beside else 2)


@pytest.mark.parametrize("head_dim", [256, 128])
def test_parts_of_few_rows_are_streamed_where_they_are_many(head_dim):
    """Pairs of 12 rows: by tiles alone, streamed where there are many or own keys are
    nearly all; threes of 18 rows by tiles."""
    def plan(n, members, max_len):
        groups = [(list(range(g * members, (g + 1) * members)), 500) for g in range(n)]
        return _Plan(groups, [1] * n * members, 24, 4, head_dim, torch.device("cpu"), 256,
                     max_len, 0)
    assert plan(2, 2, 600).n_pieces
    assert not plan(40, 2, 600).n_pieces and plan(40, 2, 600).n_shared == 40
    assert not plan(2, 2, 9000).n_pieces
    assert plan(40, 3, 600).n_pieces


def test_long_prompts_on_long_contexts_are_cut():
    def plan(max_len):
        return _Plan([([0, 1], 500)], [1, 1, 64], 24, 4, 256, torch.device("cpu"), 256, max_len, 0)
    assert plan(60000).route.split and not plan(800).route.split
    assert plan(800).n_work == plan(60000).n_work == 8


def test_layouts_are_bounded(monkeypatch):
    """One object over many layouts keeps the lists of the latest alone."""
    monkeypatch.setattr("tokenfactory_amd.shared_prefix._cu_count", lambda device: 256)
    shared = SharedPrefixes([([0, 1], 100)])
    plans = []
    for new in range(1, MAX_LAYOUTS + 3):
        b = small_case([200, 200], [1, new], d=128, dtype=torch.bfloat16).batch
        n_tok = sum(b.extend_lens)
        plans.append(shared._plan(b, n_tok, 24, 4, 128, 0, torch.device("cpu")))
        assert shared._plan(b, n_tok, 24, 4, 128, 0, torch.device("cpu")) is plans[-1]
    assert len(shared._plans) == MAX_LAYOUTS


@pytest.mark.parametrize("head_dim", [256, 128, 192])
def test_plan_covers_every_row_and_key_once(head_dim):
    """Each output row has one own part; own and shared parts meet at the shared length; a
    row's place in the shared part names the same token; pieces cover a unit's keys."""
    group, n_kv = 6, 4
    plan = _Plan(GROUPS, EXT, 24, n_kv, head_dim, torch.device("cpu"), 64, 3000, False)
    long_ = {4} if head_dim == 256 else set()
    items, work, pieces, toks, units = lists(plan)
    unit = 16 * plan.row_groups
    starts = np.concatenate([[0], np.cumsum(EXT)])
    rows = set()
    for b, tok0, n, row0, k0, k1, pfx, pfx_tok in items[plan.n_shared:]:
        assert k1 == -1 and row0 % unit == 0
        shares = [length for m, length in GROUPS if b in m and len(set(m) - long_) > 1]
        assert k0 == (shares[0] if shares else 0) and (pfx >= 0) == bool(shares)
        for rho in range(row0, min(row0 + unit, n * group)):
            t = rho // group
            assert toks[tok0 + t].tolist() == [starts[b] + t, b, EXT[b] - 1 - t, 0]
            rows.add((b, rho))
            if pfx < 0:
                continue
            rp = (pfx_tok + t) * group + rho % group
            if head_dim == 192:
                front = items[pfx + rp // unit]
                assert front[3] == rp // unit * unit and front[4] == 0 and front[5] == k0
                assert toks[front[1] + pfx_tok + t].tolist() == toks[tok0 + t].tolist()
                assert rp < front[2] * group
                continue
            for hk in range(n_kv):
                slot, n_parts = units[pfx + rp // 256 * n_kv + hk]
                cut = pieces[slot:slot + n_parts]
                assert (cut[:, 1] == hk).all() and (cut[:, 2] == rp // 256 * 256).all()
                assert cut[:, 7].tolist() == list(range(slot + 1, slot + n_parts + 1))
                assert cut[0, 5] == 0 and cut[-1, 6] == k0
                assert (cut[1:, 5] == cut[:-1, 6]).all() and (cut[:, 5] < cut[:, 6]).all()
                for _, _, _, front, n_front, *_ in cut:
                    assert toks[front + pfx_tok + t].tolist() == toks[tok0 + t].tolist()
                    assert rp < n_front * group
    assert rows == {(b, r) for b, e in enumerate(EXT) if b not in long_ for r in range(e * group)}
    assert set(work[:, 0].tolist()) == long_
    assert (len(pieces) > 0) == (head_dim != 192) and len(pieces) <= 64


@pytest.mark.parametrize("steps,cus", [([256] * 8, 256), ([1024] * 24, 256), ([1], 256),
                                       ([1, 500, 3], 16), ([100] * 300, 256), ([8] * 31, 256)])
def test_cuts(steps, cus):
    cuts = cut_units(steps, cus)
    assert len(cuts) == len(steps)
    assert sum(cuts) <= max(cus, len(steps))
    assert all(1 <= c <= max(1, -(-s // MIN_STEPS)) for c, s in zip(cuts, steps))
