"""shared_prefix_attention's and SharedPrefixes' refusals, and the lists of a plan (CPU)."""
import numpy as np
import pytest
import torch

from tests.helpers import small_case
from tokenfactory_amd import SharedPrefixes, shared_prefix_attention
from tokenfactory_amd.shared_prefix import _Plan


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
        SharedPrefixes([([0, 2], 4)])._plan(wl.batch, [1, 1], 4, 1, 64, dev)
    with pytest.raises(ValueError, match="width"):
        SharedPrefixes([([0, 1], 400)])._plan(wl.batch, [1, 1], 4, 1, 64, dev)


@pytest.mark.parametrize("head_dim", [256, 128])
def test_plan_covers_every_row_and_key_once(head_dim):
    """Each output row has one own part; own and shared parts meet at the shared length;
    a row's place in the shared part names the same token."""
    ext = [1, 4, 2, 1, 70, 1]
    groups = [([0, 1, 5], 100), ([2, 4], 50)]
    group = 6
    plan = _Plan(groups, ext, 24, 4, head_dim, torch.device("cpu"))
    long_ = {4} if head_dim == 256 else set()
    items = plan._host[:8 * plan.n_items].reshape(-1, 8)
    toks = plan._host[8 * (plan.n_items + plan.n_work):].reshape(-1, 4)
    unit = 16 * plan.row_groups
    starts = np.concatenate([[0], np.cumsum(ext)])
    rows = set()
    for b, tok0, n, row0, k0, k1, pfx, pfx_tok in items[plan.n_shared:]:
        assert k1 == -1 and row0 % unit == 0
        shares = [length for m, length in groups if b in m and len(set(m) - long_) > 1]
        assert k0 == (shares[0] if shares else 0) and (pfx >= 0) == bool(shares)
        for rho in range(row0, min(row0 + unit, n * group)):
            t = rho // group
            assert toks[tok0 + t].tolist() == [starts[b] + t, b, ext[b] - 1 - t, 0]
            rows.add((b, rho))
            if pfx >= 0:
                rp = (pfx_tok + t) * group + rho % group
                front = items[pfx + rp // unit]
                assert front[3] == rp // unit * unit and front[4] == 0 and front[5] == k0
                assert toks[front[1] + pfx_tok + t].tolist() == toks[tok0 + t].tolist()
                assert rp < front[2] * group
    assert rows == {(b, r) for b, e in enumerate(ext) if b not in long_ for r in range(e * group)}
    work = plan._host[8 * plan.n_items:8 * (plan.n_items + plan.n_work)].reshape(-1, 8)
    assert set(work[:, 0].tolist()) == long_
