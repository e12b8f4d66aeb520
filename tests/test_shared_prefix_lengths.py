"""A SharedPrefixes that is kept while contexts grow plans as a new one does (CPU)."""
import pytest
import torch

from tests.helpers import small_case
from tokenfactory_amd import SharedPrefixes
from tokenfactory_amd.shared_prefix import MAX_LAYOUTS, planned_length


@pytest.fixture(autouse=True)
def cus(monkeypatch):
    monkeypatch.setattr("tokenfactory_amd.shared_prefix._cu_count", lambda device: 256)


def plan_at(shared, batch, max_len):
    batch.max_seq_len = max_len
    return shared._plan(batch, sum(batch.extend_lens), 24, 4, 256, 0, torch.device("cpu"))


def same(a, b):
    return (a.n_stream, a.n_pieces, a.n_items, a.n_shared) == \
        (b.n_stream, b.n_pieces, b.n_items, b.n_shared) and (a._host == b._host).all() \
        and (a.route and a.route.split) == (b.route and b.route.split)


@pytest.mark.parametrize("ext", [[1] * 16, [4] * 16, [1] * 15 + [64]])
def test_a_kept_object_plans_as_a_new_one(ext):
    groups = [(list(range(12)), 5000)]
    batch = small_case([64] * 16, ext, d=64, dtype=torch.bfloat16).batch
    batch.req_to_token = torch.zeros((16, 40000), dtype=torch.int64)
    kept, seen = SharedPrefixes(groups), set()
    for own in (1, 2, 70, 300, 1024, 4096, 9000, 30000, 1):
        plan = plan_at(kept, batch, 5000 + own)
        assert same(plan, plan_at(SharedPrefixes(groups), batch, 5000 + own)), own
        seen.add(plan.n_stream)
    assert len(seen) > 3   # (that lengths matter at all)


def test_prompts_are_cut_once_their_contexts_are_long():
    batch = small_case([70, 70, 70], [1, 1, 64], d=64, dtype=torch.bfloat16).batch
    batch.req_to_token = torch.zeros((8, 40000), dtype=torch.int64)
    kept = SharedPrefixes([([0, 1], 500)])
    assert not plan_at(kept, batch, 800).route.split
    assert plan_at(kept, batch, 30000).route.split


def test_lists_stay_while_lengths_grow_a_little():
    batch = small_case([64] * 4, [1] * 4, d=64, dtype=torch.bfloat16).batch
    batch.req_to_token = torch.zeros((8, 40000), dtype=torch.int64)
    kept = SharedPrefixes([([0, 1, 2, 3], 1000)])
    plans = {id(plan_at(kept, batch, n)) for n in range(1001, 20000)}
    assert len(plans) <= 40 and len(kept._plans) <= MAX_LAYOUTS
    assert plan_at(kept, batch, 1001) is plan_at(kept, batch, 1063)


@pytest.mark.parametrize("longest", [0, 1, 63, 300, 8192])
def test_planned_lengths(longest):
    """Within an eighth of what lies behind the longest shared part, 32 below 64; in order."""
    last = 0
    for n in range(40000):
        m = planned_length(n, longest)
        base = 0 if n <= longest else longest
        assert abs(m - n) <= max(32, (n - base) / 8) and m >= last
        assert (m <= longest) == (n <= longest)
        last = m


def test_planned_lengths_of_far_contexts():
    assert abs(planned_length((1 << 40) + 5, 7) - (1 << 40)) <= 1 << 37
