"""evict_tokens against a plain sort on the host: whole numbers and moved scores, equal."""
import random

import pytest
import torch

from tokenfactory_amd import evict_tokens

pytestmark = pytest.mark.gpu


def expected(table, scores, rows, lens, keep, firsts, recent, out_rows, width):
    table, scores = table.cpu().clone(), scores.cpu().clone()
    src_t, src_s = table.clone(), scores.clone()
    freed = torch.full((len(rows), width), -1, dtype=torch.int64)
    new = []
    for b, (row, to, n, first) in enumerate(zip(rows, out_rows, lens, firsts)):
        first = max(0, min(first, n))
        end = max(first, n - recent)
        left = min(n, max(keep, first + recent))
        room = left - first - (n - end)
        v = src_s[row, first:end].double()
        v = torch.where(torch.isnan(v), torch.tensor(-float("inf"), dtype=v.dtype), v).tolist()
        isnan = torch.isnan(src_s[row, first:end]).tolist()
        best = sorted(range(len(v)), key=lambda i: (isnan[i], -v[i], i))[:max(0, room)]
        stay = list(range(first)) + sorted(first + i for i in best) + list(range(end, n))
        gone = sorted(set(range(n)) - set(stay))
        table[to, :n], scores[to, :n] = -1, 0.0
        table[to, :len(stay)] = src_t[row, stay]
        scores[to, :len(stay)] = src_s[row, stay]
        freed[b, :len(gone)] = src_t[row, gone]
        new.append(len(stay))
    return new, freed, table, scores


def run(lens, keep, first=0, recent=0, values=None, moved=False, width=None, seed=0, pad=0):
    gen = torch.Generator("cuda").manual_seed(seed)
    n = len(lens)
    max_len = max(lens)
    cols = width or max_len + 3
    table = torch.randint(1, 1 << 40, (2 * n + 1, cols + pad), generator=gen, device="cuda")[:, :cols]
    scores = torch.rand((2 * n + 1, cols + 2 * pad), generator=gen, device="cuda")[:, :cols]
    if values is not None:
        values(scores, gen)
    perm = torch.randperm(2 * n + 1, generator=gen, device="cuda")
    rows, out_rows = perm[:n].contiguous(), perm[n:2 * n].contiguous()
    seq = torch.tensor(lens, device="cuda")
    firsts = first.tolist() if isinstance(first, torch.Tensor) else [first] * n
    want = expected(table, scores, rows.tolist(), lens, keep, firsts, recent,
                    (out_rows if moved else rows).tolist(), max(0, max_len - keep))
    got_lens, freed = evict_tokens(table, scores, rows, seq, keep, max_seq_len=max_len, first=first,
                                   recent=recent, out_rows=out_rows if moved else None)
    assert got_lens.tolist() == want[0]
    assert torch.equal(freed.cpu(), want[1])
    assert torch.equal(table.cpu(), want[2])
    assert torch.equal(scores.cpu().nan_to_num(7.5), want[3].nan_to_num(7.5))


@pytest.mark.parametrize("moved", [False, True])
@pytest.mark.parametrize("lens,keep,first,recent", [
    ([1, 2, 3, 0], 1, 0, 0), ([1, 2, 3, 0], 0, 0, 0), ([10, 4, 9], 4, 1, 1), ([10], 10, 0, 0),
    ([10, 64], 63, 60, 3), ([300, 1000, 65], 64, 0, 0), ([300, 1000, 65], 64, 64, 0),
    ([300, 1000, 65], 64, 0, 64), ([300, 1000, 65], 64, 100, 50), ([4096, 4097, 4095], 1000, 4, 32),
    ([8193, 5000], 4096, 1, 4000), ([20000, 12288, 12289, 100], 5000, 17, 333),
    ([65536, 70001], 9000, 4, 64), ([150000], 20000, 4, 1024), ([7, 7], 100, 3, 3)])
def test_lengths(gpu, lens, keep, first, recent, moved):
    print(f"[evict] {lens} keep {keep} first {first} recent {recent} moved {moved}", flush=True)
    run(lens, keep, first, recent, moved=moved, seed=sum(lens))


def few_values(scores, gen):
    scores.copy_(torch.randint(0, 5, scores.shape, generator=gen, device="cuda") * 0.25)


def one_value(scores, gen):
    scores.fill_(0.125)


def zeros(scores, gen):
    scores.fill_(0.0)
    scores[:, ::3] = -0.0


def wide(scores, gen):
    """Every exponent, denormals among them, and both signs."""
    bits = torch.randint(-(1 << 31), 1 << 31, scores.shape, generator=gen, device="cuda")
    x = bits.to(torch.int32).view(torch.float32)
    scores.copy_(torch.where(torch.isfinite(x), x, torch.zeros_like(x)))


def near(scores, gen):
    """Neighbouring numbers: they differ in the last bits."""
    bits = 0x3F800000 + torch.randint(0, 40, scores.shape, generator=gen, device="cuda")
    scores.copy_(bits.to(torch.int32).view(torch.float32))


def odd(scores, gen):
    x = torch.randint(0, 12, scores.shape, generator=gen, device="cuda")
    scores[x == 0] = float("nan")
    scores[x == 1] = float("inf")
    scores[x == 2] = -float("inf")
    scores[x == 3] = -1.0


@pytest.mark.parametrize("moved", [False, True])
@pytest.mark.parametrize("values", [few_values, one_value, zeros, wide, near, odd])
def test_values(gpu, values, moved):
    run([3000, 9000, 77, 500], 400, 4, 16, values=values, moved=moved, seed=3)
    run([40000, 33000], 12000, 4, 16, values=values, moved=moved, seed=4)


def test_prefix_lengths_per_request(gpu):
    first = torch.tensor([0, 100, 5000, 64, 1 << 40, -5], device=gpu)
    run([500, 500, 500, 30, 700, 90], 200, first, 50, seed=5)
    run([500, 500, 500, 30, 700, 90], 200, first, 50, seed=5, moved=True)


@pytest.mark.parametrize("which", ["keep", "first", "recent"])
@pytest.mark.parametrize("longest", [300, 20000])
def test_sizes_beyond_every_row(gpu, which, longest):
    run([longest, 70, 0], **{"keep": 40, "first": 3, "recent": 5, which: 2 ** 63 - 1})


def test_strided_tables_and_other_columns_stay(gpu):
    run([500, 300], 128, 4, 16, pad=5, width=900, seed=6)


def test_random_cases(gpu):
    rng = random.Random(8)
    for i in range(30):
        lens = [rng.randint(0, rng.choice([20, 600, 9000, 40000])) for _ in range(rng.randint(1, 5))]
        lens[0] = max(1, lens[0])
        keep = rng.randint(0, max(lens))
        first = rng.randint(0, keep)
        values = rng.choice([None, few_values, wide, odd])
        run(lens, keep, first, rng.randint(0, keep), values=values, moved=rng.random() < 0.5, seed=i)


def test_lengths_outside_the_table_are_clamped(gpu):
    table = torch.arange(400, device=gpu).view(4, 100)
    scores = torch.zeros((4, 100), device=gpu)
    rows = torch.tensor([0, 2], device=gpu)
    lens, freed = evict_tokens(table, scores, rows, torch.tensor([5000, -3], device=gpu), 10,
                               max_seq_len=40)
    assert lens.tolist() == [10, 0]
    assert freed[0].tolist() == list(range(10, 40)) and (freed[1] == -1).all()
    assert table[0, 40:].tolist() == list(range(40, 100)) and (table[0, 10:40] == -1).all()


def test_captured_and_replayed(gpu):
    """In place, replayed on new rows and lengths, with eager work between."""
    gen = torch.Generator("cuda").manual_seed(1)
    table = torch.zeros((6, 5000), dtype=torch.int64, device=gpu)
    scores = torch.zeros((6, 5000), device=gpu)
    rows = torch.tensor([1, 3, 4], device=gpu)
    seq = torch.tensor([1, 1, 1], device=gpu)
    call = lambda t, s: evict_tokens(t, s, rows, seq, 300, max_seq_len=5000, first=4, recent=16)
    call(table, scores)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lens, freed = call(table, scores)
    for step in range(4):
        table.copy_(torch.randint(1, 1 << 40, table.shape, generator=gen, device=gpu))
        scores.copy_(torch.rand(scores.shape, generator=gen, device=gpu))
        seq.copy_(torch.tensor([5000 - step, 200, 301 + step]))
        t, s = table.clone(), scores.clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = call(t, s)
        assert torch.equal(lens, want[0]) and torch.equal(freed, want[1])
        assert torch.equal(table, t) and torch.equal(scores, s)


def test_streams(gpu):
    table = torch.randint(1, 1 << 40, (8, 60000), device=gpu)
    scores = torch.rand((8, 60000), device=gpu)
    rows, seq = torch.tensor([0, 5], device=gpu), torch.tensor([60000, 1000], device=gpu)
    kw = dict(max_seq_len=60000, first=4, recent=16)
    copies = [(table.clone(), scores.clone()) for _ in range(3)]
    want = evict_tokens(table, scores, rows, seq, 500, **kw)
    torch.cuda.synchronize()
    got = [evict_tokens(t, s, rows, seq, 500, stream=torch.cuda.Stream(), **kw) for t, s in copies]
    filler = [torch.full((2, 59500), 9, device=gpu) for _ in range(20)]
    torch.cuda.synchronize()
    for (t, s), (lens, freed) in zip(copies, got):
        assert torch.equal(t, table) and torch.equal(s, scores)
        assert torch.equal(lens, want[0]) and torch.equal(freed, want[1])
    del filler


def test_empty_batch(gpu):
    empty = torch.zeros(0, dtype=torch.int64, device=gpu)
    lens, freed = evict_tokens(torch.ones((2, 9), dtype=torch.int64, device=gpu),
                               torch.zeros((2, 9), device=gpu), empty, empty, 4, max_seq_len=9)
    assert lens.shape == (0,) and freed.shape == (0, 5)


@pytest.mark.parametrize("change,match", [
    (dict(keep=-1), "keep"), (dict(recent=-1), "recent"), (dict(first=-2), "first"),
    (dict(max_seq_len=10), "width"), (dict(max_seq_len=-1), "width"),
    (dict(seq="int32"), "seq_lens"), (dict(rows="long"), "seq_lens"), (dict(out="short"), "out_rows"),
    (dict(first="cpu"), "first"), (dict(scores="half"), "scores"), (dict(table="int32"), "table|req_to")])
def test_refusals(gpu, change, match):
    table = torch.ones((4, 9), dtype=torch.int64, device=gpu)
    scores = torch.zeros((4, 9), device=gpu)
    rows, seq = torch.tensor([0, 1], device=gpu), torch.tensor([9, 9], device=gpu)
    args = dict(keep=4, max_seq_len=9, first=0, recent=0, out_rows=None)
    for k, v in change.items():
        if k in ("keep", "recent", "max_seq_len") or (k == "first" and v != "cpu"):
            args[k] = v
    if change.get("seq"):
        seq = seq.int()
    if change.get("rows"):
        rows = torch.tensor([0, 1, 2], device=gpu)
    if change.get("out"):
        args["out_rows"] = rows[:1]
    if change.get("first") == "cpu":
        args["first"] = torch.zeros(2, dtype=torch.int64)
    if change.get("scores"):
        scores = scores.half()
    if change.get("table"):
        table = table.int()
    keep = args.pop("keep")
    with pytest.raises(ValueError, match=match):
        evict_tokens(table, scores, rows, seq, keep, **args)
    assert (table == 1).all() and (scores == 0).all()


def test_runs_on_devices_only(gpu):
    t = torch.ones((2, 9), dtype=torch.int64)
    with pytest.raises(RuntimeError, match="ROCm"):
        evict_tokens(t, torch.zeros((2, 9)), torch.zeros(1).long(), torch.ones(1).long(), 4,
                     max_seq_len=9)
