"""shared_prefix_attention with an object that is kept while contexts grow."""
import pytest
import torch

from tests.part_oracle import assert_attention, attention64
from tests.test_gpu_shared_prefix import call, shared_case
from tokenfactory_amd import SharedPrefixes

pytestmark = pytest.mark.gpu


def set_lens(wl, lens):
    wl.batch.seq_lens.copy_(torch.tensor(lens))
    wl.batch.max_seq_len = max(lens)


def right(wl, got, what):
    want, spread, _ = attention64(wl, seq_lens=wl.batch.seq_lens.tolist())
    assert_attention(got, want, spread, wl, what)


@pytest.mark.parametrize("d,fp8", [(256, False), (256, True), (128, False)])
def test_growing_contexts(gpu, d, fp8):
    """The same bits as of an object made for the step: the work is cut alike."""
    n = 24
    wl, members = shared_case([600], [1500 - 7 * b for b in range(n)], [0] * n, d=d, seed=60,
                              fp8=fp8)
    kept = SharedPrefixes(members)
    for own in (1, 100, 700, 1500, 60):
        set_lens(wl, [600 + max(1, own - 7 * b) for b in range(n)])
        got = call(wl, kept)
        assert torch.equal(got, call(wl, SharedPrefixes(members))), own
    right(wl, got, f"own {own}")


def test_captured_at_other_lengths(gpu):
    """A capture takes the lists that an eager call at other lengths made, and a replay the
    lengths of its time."""
    wl, members = shared_case([500], [1200, 900, 3, 40, 700], [0] * 5, seed=61)
    full = wl.batch.seq_lens.tolist()
    kept = SharedPrefixes(members)
    set_lens(wl, [502, 501, 501, 501, 501])
    call(wl, kept)
    wl.batch.max_seq_len = max(full)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(wl, kept)
    del kept
    for lens in (full, [501] * 5, [600, 503, 502, 0, 1200], full):
        wl.batch.seq_lens.copy_(torch.tensor(lens))
        filler = [torch.full((4096,), -1, dtype=torch.int32, device=gpu) for _ in range(20)]
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        right(wl, out, f"replayed {lens}")
        del filler
