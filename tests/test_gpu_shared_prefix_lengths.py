"""shared_prefix_attention with an object that is kept while contexts grow."""
import dataclasses

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


def step_of(wl, lens):
    """A batch object of its own for the step with these lengths."""
    wl.batch = dataclasses.replace(wl.batch, seq_lens=torch.tensor(lens, device=wl.q.device),
                                   max_seq_len=max(lens))


@pytest.mark.parametrize("fp8", [False, True])
def test_prompt_beside_a_longer_context(gpu, fp8):
    """A prompt whose context grows while another request's is the longest: its entries are
    cut by the lengths of the step, as by an object made for it."""
    ext = [1, 1, 1, 200, 1]
    wl, members = shared_case([700, 0], [9, 1, 40, 5900, 5300], [0, 0, 0, 1, 0], ext=ext, seed=62,
                              fp8=fp8)
    kept = SharedPrefixes(members)
    for prompt in (200, 5900, 900):
        step_of(wl, [709, 701, 740, prompt, 6000])
        got = call(wl, kept)
        assert torch.equal(got, call(wl, kept)), prompt   # (the next layer)
        step_of(wl, wl.batch.seq_lens.tolist())
        assert torch.equal(got, call(wl, SharedPrefixes(members))), prompt
        right(wl, got, f"prompt {prompt}")


def test_prompt_pieces_on_several_streams(gpu):
    """One stream's pieces read by others, and dropped with their batch while they run."""
    wl, members = shared_case([700, 0], [9, 1, 40, 3000], [0, 0, 0, 1], ext=[1, 1, 1, 100],
                              seed=63)
    want = call(wl, SharedPrefixes(members))
    kept = SharedPrefixes(members)
    side = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(2):
        step_of(wl, wl.batch.seq_lens.tolist())
        torch.cuda.synchronize()
        outs = [call(wl, kept, stream=s) for s in side]
        wl.batch = dataclasses.replace(wl.batch)
        filler = [torch.full((2048,), -1, dtype=torch.int32, device=gpu) for _ in range(50)]
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o, want)
        del filler


def test_captured_prompts_follow_the_lengths(gpu):
    """A replay cuts the prompt by the lengths of its time."""
    wl, members = shared_case([700, 0], [9, 1, 40, 5900, 5300], [0, 0, 0, 1, 0],
                              ext=[1, 1, 1, 200, 1], seed=64)
    kept = SharedPrefixes(members)
    step_of(wl, [709, 701, 740, 200, 6000])
    call(wl, kept)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(wl, kept)
    lens = wl.batch.seq_lens
    for prompt in (5900, 200, 1700, 5900):
        lens.copy_(torch.tensor([709, 701, 740, prompt, 6000]))
        out.fill_(float("nan"))
        filler = [torch.full((2048,), -1, dtype=torch.int32, device=gpu) for _ in range(20)]
        graph.replay()
        torch.cuda.synchronize()
        wl.batch = dataclasses.replace(wl.batch)
        assert torch.equal(out, call(wl, SharedPrefixes(members))), prompt
        right(wl, out, f"replayed {prompt}")
        del filler
