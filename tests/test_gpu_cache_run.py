"""The cache operators as a serving engine uses them, through the modules: a prompt is
prefilled and scored, requests fork from it and decode on the shared prefix, their own
tokens are scored and evicted, and decoding goes on with the shortened rows."""
import threading
from types import SimpleNamespace

import pytest
import torch

from tests.test_gpu_evict import expected
from tokenfactory_amd import (ForwardBatch, FullAttention, FullAttnKVPool, SharedPrefixes,
                              evict_tokens, scored_attention)
from tokenfactory_amd.req_to_token import DeviceReqToTokenTable

pytestmark = pytest.mark.gpu
HIDDEN = 256


class Engine:
    """Two full-attention layers, a pool, a table and the host's bookkeeping."""

    def __init__(self, gpu, head_dim, heads=(12, 2), fp8=False):
        torch.manual_seed(head_dim)
        cfg = SimpleNamespace(
            hidden_size=HIDDEN, num_attention_heads=heads[0], num_key_value_heads=heads[1],
            head_dim=head_dim, rms_norm_eps=1e-6, partial_rotary_factor=0.25, rope_theta=1e4,
            mrope_section=None, layer_types=["full_attention"] * 2)
        self.heads = heads[0]
        with torch.no_grad():
            self.layers = [FullAttention(cfg, i).to(gpu) for i in range(2)]
        self.pool = FullAttnKVPool.from_config(
            cfg, 8192, gpu, torch.float8_e4m3fn if fp8 else torch.bfloat16)
        if fp8:
            for i in range(2):
                self.pool.set_kv_scales(i, 0.02, 0.02)
        self.table = DeviceReqToTokenTable(8, 4096, gpu)
        self.scores = torch.zeros((8, 4096), device=gpu)
        self.free = torch.randperm(8191)[:].add(1).tolist()
        self.positions = {}          # row -> the next token's position
        self.gpu = gpu
        self.gen = torch.Generator(gpu).manual_seed(1)

    def batch(self, rows, lens, new, **extra):
        """A step of ``new`` tokens behind ``lens`` cached ones, its slots in the table."""
        dev = lambda x: torch.tensor(x, device=self.gpu)
        loc = []
        for row, n, e in zip(rows, lens, new):
            slots = [self.free.pop() for _ in range(e)]
            self.table.tensor[row, n:n + e] = dev(slots)
            loc += slots
        total = [n + e for n, e in zip(lens, new)]
        return ForwardBatch(
            batch_size=len(rows), req_pool_indices=dev(rows), seq_lens=dev(total),
            prefix_lens=dev(lens), extend_lens=list(new), out_cache_loc=dev(loc),
            req_to_token=self.table.tensor, is_prefill=max(new) > 1, max_seq_len=max(total),
            **extra)

    def step(self, batch, hidden=None):
        """Both layers' outputs on random hidden states."""
        rows, new = batch.req_pool_indices_list, batch.extend_lens
        pos = []
        for row, e in zip(rows, new):
            at = self.positions.get(row, 0)
            pos += range(at, at + e)
            self.positions[row] = at + e
        if hidden is None:
            hidden = torch.randn((len(pos), HIDDEN), generator=self.gen,
                                 device=self.gpu).to(torch.bfloat16)
        pos = torch.tensor(pos, device=self.gpu)
        out = []
        with torch.no_grad():
            for layer in self.layers:
                hidden = layer(hidden, pos, self.pool, batch)
                out.append(hidden)
        return out

    def both(self, make, **extra):
        """The step with the batch's extras and without, on the same inputs."""
        before = dict(self.positions)
        plain = make()
        n_tok = sum(plain.extend_lens)
        hidden = torch.randn((n_tok, HIDDEN), generator=self.gen, device=self.gpu)
        want = self.step(plain, hidden.to(torch.bfloat16))
        self.positions = before
        plain.__dict__.update(extra)
        got = self.step(plain, hidden.to(torch.bfloat16))
        return got, want


def close(got, want):
    """Both sides round P and the attention to bf16, then share the same output
    projection: a few bf16 steps of the largest output."""
    for g, w in zip(got, want):
        assert torch.isfinite(g.float()).all()
        assert (g.float() - w.float()).abs().max() <= 2.0 ** -5 * w.float().abs().max()


@pytest.mark.parametrize("head_dim,fp8", [(256, False), (256, True), (128, False), (64, False)])
def test_prompt_fork_decode_evict_decode(gpu, head_dim, fp8):
    print(f"[cache run] D={head_dim} fp8={fp8}", flush=True)
    e = Engine(gpu, head_dim, fp8=fp8)
    prompt = 1800
    # The prompt: its last 32 tokens say what of it matters.
    got, want = e.both(lambda: e.batch([5], [0], [prompt]), token_scores=e.scores)
    close(got, want)
    total = e.scores[5].double().sum().item()
    assert abs(total - 2 * 32 * e.heads) < 2 * 32 * e.heads * 2.0 ** -10
    assert (e.scores[5, prompt:] == 0).all() and (e.scores[:5] == 0).all()

    # Three requests on it, some tokens of their own each.
    rows, lens = [2, 7, 0], [prompt] * 3
    e.table.tensor[rows] = e.table.tensor[5].clone()
    for row in rows:
        e.positions[row] = prompt
    shared = SharedPrefixes([([0, 1, 2], prompt)])
    for new in ([4, 1, 2], [1, 1, 1], [1, 1, 1]):
        got, want = e.both(lambda: e.batch(rows, lens, new), shared_prefixes=shared)
        close(got, want)
        lens = [n + k for n, k in zip(lens, new)]

    # A turn of their own, scored, decodes that add to it, then half of it leaves.
    scores = e.scores
    new = [60, 33, 1]
    got, want = e.both(lambda: e.batch(rows, lens, new), token_scores=scores)
    close(got, want)
    lens = [n + k for n, k in zip(lens, new)]
    for _ in range(3):
        got, want = e.both(lambda: e.batch(rows, lens, [1, 1, 1]), token_scores=scores)
        close(got, want)
        lens = [n + 1 for n in lens]
    want_sum = [2 * e.heads * (min(32, k) + 3) for k in new]
    for row, n, s in zip(rows, lens, want_sum):
        assert abs(scores[row, :n].double().sum().item() - s) < s * 2.0 ** -10
    keep = prompt + 24
    model = expected(e.table.tensor, scores, rows, lens, keep, [prompt] * 3, 8, rows,
                     max(lens) - keep)
    rows_t = torch.tensor(rows, device=gpu)
    new_lens, freed = evict_tokens(e.table.tensor, scores, rows_t, torch.tensor(lens, device=gpu),
                                   keep, max_seq_len=max(lens), first=prompt, recent=8)
    assert new_lens.tolist() == model[0] and torch.equal(freed.cpu(), model[1])
    assert torch.equal(e.table.tensor.cpu(), model[2]) and torch.equal(scores.cpu(), model[3])
    assert new_lens.tolist() == [min(n, keep) for n in lens]
    prefix = set(e.table.tensor[5, :prompt].tolist())
    back = freed[freed >= 0].tolist()
    assert len(set(back)) == len(back) and not prefix & set(back)
    e.free += back
    lens = new_lens.tolist()
    e.table.mark_synced(rows, lens)

    # The prefix is still shared; the freed slots hold new tokens.
    for _ in range(3):
        got, want = e.both(lambda: e.batch(rows, lens, [1, 1, 1]), shared_prefixes=shared)
        close(got, want)
        lens = [n + 1 for n in lens]


def test_decode_run_in_a_graph(gpu):
    """Write, scored decode and eviction of one layer captured together and replayed on new
    tokens equal the eager run."""
    e = Engine(gpu, 256)
    rows, lens = [1, 4], [200, 120]
    e.step(e.batch(rows, [0, 0], lens))
    batch = e.batch(rows, lens, [1, 1], token_scores=e.scores)
    hidden = torch.randn((2, HIDDEN), device=gpu).to(torch.bfloat16)
    pos = torch.tensor([200, 120], device=gpu)
    layer = e.layers[0]

    def run():
        with torch.no_grad():
            out = layer(hidden, pos, e.pool, batch)
        return (out, *evict_tokens(e.table.tensor, e.scores, batch.req_pool_indices,
                                   batch.seq_lens, 150, max_seq_len=201, first=4, recent=16))

    state = (e.table.tensor, e.scores, e.pool.k_buffer, e.pool.v_buffer)
    saved = [t.clone() for t in state]

    def restore():
        for t, s in zip(state, saved):
            t.copy_(s)

    run()
    restore()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for step in range(3):
        hidden.copy_(torch.randn((2, HIDDEN), device=gpu))
        saved[1].uniform_()
        restore()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*captured, *state)]
        restore()
        want = [*run(), *state]
        for a, b in zip(got, want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), step


def test_threads_with_streams_of_their_own(gpu):
    """Two threads, a stream each: one SharedPrefixes object and pool for both, scores and
    tables of their own; every result is the one of a call alone."""
    from tests.test_gpu_shared_prefix import call as shared_call
    from tests.test_gpu_shared_prefix import shared_case

    # a long prompt beside the parts: the second stream is the threads' common one
    wl, members = shared_case([500, 0], [9, 1, 40, 3, 1500], [0, 0, 0, 0, 1],
                              ext=[1, 1, 1, 1, 60], seed=31)
    decode, _ = shared_case([500], [9, 1, 40, 3], [0] * 4, seed=32)
    shared = SharedPrefixes(members)
    table = decode.batch.req_to_token

    def step():
        out = shared_call(wl, shared)
        scores = torch.zeros(table.shape, device=gpu)
        own = table.clone()
        scored = scored_attention(decode.q, decode.k_pool, decode.v_pool, decode.batch, scores)
        lens, freed = evict_tokens(own, scores, decode.batch.req_pool_indices,
                                   decode.batch.seq_lens, 300, max_seq_len=table.shape[1],
                                   first=4, recent=16)
        return out, scored, own, scores, lens, freed

    want = step()
    torch.cuda.synchronize()
    failures = []

    def work():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = step()
                    torch.cuda.current_stream().synchronize()
                    failures.extend(i for i, (a, b) in enumerate(zip(got, want))
                                    if not torch.equal(a, b))
        except Exception as error:   # (a thread's own would be lost)
            failures.append(error)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures
