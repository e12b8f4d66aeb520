"""scored_attention: the attention of slot_based_attention, and weights against 64 bits."""
import pytest
import torch

from tests.helpers import small_case
from tests.part_oracle import assert_attention, attention64, score_error
from tokenfactory_amd import scored_attention, slot_based_attention, workloads

pytestmark = pytest.mark.gpu


def case(seq, ext, heads=(24, 4), d=256, seed=0, fp8=False, **kw):
    return workloads.build("scored", seq, ext, num_q_heads=heads[0], num_kv_heads=heads[1],
                           head_dim=d, pool_slots=2 * sum(seq) + 64, device="cuda", seed=seed,
                           kv_fp8=fp8, **kw)


def call(wl, scores, **kw):
    return scored_attention(wl.q, wl.k_pool, wl.v_pool, wl.batch, scores, scaling=wl.scale,
                            k_scale=wl.k_scale, v_scale=wl.v_scale, **kw)


def new_scores(wl, fill=None):
    table = wl.batch.req_to_token
    if fill is None:
        gen = torch.Generator("cuda").manual_seed(7)
        return torch.rand(table.shape, generator=gen, device="cuda")
    return torch.full(table.shape, fill, device="cuda")


def assert_scores(got, before, wl, weights, add, lens=None, window=None, what=""):
    """Relative bound of a weight: twice a score's (its own and that of the row's sum), of
    the sum of 2^s, whose additions and rescalings are fewer than keys / 32 + 64 deep and
    round by 2^-22 each, and N fp32 additions of positive terms; then one rounding where
    it is added to a score.  Weights below 2^-100 may vanish.  Everything else stays."""
    lens = lens or wl.seq_lens
    got, before = got.double().cpu(), before.double().cpu()
    touched = torch.zeros_like(got, dtype=torch.bool)
    for b, (row, n, w) in enumerate(zip(wl.rows, lens, weights)):
        terms = wl.num_q_heads * min(wl.ext_lens[b], window or wl.ext_lens[b])
        rel = 2 * score_error(wl) + (n / 32 + 64) * 2.0 ** -22 + terms * 2.0 ** -24
        want = w + (before[row, :n] if add else 0)
        bound = w * rel * 1.01 + want * 2.0 ** -24 + 2.0 ** -100
        err = (got[row, :n] - want).abs()
        assert (err <= bound).all(), f"{what} request {b}: {(err / bound).max():.2f} of its bound"
        touched[row, :n] = True
    assert torch.equal(got[~touched], before[~touched]), what


def check(wl, window=32, add=True, what=""):
    print(f"[scored] {what}", flush=True)
    scores = new_scores(wl)
    before = scores.clone()
    got = call(wl, scores, window=window, add=add)
    want, spread, weights = attention64(wl, window)
    assert_attention(got, want, spread, wl, what)
    assert_scores(scores, before, wl, weights, add, window=window, what=what)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads", [(24, 4), (16, 2), (6, 1), (8, 8), (20, 1), (34, 2)])
def test_head_layouts(gpu, heads, fp8):
    wl = case([5, 1, 140, 17, 300], [1] * 5, heads=heads, seed=1, fp8=fp8)
    check(wl, what=f"{heads} fp8={fp8}")


@pytest.mark.parametrize("d,fp8", [(128, False), (128, True), (64, False), (64, True), (32, False),
                                   (80, False), (192, False), (208, True), (8, False), (16, True),
                                   (40, True), (24, False)])
@pytest.mark.parametrize("ext", [1, 9])
def test_head_dims(gpu, d, fp8, ext):
    wl = case([ext + 3, ext, 150, 33], [ext] * 4, heads=(12, 3), d=d, seed=d, fp8=fp8)
    check(wl, window=5, add=ext == 1, what=f"D={d} fp8={fp8} ext={ext}")


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 127, 128, 129, 255, 257, 1024, 2049, 9001])
def test_decode_lengths(gpu, n):
    check(case([n], [1], seed=n), what=f"one request of {n}")
    if n < 3000:
        check(case([n, 3, n + 5, 64], [1] * 4, seed=n), add=False, what=f"{n} in a batch")


@pytest.mark.parametrize("window", [1, 2, 7, 32, 1000])
@pytest.mark.parametrize("fp8", [False, True])
def test_windows(gpu, window, fp8):
    """Prompts, chunks behind a prefix, turns shorter than the window and decodes."""
    wl = case([70, 200, 140, 5, 90, 33], [70, 40, 1, 5, 2, 33], seed=window, fp8=fp8)
    check(wl, window=window, add=window % 2 == 0, what=f"window {window}")


def test_one_prompt(gpu):
    check(case([333], [333], seed=2), window=16, what="one prompt")
    check(case([333], [1], seed=2), window=16, what="one decode")


@pytest.mark.parametrize("d", [256, 128])
def test_large_scores(gpu, d):
    """Softmax that is one key, with a maximum of several hundred."""
    check(case([600, 90], [1, 1], d=d, seed=3, q_std=40.0), what="large scores")
    check(case([600, 90], [20, 9], d=d, seed=3, q_std=40.0), what="large scores, prompts")


@pytest.mark.parametrize("d", [256, 64])
def test_weights_of_a_request_sum_to_its_heads(gpu, d):
    wl = case([4000, 1000, 77], [1, 1, 1], d=d, seed=4)
    scores = new_scores(wl, 0.0)
    call(wl, scores)
    again = new_scores(wl, 0.0)
    call(wl, again)
    assert torch.equal(scores, again)   # the same sums in the same order
    call(wl, again)                     # another layer: adds up
    for row in wl.rows:
        assert abs(scores[row].double().sum().item() - 24) < 24 * 4100 * 2.0 ** -22
    assert (again - 2 * scores).abs().max() <= scores.max() * 2.0 ** -22


@pytest.mark.parametrize("ext", [1, 4])
@pytest.mark.parametrize("d", [256, 128])
def test_empty_requests_and_changed_lengths(gpu, ext, d):
    """Lengths in place: padding requests get zeros and leave their scores alone."""
    wl = case([200, 90, 60, 300], [ext] * 4, d=d, seed=5)
    for lens in ([200, 0, 60, 7], [0, 90, 1, 300], [13, 14, 15, 16]):
        wl.batch.seq_lens.copy_(torch.tensor(lens))
        scores = new_scores(wl)
        before = scores.clone()
        got = call(wl, scores, window=3)
        want, spread, weights = attention64(wl, 3, seq_lens=lens)
        if ext == 1:
            assert_attention(got, want, spread, wl, f"{lens}")
        assert_scores(scores, before, wl, weights, True, lens=lens, window=3, what=f"{lens}")


@pytest.mark.parametrize("d,fp8", [(256, False), (256, True), (128, False)])
@pytest.mark.parametrize("ext", [1, 3])
def test_masked_values(gpu, d, fp8, ext):
    """NaN and large values in unused slots leave everything alone; in a later token's
    key, the rows before it."""
    wl = case([50, 77], [ext, ext], d=d, seed=6, fp8=fp8)
    scores = new_scores(wl)
    before = scores.clone()
    table = wl.batch.req_to_token
    bad = torch.ones(wl.k_pool.shape[0], dtype=torch.bool, device=gpu)
    bad[table[table >= 0].unique()] = False
    want, spread, weights = attention64(wl, 2)
    nan = torch.tensor(float("nan"), device=gpu).to(wl.k_pool.dtype)
    wl.k_pool[bad], wl.v_pool[bad] = nan, nan
    got = call(wl, scores, window=2)
    assert_attention(got, want, spread, wl, "unused slots")
    assert_scores(scores, before, wl, weights, True, window=2, what="unused slots")
    # A NaN key makes every weight of the rows that see it NaN, and no other request's.
    wl.k_pool[table[wl.rows[0], 10]] = nan
    scores = before.clone()
    call(wl, scores, window=2)
    assert torch.isnan(scores[wl.rows[0], :50]).all()
    assert torch.equal(scores[wl.rows[0], 50:], before[wl.rows[0], 50:])
    assert not torch.isnan(scores[wl.rows[1]]).any()


@pytest.mark.parametrize("ext", [1, 5])
def test_gate_amax_out_and_strides(gpu, ext):
    wl = case([150, 40], [ext, ext], heads=(12, 2), d=256, seed=8)
    plain = call(wl, new_scores(wl, 0.0))
    table = wl.batch.req_to_token
    wide = torch.full((table.shape[0] + 2, table.shape[1] + 5), 3.0, device=gpu)
    gate = torch.randn((2 * ext, 12, 512), device=gpu).to(torch.bfloat16)[:, :, 256:]
    amax = torch.zeros(1, dtype=torch.int32, device=gpu)
    out = torch.full((2 * ext, 13, 256), 7.0, dtype=torch.bfloat16, device=gpu)
    q = torch.zeros((2 * ext, 12, 264), dtype=torch.bfloat16, device=gpu)
    q[:, :, :256] = wl.q
    wl.q = q[:, :, :256]
    got = call(wl, wide, add=False, gate=gate, out_amax=amax, out=out[:, :12])
    assert got.data_ptr() == out.data_ptr() and (out[:, 12] == 7).all()
    silu = torch.nn.functional.silu(gate.float()).to(torch.bfloat16)
    want = (plain.float() * silu.float()).to(torch.bfloat16).float()
    assert ((got.float() - want).abs() <= 2.0 ** -7 * want.abs()).all()   # silu: one ulp of bf16
    bits = got.contiguous().view(torch.int16).to(torch.int32) & 0x7FFF
    assert amax.item() == bits.max().item()
    _, _, weights = attention64(wl, 32)
    before = torch.full_like(wide, 3.0)
    assert_scores(wide, before, wl, weights, False, window=32)


@pytest.mark.parametrize("ext", [1, 3])
def test_captured_and_replayed(gpu, ext):
    """Replays follow lengths and queries in place, with eager work between them."""
    wl = case([300, 40, 500], [ext] * 3, seed=9)
    lens = wl.batch.seq_lens
    scores = new_scores(wl, 0.0)
    call(wl, scores)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(wl, scores)
    for step in range(4):
        lens.copy_(torch.tensor([300 - step, 40 + step, 500 - 100 * step]))
        wl.q.copy_(torch.randn_like(wl.q))
        scores.fill_(step)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.full_like(scores, step)
        want = call(wl, eager)
        assert torch.equal(out, want) and torch.equal(scores, eager), step


def test_streams(gpu):
    wl = case([900, 300, 77], [1, 1, 1], seed=10)
    tables = [new_scores(wl) for _ in range(4)]
    want = call(wl, tables[0])
    torch.cuda.synchronize()
    outs = [call(wl, t, stream=torch.cuda.Stream()) for t in tables[1:]]
    filler = [torch.full((1 << 18,), float("nan"), device=gpu) for _ in range(20)]
    torch.cuda.synchronize()
    for o, t in zip(outs, tables[1:]):
        assert torch.equal(o, want) and torch.equal(t, tables[0])
    del filler


def test_output_is_the_plain_calls(gpu):
    """At head_dim 256, prompts: the attention itself is slot_based_attention's."""
    wl = case([300, 140], [300, 40], seed=11)
    want = slot_based_attention(wl.q, wl.k_pool, wl.v_pool, wl.batch, scaling=wl.scale)
    assert torch.equal(call(wl, new_scores(wl)), want)


def test_many_requests(gpu):
    b = 2048
    wl = small_case([1 + i % 40 for i in range(b)], [1] * b, hq=2, hkv=1, d=64, seed=17,
                    device=gpu, dtype=torch.bfloat16)
    check(wl, add=False, what="2048 requests")


def test_slots_behind_2_gib(gpu):
    wl = case([60, 9], [1, 1], seed=16)
    slots = 1_300_000            # x 2 KB
    want, spread, weights = attention64(wl, 32)
    n = wl.k_pool.shape[0]
    k = torch.empty((slots, 4, 256), dtype=torch.bfloat16, device=gpu)
    v = torch.empty_like(k)
    k[slots - n:], v[slots - n:] = wl.k_pool, wl.v_pool
    table = wl.batch.req_to_token
    table[table >= 0] += slots - n
    small = (wl.k_pool, wl.v_pool)
    wl.k_pool, wl.v_pool = k, v
    scores = new_scores(wl)
    before = scores.clone()
    got = call(wl, scores)
    wl.k_pool, wl.v_pool = small
    assert_attention(got, want, spread, wl, "far slots")
    assert_scores(scores, before, wl, weights, True, what="far slots")


@pytest.mark.parametrize("ext", [[1, 1], [7, 70]])
@pytest.mark.parametrize("heads,d", [((24, 4), 256), ((32, 8), 128)])
def test_slots_behind_4_gib(gpu, heads, d, ext):
    wl = case([60, 90], ext, heads=heads, d=d, seed=17)
    want, spread, weights = attention64(wl, 32)
    n = wl.k_pool.shape[0]
    slots = (1 << 32) // (2 * heads[1] * d) + 1 + n
    k = torch.empty((slots, heads[1], d), dtype=torch.bfloat16, device=gpu)
    v = torch.empty_like(k)
    k[slots - n:], v[slots - n:] = wl.k_pool, wl.v_pool
    table = wl.batch.req_to_token
    table[table >= 0] += slots - n
    small = (wl.k_pool, wl.v_pool)
    wl.k_pool, wl.v_pool = k, v
    scores = new_scores(wl)
    before = scores.clone()
    got = call(wl, scores)
    wl.k_pool, wl.v_pool = small
    assert_attention(got, want, spread, wl, f"far slots {heads} {ext}")
    assert_scores(scores, before, wl, weights, True, window=32, what=f"far slots {heads} {ext}")


def test_refusals(gpu):
    """Raised on the host before anything is launched: the scores stay."""
    wl = case([9, 30, 4], [1, 1, 1], seed=30)
    scores = new_scores(wl, 0.0)

    def refused(match, error=ValueError, **kw):
        with pytest.raises(error, match=match):
            call(wl, scores, **kw)

    refused("window", window=0)
    refused("out must match", out=torch.empty_like(wl.q)[:2])
    refused("gate", gate=torch.empty_like(wl.q, dtype=torch.float32))
    refused("out_amax", out_amax=torch.zeros(1, device=gpu))
    wl.batch.req_pool_indices_list = [1, 2, 1]
    refused("twice")
    wl.batch.req_pool_indices_list = None
    wl.batch.extend_lens, wl.batch.max_extend_len = [1, 2], 1
    refused("decode batch of 3")
    wl.batch.extend_lens, wl.batch.max_extend_len = [1, 1, 1], 2
    wl.batch.extend_lens_tensor = wl.batch.extend_lens_tensor.to(torch.int32)
    refused("extend_lens_tensor")
    assert not scores.any()
    wl = case([9, 30], [1, 1], seed=31, fp8=True)
    with pytest.raises(ValueError, match="k_scale"):
        scored_attention(wl.q, wl.k_pool, wl.v_pool, wl.batch, new_scores(wl))
