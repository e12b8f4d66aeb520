"""shared_prefix_attention against attention in 64 bits, over layouts, types and masks."""
import pytest
import torch

from tests.helpers import small_case
from tests.part_oracle import assert_attention, attention64
from tokenfactory_amd import SharedPrefixes, shared_prefix_attention, slot_based_attention, workloads

pytestmark = pytest.mark.gpu


def shared_case(prefixes, own, groups, ext=None, heads=(24, 4), d=256, seed=0, fp8=False,
                device="cuda", q_std=1.0):
    """(workload, its groups): request b holds prefixes[groups[b]] shared keys and own[b]."""
    ext = ext or [1] * len(own)
    seq = [prefixes[g] + n for g, n in zip(groups, own)]
    wl = workloads.build("shared", seq, ext, num_q_heads=heads[0], num_kv_heads=heads[1],
                         head_dim=d, pool_slots=2 * sum(seq) + 64, device=device, seed=seed,
                         prefix_groups=groups, shared_prefix_lens=prefixes, kv_fp8=fp8,
                         q_std=q_std)
    members = [([b for b, x in enumerate(groups) if x == g], n) for g, n in enumerate(prefixes)]
    return wl, members


def call(wl, shared, **kw):
    return shared_prefix_attention(wl.q, wl.k_pool, wl.v_pool, wl.batch, shared,
                                   scaling=wl.scale, k_scale=wl.k_scale, v_scale=wl.v_scale, **kw)


def check(wl, groups, what=""):
    print(f"[shared] {what}", flush=True)
    got = call(wl, SharedPrefixes(groups))
    want, spread, _ = attention64(wl)
    assert_attention(got, want, spread, wl, what)
    return got


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads", [(24, 4), (16, 2), (6, 1), (8, 8), (20, 1), (34, 2)])
def test_head_layouts(gpu, heads, fp8):
    wl, groups = shared_case([300], [5, 1, 40, 17, 16], [0] * 5, heads=heads, seed=1, fp8=fp8)
    check(wl, groups, f"{heads} fp8={fp8}")


@pytest.mark.parametrize("d,fp8", [(128, False), (128, True), (64, False), (64, True), (32, False),
                                   (80, False), (192, False), (208, True), (8, False), (16, True),
                                   (40, True)])
def test_head_dims(gpu, d, fp8):
    wl, groups = shared_case([130, 47], [5, 1, 60, 17, 16, 33, 2], [0, 1, 0, 1, 0, 0, 1],
                             heads=(12, 3), d=d, seed=d, fp8=fp8)
    check(wl, groups, f"D={d} fp8={fp8}")


@pytest.mark.parametrize("prefix", [1, 15, 16, 17, 31, 33, 255, 256, 257, 1023, 1025, 2047, 2049,
                                    4133])
def test_prefix_lengths(gpu, prefix):
    wl, groups = shared_case([prefix], [1, 2, 9], [0] * 3, seed=prefix)
    check(wl, groups, f"prefix {prefix}")


@pytest.mark.parametrize("members", [2, 3, 5, 43, 90])
def test_group_sizes(gpu, members):
    """Row blocks of the shared part: 6 rows a member."""
    wl, groups = shared_case([777], [1 + 7 * b % 50 for b in range(members)], [0] * members,
                             heads=(6, 1), seed=members)
    check(wl, groups, f"{members} members")


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("d", [256, 128])
def test_several_tokens_and_groups(gpu, d, fp8):
    """Verify steps of different lengths, groups interleaved in the batch, an empty and a
    single-member group, and requests outside of any."""
    groups = [0, 1, 2, 0, 1, 3, 0, 4, 1]
    ext = [4, 1, 2, 3, 1, 5, 10, 1, 6]
    own = [9, 1, 30, 3, 200, 5, 11, 64, 6]
    wl, members = shared_case([500, 90, 60, 0, 35], own, groups, ext=ext, d=d, seed=5, fp8=fp8)
    check(wl, members, f"several D={d} fp8={fp8}")


@pytest.mark.parametrize("d", [256, 64])
def test_beside_long_prompts(gpu, d):
    """A prompt chunk in a group, and one outside, beside decodes that share."""
    wl, members = shared_case([400, 0], [1, 70, 20, 3, 100], [0, 0, 0, 0, 1],
                              ext=[1, 70, 1, 3, 100], d=d, seed=9)
    check(wl, members, f"prompts D={d}")


def test_large_scores(gpu):
    """Scores of several hundred: the parts' maxima differ by far more than fp32 holds."""
    wl, members = shared_case([600], [40, 3, 1], [0] * 3, seed=3, q_std=40.0)
    check(wl, members, "large scores")


def test_equal_to_the_unshared_call(gpu):
    """Same inputs, same answer up to the last bits, on a large group."""
    wl, members = shared_case([3000], [1 + 13 * b for b in range(70)], [0] * 70, seed=4)
    got = call(wl, SharedPrefixes(members)).float()
    want = slot_based_attention(wl.q, wl.k_pool, wl.v_pool, wl.batch, scaling=wl.scale).float()
    # both round P and the result to bf16 (see assert_attention); spread <= max |v| here
    bound = 2.0 ** -7 * want.abs() + 2.0 ** -7 * 1.1 * 0.9
    assert ((got - want).abs() <= bound).all()
    again = call(wl, SharedPrefixes(members)).float()
    assert torch.equal(got, again)


def test_nothing_shared_is_the_plain_call(gpu):
    wl, _ = shared_case([64], [5, 9], [0, 0], seed=6)
    want = slot_based_attention(wl.q, wl.k_pool, wl.v_pool, wl.batch, scaling=wl.scale)
    for groups in ([], [([0], 64)], [([0, 1], 0)], [([], 5)]):
        assert torch.equal(call(wl, SharedPrefixes(groups)), want)


@pytest.mark.parametrize("d", [256, 128])
def test_padding_and_short_members(gpu, d):
    """A padding request (length 0) in a group gets zeros; a member whose context ends
    inside the shared part sees its own keys alone; one outside with a length of 0."""
    wl, members = shared_case([200, 0], [5, 8, 1, 30, 4], [0, 0, 0, 0, 1], d=d, seed=7,
                              ext=[1, 3, 1, 2, 1])
    shared = SharedPrefixes(members)
    for lens in ([205, 208, 0, 100, 4], [0, 2, 1, 1, 0], [205, 199, 17, 230, 3]):
        wl.batch.seq_lens.copy_(torch.tensor(lens))
        want, spread, _ = attention64(wl, seq_lens=lens)
        got = call(wl, shared)
        assert_attention(got, want, spread, wl, f"lens {lens}")
        at = 0
        for n, e in zip(lens, wl.ext_lens):
            for t in range(e):
                if n - e + t + 1 <= 0:
                    assert (got[at + t] == 0).all()
            at += e


@pytest.mark.parametrize("d,fp8", [(256, False), (256, True), (128, False)])
def test_values_that_rows_do_not_see(gpu, d, fp8):
    """NaN and infinities in unused slots, in slot 0 and in tokens later than a row's own
    stay with the rows that see them."""
    wl, members = shared_case([77], [6, 9, 12], [0] * 3, ext=[4, 1, 6], d=d, seed=8, fp8=fp8)
    want, spread, _ = attention64(wl)
    table = wl.batch.req_to_token
    used = table[table >= 0].unique()
    bad = torch.ones(wl.k_pool.shape[0], dtype=torch.bool, device=gpu)
    bad[used] = False
    nan = torch.tensor(float("nan"), device=gpu).to(wl.k_pool.dtype)
    k, v = wl.k_pool.clone(), wl.v_pool.clone()
    k[bad], v[bad] = nan, nan
    wl.k_pool, wl.v_pool = k, v
    assert_attention(call(wl, SharedPrefixes(members)), want, spread, wl, "unused slots")
    # request 0's last token: its rows 0 .. 2 do not see it
    slot = table[wl.rows[0], wl.seq_lens[0] - 1]
    v[slot] = nan
    k[slot, 0] = nan
    got = call(wl, SharedPrefixes(members))
    rows = [0, 1, 2] + list(range(4, got.shape[0]))
    assert torch.isnan(got[3].float()).all()
    got[3] = 0
    for t in (want, spread):
        t[3] = 0
    assert_attention(got, want, spread, wl, "later token")
    if not fp8:
        v[slot] = float("inf")
        k[slot, 0] = 0
        got = call(wl, SharedPrefixes(members))
        assert (got[3].float() == float("inf")).all()
        assert torch.isfinite(got[rows].float()).all()


def test_infinite_scores_of_masked_keys(gpu):
    """A key of the type's largest value, behind what the other rows see."""
    wl, members = shared_case([50], [4, 7], [0] * 2, ext=[3, 2], seed=12)
    big = torch.finfo(torch.bfloat16).max
    slot = wl.batch.req_to_token[wl.rows[1], wl.seq_lens[1] - 1]
    want, spread, _ = attention64(wl)
    wl.k_pool[slot] = big
    wl.v_pool[slot] = big
    got = call(wl, SharedPrefixes(members))
    keep = [0, 1, 2, 3]
    wl2 = wl
    got, want, spread = got[keep], want[keep], spread[keep]
    wl2.k_pool = wl.k_pool.clone()
    wl2.k_pool[slot] = 0
    assert_attention(got, want, spread, wl2, "masked key")


@pytest.mark.parametrize("d,fp8", [(256, False), (256, True), (64, False)])
def test_gate_amax_out_and_strides(gpu, d, fp8):
    """The output gate, the amax of what is written, an output buffer with a token stride
    whose other columns stay, and queries with strided heads."""
    wl, members = shared_case([150], [5, 9, 33], [0] * 3, ext=[1, 2, 1], heads=(12, 2), d=d,
                              seed=11, fp8=fp8)
    plain = call(wl, SharedPrefixes(members))
    gate = torch.randn((4, 12, 2 * d), device=gpu).to(torch.bfloat16)[:, :, d:]
    amax = torch.zeros(1, dtype=torch.int32, device=gpu)
    wide = torch.full((4, 13, d), 7.0, dtype=torch.bfloat16, device=gpu)
    q = torch.zeros((4, 12, d + 8), dtype=torch.bfloat16, device=gpu)
    q[:, :, :d] = wl.q
    wl.q = q[:, :, :d]
    got = call(wl, SharedPrefixes(members), gate=gate, out_amax=amax, out=wide[:, :12])
    assert got.data_ptr() == wide.data_ptr() and (wide[:, 12] == 7).all()
    silu = torch.nn.functional.silu(gate.float()).to(torch.bfloat16)
    want = (plain.float() * silu.float()).to(torch.bfloat16).float()
    assert ((got.float() - want).abs() <= 2.0 ** -7 * want.abs()).all()   # silu: one ulp of bf16
    bits = got.contiguous().view(torch.int16).to(torch.int32) & 0x7FFF
    assert amax.item() == bits.max().item()


def test_captured_and_replayed(gpu):
    """A captured call follows lengths, queries and slots in place; every replay equals
    the eager call, with other work between them."""
    wl, members = shared_case([300], [40, 50, 60], [0] * 3, seed=13)
    shared = SharedPrefixes(members)
    lens = wl.batch.seq_lens
    full = lens.clone()
    eager = call(wl, shared)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(wl, shared)
    del shared   # (the graph keeps what it reads)
    for step in range(4):
        lens.copy_(full - 3 * step)
        wl.q.copy_(torch.randn_like(wl.q))
        filler = [torch.full((4096,), -1, dtype=torch.int32, device=gpu) for _ in range(20)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = call(wl, SharedPrefixes(members))
        assert torch.equal(out, eager), step
        del filler


def test_capture_needs_an_eager_call(gpu):
    wl, members = shared_case([30], [4, 5], [0] * 2, seed=14)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="once before"):
        with torch.cuda.graph(graph):
            call(wl, SharedPrefixes(members))
    torch.cuda.synchronize()


def test_streams(gpu):
    """Lists uploaded by one stream, read by others, dropped while they run."""
    wl, members = shared_case([900], [40, 50, 60, 7], [0] * 4, seed=15)
    want = call(wl, SharedPrefixes(members))
    shared = SharedPrefixes(members)
    side = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = [call(wl, shared, stream=s) for s in side]
    del shared
    filler = [torch.full((2048,), -1, dtype=torch.int32, device=gpu) for _ in range(50)]
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)
    del filler


def test_slots_behind_2_gib(gpu):
    """Slots whose byte offsets pass 32 bits."""
    wl, members = shared_case([60], [5, 9], [0] * 2, seed=16)
    slots = 1_300_000            # x 2 KB
    want, spread, _ = attention64(wl)
    n = wl.k_pool.shape[0]
    k = torch.empty((slots, 4, 256), dtype=torch.bfloat16, device=gpu)
    v = torch.empty_like(k)
    k[slots - n:], v[slots - n:] = wl.k_pool, wl.v_pool
    table = wl.batch.req_to_token
    table[table >= 0] += slots - n
    small = (wl.k_pool, wl.v_pool)
    wl.k_pool, wl.v_pool = k, v
    got = call(wl, SharedPrefixes(members))
    wl.k_pool, wl.v_pool = small
    assert_attention(got, want, spread, wl, "far slots")


@pytest.mark.parametrize("heads,d,members", [((24, 4), 256, 3), ((32, 8), 128, 5),
                                             ((16, 8), 128, 2), ((24, 4), 192, 3)])
def test_slots_behind_4_gib(gpu, heads, d, members):
    """Tiles of 256 and of 128 dims, and streamed parts, behind 2^32 bytes."""
    wl, groups = shared_case([60], [5, 9, 1, 33, 2][:members], [0] * members, heads=heads, d=d,
                             seed=18)
    want, spread, _ = attention64(wl)
    n = wl.k_pool.shape[0]
    slots = (1 << 32) // (2 * heads[1] * d) + 1 + n
    k = torch.empty((slots, heads[1], d), dtype=torch.bfloat16, device=gpu)
    v = torch.empty_like(k)
    k[slots - n:], v[slots - n:] = wl.k_pool, wl.v_pool
    table = wl.batch.req_to_token
    table[table >= 0] += slots - n
    small = (wl.k_pool, wl.v_pool)
    wl.k_pool, wl.v_pool = k, v
    got = call(wl, SharedPrefixes(groups))
    wl.k_pool, wl.v_pool = small
    assert_attention(got, want, spread, wl, f"far slots {heads} D={d}")


@pytest.mark.parametrize("d", [64, 192])
def test_many_requests(gpu, d):
    """As many parts as one launch takes; at 192 dims, where the shared ones are parts too,
    more than that: the unshared path answers."""
    b = 2000
    wl = small_case([40] * b, [1] * b, hq=2, hkv=1, d=d, seed=17, device=gpu,
                    dtype=torch.bfloat16, groups=[0] * b, prefixes=[30])
    groups = [(list(range(b)), 30)]
    if d == 64:
        check(wl, groups, "2000 requests")
    else:
        want = slot_based_attention(wl.q, wl.k_pool, wl.v_pool, wl.batch, scaling=wl.scale)
        assert torch.equal(call(wl, SharedPrefixes(groups)), want)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads", [(24, 4), (16, 2), (6, 1), (8, 8), (20, 1), (34, 2)])
def test_long_prefixes_in_pieces(gpu, heads, fp8):
    wl, groups = shared_case([1700], [5, 1, 40, 17, 16], [0] * 5, heads=heads, seed=21, fp8=fp8)
    check(wl, groups, f"pieces {heads} fp8={fp8}")


@pytest.mark.parametrize("prefix", [1537, 1568, 1600, 2047, 2049, 4133, 8191])
def test_long_prefix_lengths(gpu, prefix):
    wl, groups = shared_case([prefix], [1, 2, 9], [0] * 3, heads=(6, 1), seed=prefix)
    check(wl, groups, f"pieces of {prefix}")


@pytest.mark.parametrize("members", [2, 3, 5, 6, 11, 43, 90])
def test_pieces_of_group_sizes(gpu, members):
    """Row blocks of 256, whole waves of them without rows, several groups in one launch."""
    b = 2 * members
    wl, groups = shared_case([1600, 333], [1 + 7 * i % 50 for i in range(b)],
                             [i % 2 for i in range(b)], heads=(6, 1), seed=members)
    check(wl, groups, f"pieces of {members} members")


@pytest.mark.parametrize("fp8", [False, True])
def test_pieces_with_several_tokens_and_prompts(gpu, fp8):
    groups = [0, 1, 2, 0, 1, 0, 0, 1, 0]
    ext = [4, 1, 2, 3, 1, 10, 1, 6, 40]
    own = [9, 1, 30, 3, 200, 11, 64, 6, 50]
    wl, members = shared_case([1900, 90, 0], own, groups, ext=ext, seed=25, fp8=fp8)
    check(wl, members, f"pieces, tokens, fp8={fp8}")


def test_pieces_with_short_members_and_masked_values(gpu):
    """Contexts that end inside the shared part, before its first key, or nowhere near;
    NaN in slots that nothing uses."""
    wl, members = shared_case([1800], [5, 8, 1, 30], [0] * 4, seed=27, ext=[1, 3, 1, 2])
    table = wl.batch.req_to_token
    bad = torch.ones(wl.k_pool.shape[0], dtype=torch.bool, device=gpu)
    bad[table[table >= 0].unique()] = False
    wl.k_pool[bad] = float("nan")
    wl.v_pool[bad] = float("nan")
    shared = SharedPrefixes(members)
    for lens in ([1805, 1808, 0, 1700], [0, 2, 1, 1], [1805, 1799, 17, 1830]):
        wl.batch.seq_lens.copy_(torch.tensor(lens))
        want, spread, _ = attention64(wl, seq_lens=lens)
        assert_attention(call(wl, shared), want, spread, wl, f"lens {lens}")


def test_pieces_large_scores(gpu):
    wl, members = shared_case([1600], [40, 3, 1], [0] * 3, seed=23, q_std=40.0)
    check(wl, members, "pieces, large scores")


def test_pieces_captured_and_replayed(gpu):
    wl, members = shared_case([1600], [40, 50, 60], [0] * 3, seed=13)
    shared = SharedPrefixes(members)
    full = wl.batch.seq_lens.clone()
    call(wl, shared)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(wl, shared)
    for step in range(3):
        wl.batch.seq_lens.copy_(full - 7 * step)
        wl.q.copy_(torch.randn_like(wl.q))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call(wl, SharedPrefixes(members))), step


@pytest.mark.parametrize("d", [128, 64, 32, 80, 8, 120])
@pytest.mark.parametrize("heads", [(32, 8), (6, 1), (34, 2)])
def test_pieces_at_other_head_dims(gpu, d, heads):
    wl, groups = shared_case([1700, 130], [5, 1, 40, 17, 16, 8], [0, 0, 1, 0, 1, 0], heads=heads,
                             d=d, seed=31)
    check(wl, groups, f"pieces {heads} D={d}")


@pytest.mark.parametrize("prefix", [1537, 1600, 1601, 1663, 4133])
def test_piece_lengths_at_128_dims(gpu, prefix):
    wl, groups = shared_case([prefix], [1, 2, 9], [0] * 3, heads=(4, 1), d=128, seed=prefix)
    check(wl, groups, f"pieces of {prefix}, D=128")


@pytest.mark.parametrize("members", [2, 9, 65, 130])
def test_piece_rows_at_128_dims(gpu, members):
    """Row blocks of 256, 4 rows a member; waves and blocks partly filled."""
    wl, groups = shared_case([1600], [1 + 7 * i % 50 for i in range(members)], [0] * members,
                             heads=(4, 1), d=128, seed=members)
    check(wl, groups, f"pieces of {members} members, D=128")


@pytest.mark.parametrize("d", [128, 64])
def test_pieces_with_prompts_at_other_head_dims(gpu, d):
    """Prompt chunks in a group: hundreds of rows of one request, causal in their own part."""
    wl, members = shared_case([1700, 0], [1, 70, 20, 3, 100], [0, 0, 0, 0, 1],
                              ext=[1, 70, 1, 3, 100], heads=(8, 2), d=d, seed=33)
    check(wl, members, f"pieces, prompts, D={d}")


def test_short_members_and_odd_values_at_128_dims(gpu):
    wl, members = shared_case([1800], [5, 8, 1, 30], [0] * 4, seed=37, ext=[1, 3, 1, 2],
                              heads=(8, 2), d=128)
    table = wl.batch.req_to_token
    bad = torch.ones(wl.k_pool.shape[0], dtype=torch.bool, device=gpu)
    bad[table[table >= 0].unique()] = False
    wl.k_pool[bad] = float("nan")
    wl.v_pool[bad] = float("nan")
    shared = SharedPrefixes(members)
    for lens in ([1805, 1808, 0, 1700], [0, 2, 1, 1], [1805, 1799, 17, 1830]):
        wl.batch.seq_lens.copy_(torch.tensor(lens))
        want, spread, _ = attention64(wl, seq_lens=lens)
        assert_attention(call(wl, shared), want, spread, wl, f"lens {lens}")
    # a NaN value of a shared key: NaN for the rows that see it, the others as before
    lens = [1805, 1808, 100, 1700]
    wl.batch.seq_lens.copy_(torch.tensor(lens))
    want, spread, _ = attention64(wl, seq_lens=lens)
    wl.v_pool[table[wl.rows[0], 900]] = float("nan")
    got = call(wl, shared)
    at = [0, 1, 4, 5, 7]       # first q row of each request (new tokens 1, 3, 1, 2)
    assert torch.isnan(got[[0, 1, 2, 3, 5, 6]].float()).all()
    assert_attention(got[4:5], want[4:5], spread[4:5], wl, "a row that ends before it")
    assert at[-1] == got.shape[0]


def test_large_scores_at_128_dims(gpu):
    wl, members = shared_case([1600], [40, 3, 1], [0] * 3, heads=(8, 2), d=128, seed=39,
                              q_std=40.0)
    check(wl, members, "pieces, large scores, D=128")


@pytest.mark.parametrize("d,fp8", [(256, False), (256, True), (128, False)])
def test_many_pairs(gpu, d, fp8):
    """Shared parts of at most 16 rows, streamed with the requests' own: 40 pairs, some of
    contexts that end inside the shared part."""
    groups = [b % 40 for b in range(80)]
    wl, members = shared_case([1 + 17 * g for g in range(40)],
                              [1 + 11 * b % 60 for b in range(80)], groups, d=d, seed=40, fp8=fp8)
    wl.batch.seq_lens[77] = 1 + 17 * 37 - 30
    got = call(wl, SharedPrefixes(members))
    want, spread, _ = attention64(wl, seq_lens=wl.batch.seq_lens.tolist())
    assert_attention(got, want, spread, wl, f"pairs D={d} fp8={fp8}")


@pytest.mark.parametrize("fp8", [False, True])
def test_long_prompts_on_long_contexts(gpu, fp8):
    """A prompt's entries cut over their keys beside decodes that share, then the same plan
    for other lengths, and captured."""
    ext = [1, 1, 1, 1, 30, 1]
    wl, members = shared_case([700, 0], [9, 1, 40, 3, 5000, 2], [0, 0, 0, 0, 1, 0], ext=ext,
                              seed=12, fp8=fp8)
    shared = SharedPrefixes(members)

    def right(got, what):
        want, spread, _ = attention64(wl, seq_lens=wl.batch.seq_lens.tolist())
        assert_attention(got, want, spread, wl, what)

    right(call(wl, shared), "split")
    out = torch.zeros_like(wl.q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(wl, shared, out=out)
    for seq in ([709, 701, 740, 703, 5000, 702], [705, 701, 703, 703, 200, 702],
                [709, 701, 740, 703, 3001, 702], [709, 701, 740, 703, 30, 702]):
        wl.batch.seq_lens.copy_(torch.tensor(seq))
        right(call(wl, shared), f"eager {seq}")
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        right(out, f"replayed {seq}")


def test_negative_scaling(gpu):
    wl, members = shared_case([200], [5, 9, 1, 30], [0] * 4, seed=13)
    wl.scale = -wl.scale
    got = call(wl, SharedPrefixes(members))
    want, spread, _ = attention64(wl)
    assert_attention(got, want, spread, wl, "negative scaling")


def test_refusals(gpu):
    """Raised on the host before anything is launched."""
    wl, members = shared_case([200], [5, 9, 1], [0] * 3, seed=50, fp8=True)
    shared = SharedPrefixes(members)

    def refused(match, **kw):
        with pytest.raises(ValueError, match=match):
            call(wl, shared, **kw)

    refused("out must match", out=torch.empty_like(wl.q)[:2])
    refused("gate", gate=torch.empty_like(wl.q, dtype=torch.float32))
    refused("out_amax", out_amax=torch.zeros(1, device=gpu))
    with pytest.raises(ValueError, match="k_scale"):
        shared_prefix_attention(wl.q, wl.k_pool, wl.v_pool, wl.batch, shared)
    with pytest.raises(ValueError, match="batch of 3"):
        call(wl, SharedPrefixes([([0, 3], 10)]))
    with pytest.raises(ValueError, match="width"):
        call(wl, SharedPrefixes([([0, 1], 100000)]))
    wl.batch.extend_lens = [1, 1, 2]
    refused("extend_lens")
