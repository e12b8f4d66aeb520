"""The operators as a decoder layer uses them (``qwen3_8/decoder_layer.py:57-81``):
norm, attention, residual sum and norm handed on quantised, gated feed-forward, sum
and norm, output projection.  Each stage is compared with the float64 oracle of that
stage on the values that the stage before really gave it, with the stage's own
tolerance; the whole run is captured, replayed, and run by two threads at once.
"""
import threading

import pytest
import torch

from oracle import block_fp8 as ob
from tests import module_golden as mg
from tests import test_gpu_add_norm as norm_test
from tests import test_gpu_gated_mlp as mlp_test
from tests.test_gpu_block_fp8 import make_weight, make_x
from tests.test_gpu_module import _Pool
from tokenfactory_amd import (FullAttention, GatedMLP, add_rms_norm, block_scaled_linear,
                              gated_mlp, quantize_blocks)

pytestmark = pytest.mark.gpu
EPS = norm_test.EPS


def linear_close(out, x, w, s):
    ref, bound = ob.product(x, ob.dequantize_weight(w, s))
    err = (out.double().cpu() - ref).abs()
    limit = 2.0 ** -8 * ref.abs() + (1 + 2.0 ** -8) * bound + 2.0 ** -22 * ref.abs()
    assert bool((err <= limit).all())


@pytest.mark.parametrize("name", mg.CASES)
def test_attention_then_feed_forward(gpu, name):
    """A layer of the reference's small model: ragged extends, decodes, one request."""
    print(f"[layer] {name}", flush=True)
    d, meta = mg.load()
    cfg = mg.config(meta)
    cfg.intermediate_size = 112
    cfg.quantization_config = {"quant_method": "fp8", "weight_block_size": [128, 128]}
    attn = FullAttention(mg.config(meta), layer_idx=3, dtype=torch.bfloat16).to(gpu)
    mg.load_weights(attn, d)
    mlp = GatedMLP(cfg).to(gpu)
    host = []
    for i, lin in enumerate((mlp.gate_proj, mlp.up_proj, mlp.down_proj)):
        w, s = make_weight(lin.out_features, lin.in_features, i)
        host.append((w, s))
        lin.weight.data.copy_(w.to(gpu))
        lin.weight_scale_inv.data.copy_(s.to(gpu))
    hidden = mg.bf16(d[f"{name}_hidden"]).to(torch.bfloat16)
    cols = hidden.shape[1]
    w0, w1, w2 = (norm_test.weights(cols, i) for i in range(3))
    head, head_s = make_weight(96, cols, 7)
    pos = torch.from_numpy(d[f"{name}_positions"]).to(gpu)
    with torch.no_grad():
        y, r0 = add_rms_norm(hidden.to(gpu), None, w0.to(gpu), EPS)
        a = attn(y, pos, _Pool(d, gpu), mg.batch(d, meta, name, gpu))
        (q, s), r1 = add_rms_norm(a, r0, w1.to(gpu), EPS, quantize=True)
        f = mlp(q, s)
        z, r2 = add_rms_norm(f, r1, w2.to(gpu), EPS)
        out = block_scaled_linear(z, head.to(gpu), head_s.to(gpu))
    norm_test.compare(y, r0, hidden, None, w0, None, None, 1.0, False)
    norm_test.compare((q, s), r1, a.cpu(), r0.cpu(), w1, None, None, 1.0, True)
    mlp_test.compare(f.double().cpu(), ob.dequantize(q.cpu(), s.cpu()), host)
    norm_test.compare(z, r2, f.cpu(), r1.cpu(), w2, None, None, 1.0, False)
    linear_close(out, ob.dequantize(*ob.quantize(z.cpu())), head, head_s)


class Layers:
    """Two layers' norms, feed-forward blocks and a projection in attention's place."""

    def __init__(self, gpu, seed, hidden=640, inter=1152, layers=2):
        put = lambda t: t.to(gpu)
        self.layers = []
        for i in range(layers):
            proj = [put(t) for t in make_weight(hidden, hidden, seed + 10 * i)]
            _, ws = mlp_test.make_mlp(hidden, inter, hidden, seed + 10 * i + 1, gpu)
            n1, n2 = (put(norm_test.weights(hidden, seed + 10 * i + j)) for j in (2, 3))
            self.layers.append((proj, ws, n1, n2))

    def __call__(self, x):
        r, (q, s) = x, quantize_blocks(x)
        for proj, ws, n1, n2 in self.layers:
            a = block_scaled_linear(q, *proj, x_scale=s)
            (q, s), r = add_rms_norm(a, r, n1, EPS, quantize=True)
            (q, s), r = add_rms_norm(gated_mlp(q, *ws, x_scale=s), r, n2, EPS, quantize=True,
                                     inplace=True)
        return q, s, r


def same(a, b):
    return torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and all(
        torch.equal(u, v) for u, v in zip(a[1:], b[1:]))


@pytest.mark.parametrize("m", [1, 2, 16, 17, 48, 130, 520])
def test_captured_and_replayed(gpu, m):
    print(f"[layers] captured m={m}", flush=True)
    run = Layers(gpu, 1)
    x = make_x(m, 640, 5).to(gpu)
    run(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(x)
    for seed in range(4):
        x.copy_(make_x(m, 640, 50 + seed))
        graph.replay()
        eager = run(x)              # (its own memory: the graph's results stay)
        torch.cuda.synchronize()
        assert same(out, eager), f"replay {seed}"


@pytest.mark.parametrize("m", [3, 70])
def test_rows_of_a_padded_batch_do_not_change_the_others(gpu, m):
    run = Layers(gpu, 2)
    x = make_x(m, 640, 6).to(gpu)
    want = run(x)
    x2 = x.clone()
    x2[m // 2] = 0.0                # a padding row
    x2[m - 1, 7] = float("nan")
    got = run(x2)
    keep = [i for i in range(m) if i not in (m // 2, m - 1)]
    assert same([t[keep] for t in got], [t[keep] for t in want])
    assert not bool(torch.isnan(got[2][m // 2].float()).any())


def test_two_threads_on_streams_of_their_own(gpu):
    """Calls of two threads at once: no scratch, launch state or error is shared."""
    print("[layers] two threads", flush=True)
    runs = [Layers(gpu, 3), Layers(gpu, 4)]
    xs = [make_x(40, 640, 8).to(gpu), make_x(200, 640, 9).to(gpu)]
    want = [run(x) for run, x in zip(runs, xs)]
    torch.cuda.synchronize()
    bad, errors = [], []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for n in range(30):
                    if not same(runs[i](xs[i]), want[i]):
                        bad.append((i, n))
        except Exception as e:      # pragma: no cover - reported below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and not bad


def test_offsets_past_32_bits(gpu):
    """Rows behind 2^31 elements and 2^32 bytes of inputs, results and scratch."""
    base, rows = make_x(64, 8192, 70), 64 * 4400
    print(f"[large] {rows} x 8192", flush=True)
    x = base.to(gpu).repeat(rows // 64, 1)
    ends = torch.tensor([0, 1, rows // 2 + 3, rows - 2, rows - 1])
    want_x = base[ends % 64]
    q, s = quantize_blocks(x)
    wq, wsc = ob.quantize(want_x)
    assert torch.equal(q.view(torch.uint8)[ends.to(gpu)].cpu(), wq.view(torch.uint8))
    assert torch.equal(s[ends.to(gpu)].cpu(), wsc)
    w = norm_test.weights(8192, 71)
    y, r = add_rms_norm(x, x, w.to(gpu), EPS)
    norm_test.compare(y[ends.to(gpu)], r[ends.to(gpu)], want_x, want_x, w, None, None, 1.0, False)
    del y, r
    w, ws = make_weight(8200, 8192, 72)         # out: 2.3e9 elements
    out = block_scaled_linear(q, w.to(gpu), ws.to(gpu), x_scale=s)
    linear_close(out[ends.to(gpu)], ob.dequantize(wq, wsc), w, ws)
    del out, q, s
    host, dev = mlp_test.make_mlp(256, 8208, 128, 73, gpu)
    out = gated_mlp(x[:, :256], *dev)           # hidden activations: 2.3e9 bytes
    mlp_test.compare(out[ends.to(gpu)].double().cpu(), ob.dequantize(*ob.quantize(want_x[:, :256])),
                     host)
