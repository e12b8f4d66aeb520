"""Performance cases of the block-scaled FP8 operators between two attention layers.

After an attention or Gated DeltaNet layer, a decoder layer adds the layer's
output to the residual stream, norms it, quantises it and runs the gated
feed-forward network.  Activations are e4m3 with one fp32 scale per row and
block of 128 columns, weights e4m3 with one per 128 x 128 block.

* ``quant`` cases call ``quantize_blocks``;
* ``linear`` cases call ``block_scaled_linear``;
* ``norm`` cases call ``add_rms_norm``;
* ``mlp`` cases call ``gated_mlp``.

``own`` False computes the operators from elementary torch operations in fp32.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
AMAX_MIN = 1e-12
EPS = 1e-6
HIDDEN = 5120            # the 27B hybrid layer's
INTER = 17408            # 3.4 x hidden


def _quant(name, rows, cols, fp32=False):
    return _named(name, dict(kind="quant", rows=rows, cols=cols, fp32=fp32))


def _linear(name, rows, n_in, n_out, bias=False, quantized=False):
    return _named(name, dict(kind="linear", rows=rows, n_in=n_in, n_out=n_out, bias=bias,
                             quantized=quantized))


def _norm(name, rows, cols, residual="bf16", post=False, gate="none", scale=1.0, quantize=False):
    return _named(name, dict(kind="norm", rows=rows, cols=cols, residual=residual, post=post,
                             gate=gate, scale=scale, quantize=quantize))


def _mlp(name, rows, hidden, inter, quantized=False):
    return _named(name, dict(kind="mlp", rows=rows, hidden=hidden, inter=inter,
                             quantized=quantized))


def _named(name, case):
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # The activations of a small decode batch, before a projection.
        _quant("quant_decode", 48, 6144),
        # The widest activations of a long prefill.
        _quant("quant_prefill", 8192, INTER),
        # One user's token through an output projection: latency.
        _linear("linear_one", 1, 6144, HIDDEN),
        # A verify step's tokens through one rank's share of a projection with a bias.
        _linear("linear_verify", 77, HIDDEN, 2592, bias=True),
        # A chunk of a prompt through a query projection, quantised by its norm.
        _linear("linear_prompt", 1900, HIDDEN, 12288, quantized=True),
        # Between attention and feed-forward on a decode batch.
        _norm("norm_decode", 48, HIDDEN, quantize=True),
        # Norms on both sides of the block, a gate and an fp32 residual stream, some turns.
        _norm("norm_sandwich", 777, 2560, residual="fp32", post=True, gate="row", scale=0.25),
        # Between attention and feed-forward on a long prefill.
        _norm("norm_prefill", 8192, HIDDEN, quantize=True),
        # One user's token: the weights are read for it alone.
        _mlp("mlp_one", 1, HIDDEN, INTER),
        # A decode batch whose norm quantised it.
        _mlp("mlp_decode", 48, HIDDEN, INTER, quantized=True),
        # One rank's share of the network on a few new turns.
        _mlp("mlp_share", 333, HIDDEN, INTER // 8),
        # A long prefill.
        _mlp("mlp_prefill", 8192, HIDDEN, INTER, quantized=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi, step):
    """A width of the range: a multiple of 128 as a rule, else of ``step``."""
    unit = BLOCK if rng.random() < 0.7 else step
    return unit * max(1, _log_int(rng, lo, hi) // unit)


def draw(rng):
    kind = rng.choice(["quant", "linear", "linear", "norm", "norm", "mlp", "mlp"])
    rows = _log_int(rng, 1, 8192)
    if kind == "quant":
        return _quant(None, rows, _width(rng, 256, INTER, 8), fp32=rng.random() < 0.3)
    if kind == "linear":
        n_in = _width(rng, 512, 8192, 16)
        n_out = _log_int(rng, 64, 16384)
        return _linear(None, rows, n_in, n_out - n_out % rng.choice([1, 4, 128]) or 128,
                       bias=rng.random() < 0.3, quantized=rng.random() < 0.5)
    if kind == "norm":
        return _norm(None, rows, _width(rng, 256, 8192, 8),
                     residual=rng.choice(["bf16", "bf16", "fp32", "none"]),
                     post=rng.random() < 0.4, gate=rng.choice(["none", "none", "row", "col", "full"]),
                     scale=rng.choice([1.0, 1.0, 0.22]), quantize=rng.random() < 0.6)
    return _mlp(None, rows, _width(rng, 1024, HIDDEN, 16), _width(rng, 512, INTER, 16),
                quantized=rng.random() < 0.5)


def _activations(rows, cols, gen, dtype=torch.bfloat16):
    """Activations whose channels differ in size, a few of them by much; of many rows
    the last is padding (zeros)."""
    x = torch.randn((rows, cols), generator=gen, device="cuda")
    size = torch.exp(0.5 * torch.randn((cols,), generator=gen, device="cuda"))
    size[torch.randint(0, cols, (max(1, cols // 500),), generator=gen, device="cuda")] *= 20.0
    x *= size
    if rows > 8:
        x[-1] = 0.0
    return x.to(dtype)


def _blocks(t):
    """[rows, cols] -> [rows, blocks, 128], zeros behind the last column."""
    rows, cols = t.shape
    n = -(-cols // BLOCK)
    if n * BLOCK != cols:
        t = torch.nn.functional.pad(t, (0, n * BLOCK - cols))
    return t.reshape(rows, n, BLOCK)


def _quantize(x):
    """(e4m3 values, fp32 scales [rows, blocks]) of fp32 rows."""
    b = _blocks(x)
    s = b.abs().amax(dim=2).clamp(min=AMAX_MIN)
    s = s / torch.full_like(s, E4M3_MAX)    # (over a number torch multiplies by its reciprocal)
    q = (b / s[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q.reshape(x.shape[0], -1)[:, : x.shape[1]], s


def _dequantize(q, s):
    b = _blocks(q.float()) * s[:, :, None]
    return b.reshape(q.shape[0], -1)[:, : q.shape[1]]


def _weight(n, k, gen):
    """A checkpoint's weight: e4m3 [n, k] and fp32 scales of its 128 x 128 blocks."""
    w = torch.randn((n, k), generator=gen, device="cuda") * (k ** -0.5)
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    pad = torch.nn.functional.pad(w, (0, kb * BLOCK - k, 0, nb * BLOCK - n))
    b = pad.view(nb, BLOCK, kb, BLOCK)
    s = b.abs().amax(dim=(1, 3)) / E4M3_MAX
    q = (b / s[:, None, :, None]).to(torch.float8_e4m3fn).view(nb * BLOCK, kb * BLOCK)
    return q[:n, :k].contiguous(), s


def _dequantize_weight(q, s):
    full = s.repeat_interleave(BLOCK, dim=0).repeat_interleave(BLOCK, dim=1)
    return q.float() * full[: q.shape[0], : q.shape[1]]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, rows = case["kind"], case["rows"]
    st = dict(case=case)
    if kind == "quant":
        st["x"] = _activations(rows, case["cols"], gen,
                               torch.float32 if case["fp32"] else torch.bfloat16)
        return st
    if kind == "norm":
        cols = case["cols"]
        st["x"] = _activations(rows, cols, gen)
        st["weight"] = 1.0 + 0.1 * torch.randn((cols,), generator=gen, device="cuda")
        st["residual"] = st["post"] = st["gate"] = None
        if case["residual"] != "none":
            r = _activations(rows, cols, gen, torch.float32) * 3.0
            st["residual"] = r if case["residual"] == "fp32" else r.to(torch.bfloat16)
        if case["post"]:
            st["post"] = 1.0 + 0.1 * torch.randn((cols,), generator=gen, device="cuda")
        shape = {"none": None, "row": (rows, 1), "col": (cols,), "full": (rows, cols)}[case["gate"]]
        if shape is not None:
            st["gate"] = torch.rand(shape, generator=gen, device="cuda").to(torch.bfloat16)
        return st
    width = case["n_in"] if kind == "linear" else case["hidden"]
    x = _activations(rows, width, gen)
    st["x"], st["x_scale"] = x, None
    if case["quantized"]:
        st["x"], st["x_scale"] = _quantize(x.float())
        st["x"] = st["x"].contiguous()
        st["x_scale"] = st["x_scale"].t().contiguous().t()   # a block's scales side by side
    if kind == "linear":
        st["w"], st["ws"] = _weight(case["n_out"], width, gen)
        st["bias"] = None
        if case["bias"]:
            st["bias"] = torch.randn((case["n_out"],), generator=gen, device="cuda").to(torch.bfloat16)
        return st
    st["gate"], st["gate_s"] = _weight(case["inter"], width, gen)
    st["up"], st["up_s"] = _weight(case["inter"], width, gen)
    st["down"], st["down_s"] = _weight(width, case["inter"], gen)
    return st


def run(st):
    kind = st["case"]["kind"]
    if kind == "quant":
        return _run_quant(st)
    if kind == "linear":
        return _run_linear(st)
    return _run_norm(st) if kind == "norm" else _run_mlp(st)


def _run_quant(st):
    if own:
        from tokenfactory_amd import quantize_blocks
        return quantize_blocks(st["x"])
    return _quantize(st["x"].float())


def _run_linear(st):
    if own:
        from tokenfactory_amd import block_scaled_linear
        return block_scaled_linear(st["x"], st["w"], st["ws"], st["bias"], x_scale=st["x_scale"])
    out = _plain_input(st) @ _dequantize_weight(st["w"], st["ws"]).t()
    if st["bias"] is not None:
        out = out + st["bias"].float()
    return out.to(torch.bfloat16)


def _plain_input(st):
    if st["x_scale"] is not None:
        return _dequantize(st["x"], st["x_scale"])
    return _dequantize(*_quantize(st["x"].float()))


def _run_norm(st):
    case = st["case"]
    if own:
        from tokenfactory_amd import add_rms_norm
        return add_rms_norm(st["x"], st["residual"], st["weight"], EPS, post_weight=st["post"],
                            gate=st["gate"], residual_scale=case["scale"],
                            quantize=case["quantize"])
    b = st["x"].float()
    if st["post"] is not None:
        b = b * torch.rsqrt(b.square().mean(dim=1, keepdim=True) + EPS) * st["post"]
    if st["gate"] is not None:
        b = b * st["gate"].float()
    r = b * case["scale"]
    if st["residual"] is not None:
        r = r + st["residual"].float()
    y = r * torch.rsqrt(r.square().mean(dim=1, keepdim=True) + EPS) * st["weight"]
    stored = r.to(torch.float32 if case["residual"] == "fp32" else torch.bfloat16)
    return (_quantize(y) if case["quantize"] else y.to(torch.bfloat16)), stored


def _run_mlp(st):
    if own:
        from tokenfactory_amd import gated_mlp
        return gated_mlp(st["x"], st["gate"], st["gate_s"], st["up"], st["up_s"], st["down"],
                         st["down_s"], x_scale=st["x_scale"])
    x = _plain_input(st)
    g = x @ _dequantize_weight(st["gate"], st["gate_s"]).t()
    h = g / (1.0 + torch.exp(-g)) * (x @ _dequantize_weight(st["up"], st["up_s"]).t())
    out = _dequantize(*_quantize(h)) @ _dequantize_weight(st["down"], st["down_s"]).t()
    return out.to(torch.bfloat16)


def work(case):
    """Each input read once and each output written once, quantised ones with their
    scales; a feed-forward pass keeps its hidden activations on the chip."""
    kind, rows = case["kind"], case["rows"]
    if kind == "quant":
        n = rows * case["cols"]
        return {"bytes": n * (4 if case["fp32"] else 2) + n + _scales(rows, case["cols"]),
                "flops": 3 * n}
    if kind == "norm":
        cols = case["cols"]
        n = rows * cols
        size = {"bf16": 2, "fp32": 4, "none": 0}[case["residual"]]
        out = n + _scales(rows, cols) if case["quantize"] else 2 * n
        gate = {"none": 0, "row": rows, "col": cols, "full": n}[case["gate"]]
        return {"bytes": 2 * n + size * n + (size or 2) * n + out + 2 * gate
                + 4 * cols * (1 + case["post"]), "flops": 10 * n}
    width = case["n_in"] if kind == "linear" else case["hidden"]
    x = rows * width + _scales(rows, width) if case["quantized"] else 2 * rows * width
    if kind == "linear":
        n = case["n_out"]
        return {"bytes": x + _weight_bytes(n, width) + 2 * rows * n + 2 * n * case["bias"],
                "flops": 2 * rows * n * width}
    i = case["inter"]
    return {"bytes": x + 2 * _weight_bytes(i, width) + _weight_bytes(width, i) + 2 * rows * width,
            "flops": 6 * rows * width * i}


def _scales(rows, cols):
    return 4 * rows * -(-cols // BLOCK)


def _weight_bytes(n, k):
    return n * k + 4 * -(-n // BLOCK) * -(-k // BLOCK)


# The operators in 64 bits.  By definition a scale is an fp32 number, and a quantised value
# is the e4m3 number nearest (ties to even) to the fp32 quotient, as torch's own tensor
# operations give it; found here from the spacing of e4m3 at its size.  (The quotient's
# rounding counts: bf16 values over a scale of their own block often meet a tie.)

def _exact_scale(blocks):
    return (blocks.abs().amax(dim=2).clamp(min=AMAX_MIN) / E4M3_MAX).float().double()


def _exact_e4m3(v):
    v = v.float().double().clamp(-E4M3_MAX, E4M3_MAX)
    exponent = torch.frexp(v.abs())[1] - 1
    step = torch.ldexp(torch.ones_like(v), exponent.clamp(min=-6) - 3)
    return torch.round(v / step) * step


def _exact_quantize(x):
    b = _blocks(x)
    s = _exact_scale(b)
    return _exact_e4m3(b / s[:, :, None]).reshape(x.shape[0], -1)[:, : x.shape[1]], s


def _exact_rows(q, s):
    return q.double() * s.double().repeat_interleave(BLOCK, dim=1)[:, : q.shape[1]]


def _exact_weight(q, s):
    s = s.double().repeat_interleave(BLOCK, dim=0).repeat_interleave(BLOCK, dim=1)
    return q.double() * s[: q.shape[0], : q.shape[1]]


def _exact_input(st):
    if st["x_scale"] is not None:
        return _exact_rows(st["x"], st["x_scale"])
    return _exact_rows(*_exact_quantize(st["x"].double()))


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "quant":
        return _exact_quantize(st["x"].double())
    if kind == "norm":
        r = st["x"].double()
        if st["post"] is not None:
            r = r / torch.sqrt((r * r).mean(dim=1, keepdim=True) + EPS) * st["post"].double()
        if st["gate"] is not None:
            r = r * st["gate"].double()
        r = r * case["scale"]
        if st["residual"] is not None:
            r = st["residual"].double() + r
        y = r / torch.sqrt((r * r).mean(dim=1, keepdim=True) + EPS) * st["weight"].double()
        return (_exact_quantize(y) if case["quantize"] else y), r
    x = _exact_input(st)
    if kind == "linear":
        out = torch.mm(x, _exact_weight(st["w"], st["ws"]).t())
        return out if st["bias"] is None else out + st["bias"].double()
    g = torch.mm(x, _exact_weight(st["gate"], st["gate_s"]).t())
    h = g / (1.0 + torch.exp(-g)) * torch.mm(x, _exact_weight(st["up"], st["up_s"]).t())
    return torch.mm(_exact_rows(*_exact_quantize(h)), _exact_weight(st["down"], st["down_s"]).t())
