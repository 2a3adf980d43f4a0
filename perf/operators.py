"""
Measured cases of the block-scaled 8-bit operators: quantisation, matrix product, and the join of a block with its
residual stream.

Format of every 8-bit operand here: e4m3 values (sign, 4 exponent and 3 mantissa bits, largest 448) in rows padded with
zeros to a multiple of 128 columns, and one power of two per row and block of 128 columns, held as its biased exponent
in a byte (value = e4m3 * 2^(byte - 127)).  The exponent of a block is the smallest that keeps its largest magnitude
within 448.

    quantise   q = e4m3(x / 2^e),  returned as the values q 2^e
    linear     y[r, o] = relu(sum_k a[r, k] w[o, k]) * scale[o] + shift[o]
    join       s = residual + alpha * gate * post(u)
               stream = s, or residual + s for the dense running sum of the SE-Res2 stack
               z = pre(s), in 16 or 32 bits, or quantised and handed to the next linear
               post, pre: none, rms (x / sqrt(mean x^2 + eps) * w), layer ((x - mean) / sqrt(var + eps) * w + b) or
               affine (x * w + b, a folded BatchNorm), over the channels of a row

Rows are frames of utterances packed one behind the other (utterance b owns rows row_off[b] .. row_off[b + 1]).
"""
import math

import torch

own = False

BLOCK = 128
FRAMES = 301                 # frames of a 3 s waveform
E4M3_MAX = 448.0


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    """The cases that are timed."""
    return [
        # the input of a first_conv of one 3 s utterance, quantised on its own: a launch-bound serving call
        {"name": "quantise_one_utterance", "op": "quantise", "rows": FRAMES, "cols": 512, "dtype": "bf16"},
        # features of a ragged list at a sampled width (536 is no multiple of the block), from the float32 path
        {"name": "quantise_ragged_536_f32", "op": "quantise", "rows": 24373, "cols": 536, "dtype": "f32"},
        # the catconv input of the benchmark batch, 256 utterances of 3 s
        {"name": "quantise_batch_1536", "op": "quantise", "rows": 256 * FRAMES, "cols": 1536, "dtype": "bf16"},
        # one pooled vector through a projection to the embedding width: a single row, bound by latency
        {"name": "linear_one_vector", "op": "linear", "rows": 1, "k": 1536, "n": 192, "relu": False, "affine": True,
         "dtype": "f32"},
        # catconv of one 3 s utterance in a serving loop
        {"name": "linear_one_utterance", "op": "linear", "rows": FRAMES, "k": 1536, "n": 1536, "relu": True,
         "affine": False, "dtype": "bf16"},
        # catconv of a sampled subnet: three blocks of 176 channels to 536, 64 utterances, float32 output
        {"name": "linear_sampled_528_536", "op": "linear", "rows": 64 * FRAMES, "k": 528, "n": 536, "relu": True,
         "affine": True, "dtype": "f32"},
        # first_conv / last_conv of the benchmark batch
        {"name": "linear_batch_512", "op": "linear", "rows": 256 * FRAMES, "k": 512, "n": 512, "relu": True,
         "affine": True, "dtype": "bf16"},
        # catconv of the benchmark batch, half of the network's operations
        {"name": "linear_batch_1536", "op": "linear", "rows": 256 * FRAMES, "k": 1536, "n": 1536, "relu": True,
         "affine": False, "dtype": "bf16"},
        # catconv of the Largest subnet at 512 utterances
        {"name": "linear_largest_2048", "op": "linear", "rows": 512 * FRAMES, "k": 2048, "n": 1536, "relu": True,
         "affine": False, "dtype": "bf16"},
        # one frame of a stream between two blocks, norms on both sides: bound by latency
        {"name": "join_one_frame", "op": "join", "rows": 1, "cols": 512, "utts": 0, "post": "rms", "pre": "rms",
         "gate": "channel", "dense": False, "dtype": "bf16", "stream": "bf16", "n": 0},
        # the end of an SE-Res2 block of the benchmark batch: gate per utterance, dense sum, 8-bit output into the next
        # block's first_conv
        {"name": "join_dense_into_linear", "op": "join", "rows": 256 * FRAMES, "cols": 512, "utts": 256, "post": "none",
         "pre": "none", "gate": "utterance", "dense": True, "dtype": "bf16", "stream": "bf16", "n": 512},
        # 1024-channel frames of a ragged list, layer norms before and after, the stream kept in 32 bits
        {"name": "join_ragged_layer_1024", "op": "join", "rows": 48611, "cols": 1024, "utts": 67, "post": "layer",
         "pre": "layer", "gate": "utterance", "dense": False, "dtype": "bf16", "stream": "f32", "n": 0},
    ]


def _spread(rng, low, high):
    """A whole number, even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    """A channel count: a sampled width (a multiple of 8), or any number."""
    v = _spread(rng, low, high)
    return v if rng.random() < 0.4 else max(8, v // 8 * 8)


def draw(rng):
    """One more case of the same ranges."""
    op = rng.choice(["quantise", "linear", "linear", "join"])
    if op == "quantise":
        return {"op": op, "rows": _spread(rng, 1, 256 * FRAMES), "cols": _width(rng, 8, 1536), "dtype": rng.choice(["bf16", "f32"])}
    if op == "linear":
        return {"op": op, "rows": _spread(rng, 1, 256 * FRAMES), "k": _width(rng, 16, 2048), "n": _width(rng, 8, 1536),
                "relu": rng.random() < 0.6, "affine": rng.random() < 0.6, "dtype": rng.choice(["bf16", "f32"])}
    rows = _spread(rng, 1, 128 * FRAMES)
    gate = rng.choice(["none", "channel", "utterance", "row"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    return {"op": op, "rows": rows, "cols": _width(rng, 8, 2048), "utts": min(rows, _spread(rng, 1, 256)) if gate == "utterance" else 0,
            "post": rng.choice(["none", "rms", "layer", "affine"]), "pre": rng.choice(["none", "rms", "layer", "affine"]),
            "gate": gate, "dense": rng.random() < 0.3, "dtype": dtype,
            "stream": "f32" if dtype == "f32" else rng.choice(["bf16", "f32"]), "n": rng.choice([0, 0, _width(rng, 16, 512)])}


# ------------------------------------------------------------------------------------------------------------- inputs
_DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 2 + 1)


def _activations(g, rows, cols):
    """Frames as a convolution leaves them: channels of unlike size, a slow change of level along the rows."""
    size = torch.exp(0.7 * torch.randn(cols, generator=g, device="cuda"))
    level = torch.exp(0.5 * torch.randn(rows, 1, generator=g, device="cuda"))
    return torch.randn(rows, cols, generator=g, device="cuda") * size * level


def _weights(g, n, k):
    return torch.randn(n, k, generator=g, device="cuda") * (torch.exp(0.3 * torch.randn(n, 1, generator=g, device="cuda")) / math.sqrt(k))


def _offsets(seed, rows, utts):
    """Row offsets of a ragged list (every utterance one row at least)."""
    g = torch.Generator().manual_seed(int(seed) * 2 + 1)
    share = torch.rand(utts, generator=g, dtype=torch.float64) + 0.1
    cuts = torch.floor(torch.cumsum(share, 0) / share.sum() * (rows - utts) + 1e-6).to(torch.int64)
    cuts[-1] = rows - utts
    return torch.cat([torch.zeros(1, dtype=torch.int64), cuts + torch.arange(1, utts + 1)]).to(torch.int32).cuda()


def _split(x):
    """(e4m3 values [rows, padded], exponent bytes [rows, padded blocks]) of float rows, in elementary operations."""
    x = x.float()
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    b = torch.nn.functional.pad(x, (0, blocks * BLOCK - cols)).reshape(rows, blocks, BLOCK)
    big = b.abs().amax(2)
    m, e = torch.frexp(big)                                    # big = m 2^e, m in [0.5, 1);  448 = 0.875 2^9
    e = torch.where(big > 0, e - 9 + (m > 0.875).to(e.dtype), torch.full_like(e, -127)).clamp(min=-127)
    q = torch.ldexp(b, -e[:, :, None]).to(torch.float8_e4m3fn)
    byte = torch.full((rows, -(-blocks // 4) * 4), 127, dtype=torch.uint8, device=x.device)
    byte[:, :blocks] = (e + 127).to(torch.uint8)
    return q.reshape(rows, blocks * BLOCK), byte


def _values(q, byte, cols):
    """The float32 values that (e4m3, exponent bytes) stand for."""
    blocks = q.shape[1] // BLOCK
    e = byte[:, :blocks].to(torch.int32) - 127
    return torch.ldexp(q.float().reshape(q.shape[0], blocks, BLOCK), e[:, :, None]).reshape(q.shape[0], -1)[:, :cols]


def _norm_of(g, kind, cols):
    if kind == "none":
        return None
    return {"kind": kind, "w": 1.0 + 0.2 * torch.randn(cols, generator=g, device="cuda"),
            "b": None if kind == "rms" else 0.1 * torch.randn(cols, generator=g, device="cuda"), "eps": 1e-5}


def _tensors(case, seed):
    """The case's inputs, from the seed alone."""
    g, op = _gen(seed), case["op"]
    if op == "quantise":
        return {"x": _activations(g, case["rows"], case["cols"]).to(_DT[case["dtype"]])}
    if op == "linear":
        a, w = _split(_activations(g, case["rows"], case["k"])), _split(_weights(g, case["n"], case["k"]))
        t = {"a": a, "w": w, "scale": None, "shift": None}
        if case["affine"]:
            t["scale"] = 1.0 + 0.3 * torch.randn(case["n"], generator=g, device="cuda")
            t["shift"] = 0.2 * torch.randn(case["n"], generator=g, device="cuda")
        return t
    rows, cols = case["rows"], case["cols"]
    t = {"u": _activations(g, rows, cols).to(_DT[case["dtype"]]), "residual": _activations(g, rows, cols).to(_DT[case["stream"]]),
         "post": _norm_of(g, case["post"], cols), "pre": _norm_of(g, case["pre"], cols), "gate": None, "row_off": None, "alpha": 0.75}
    if case["gate"] == "channel":
        t["gate"] = torch.rand(cols, generator=g, device="cuda")
    elif case["gate"] == "row":
        t["gate"] = torch.rand(rows, cols, generator=g, device="cuda").to(_DT[case["dtype"]])
    elif case["gate"] == "utterance":
        t["gate"] = torch.rand(case["utts"], cols, generator=g, device="cuda")
        t["row_off"] = _offsets(seed, rows, case["utts"])
    if case["n"]:
        t["w"] = _split(_weights(g, case["n"], cols))
    return t


def prepare(case, seed):
    """The inputs on the GPU, and the 8-bit operands as the framework holds them."""
    t = _tensors(case, seed)
    t["case"] = dict(case)
    if own:
        import sugar_amd
        k = case["k"] if case["op"] == "linear" else case.get("cols")
        for name in ("a", "w"):
            if t.get(name) is not None:
                t[name] = sugar_amd.BlockFP8(t[name][0], t[name][1], k)
        for name in ("post", "pre"):
            if t.get(name) is not None:
                p = t[name]
                t[name] = sugar_amd.RowNorm(p["kind"], p["w"], p["b"], p["eps"])
    return t


# ---------------------------------------------------------------------------------------------------------- one pass
def _norm(p, x):
    if p is None:
        return x
    if p["kind"] == "layer":
        x = x - x.mean(1, keepdim=True)
    if p["kind"] in ("rms", "layer"):
        x = x / torch.sqrt((x * x).mean(1, keepdim=True) + p["eps"])
    x = x * p["w"]
    return x if p["b"] is None else x + p["b"]


def _gate_rows(t):
    """The gate of every row, or None."""
    if t["row_off"] is None:
        return t["gate"]
    n = (t["row_off"][1:] - t["row_off"][:-1]).to(torch.int64)
    return t["gate"][torch.repeat_interleave(torch.arange(n.numel(), device=n.device), n, output_size=t["u"].shape[0])]


def _plain_linear(a, w, k):
    return _values(a[0], a[1], k) @ _values(w[0], w[1], k).T


def _run_plain(t, case):
    op = case["op"]
    if op == "quantise":
        q, byte = _split(t["x"])
        return _values(q, byte, case["cols"]).to(_DT[case["dtype"]])
    if op == "linear":
        y = _plain_linear(t["a"], t["w"], case["k"])
        if case["relu"]:
            y = torch.clamp(y, min=0.0)
        if case["affine"]:
            y = y * t["scale"] + t["shift"]
        return y.to(_DT[case["dtype"]])
    v, r, gate = _norm(t["post"], t["u"].float()), t["residual"].float(), _gate_rows(t)
    s = r + t["alpha"] * (v if gate is None else v * gate.float())
    stream = (r + s if case["dense"] else s).to(t["residual"].dtype)
    z = _norm(t["pre"], s)
    if not case["n"]:
        return [stream, z.to(t["u"].dtype)]
    return [stream, _plain_linear(_split(z), t["w"], case["cols"]).to(t["u"].dtype)]


def _run_own(t, case):
    import sugar_amd
    op = case["op"]
    if op == "quantise":
        return sugar_amd.quantize_block_fp8(t["x"]).dequantize(t["x"].dtype)
    if op == "linear":
        return sugar_amd.block_fp8_linear(t["a"], t["w"], scale=t["scale"], shift=t["shift"], relu=case["relu"],
                                          out_dtype=_DT[case["dtype"]])
    j = sugar_amd.block_join(t["u"], t["residual"], post=t["post"], gate=t["gate"], row_off=t["row_off"], alpha=t["alpha"],
                             dense=case["dense"], pre=t["pre"], normed=not case["n"], quantized=bool(case["n"]))
    if not case["n"]:
        return [j.stream, j.normed]
    return [j.stream, sugar_amd.block_fp8_linear(j.quantized, t["w"], out_dtype=t["u"].dtype)]


def run(state):
    """One pass."""
    return (_run_own if own else _run_plain)(state, state["case"])


# ---------------------------------------------------------------------------------------------------- needs, and truth
def work(case):
    """What a pass reads and writes, each value once, and its multiplications and additions."""
    size = {"bf16": 2, "f32": 4}
    if case["op"] == "quantise":
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * size[case["dtype"]] * n, "flops": 3 * n}
    if case["op"] == "linear":
        r, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": (r + n) * (k + -(-k // BLOCK)) + r * n * size[case["dtype"]] + (8 * n if case["affine"] else 0),
                "flops": 2 * r * k * n}
    r, c, n = case["rows"], case["cols"], case["n"]
    u, s = size[case["dtype"]], size[case["stream"]]
    gate = {"none": 0, "channel": 4 * c, "utterance": 4 * c * case["utts"], "row": u * r * c}[case["gate"]]
    norms = sum({"none": 0, "rms": 4, "layer": 8, "affine": 8}[case[p]] * c for p in ("post", "pre"))
    out = n * (c + -(-c // BLOCK)) + u * r * n if n else u * r * c
    return {"bytes": r * c * (u + 2 * s) + gate + norms + out, "flops": 12 * r * c + 2 * r * c * n}


def _powers_64():
    """2^-160 .. 2^160 (from the host: a device's pow may be off in the last bit, which would decide ties)."""
    return torch.tensor([2.0 ** i for i in range(-160, 161)], dtype=torch.float64, device="cuda")


def _e4m3_64(v):
    """Nearest e4m3 values of float64 numbers within +-448, ties to the even mantissa."""
    p, a = _powers_64(), v.abs()
    at = torch.bucketize(torch.clamp(a, min=2.0 ** -6), p, right=True) - 1     # p[at] <= a < p[at + 1]
    step = p[at - 3]                                                             # 3 mantissa bits below the leading one
    return torch.sign(v) * torch.round(a / step) * step


def _requantised_64(x):
    """The values that float64 rows stand for once they are held in 8 bits."""
    p, out = _powers_64(), torch.empty_like(x)
    for c in range(0, x.shape[1], BLOCK):
        part = x[:, c:c + BLOCK]
        at = torch.bucketize(part.abs().amax(1) / E4M3_MAX, p)                   # smallest power that reaches the largest / 448
        unit = p[at.clamp(min=160 - 127)][:, None]
        out[:, c:c + BLOCK] = _e4m3_64(part / unit) * unit
    return out


def _held_64(pair, cols):
    """Float64 values of 8-bit operands, block by block."""
    q, byte = pair
    x = q.to(torch.float32).double()
    for i in range(x.shape[1] // BLOCK):
        x[:, i * BLOCK:(i + 1) * BLOCK] *= _powers_64()[byte[:, i:i + 1].long() - 127 + 160]
    return x[:, :cols]


def _normed_64(p, x):
    if p is None:
        return x
    w = p["w"].double()
    if p["kind"] == "rms":
        return x * torch.rsqrt(x.square().sum(1, keepdim=True) / x.shape[1] + p["eps"]) * w
    if p["kind"] == "layer":
        x = (x - x.mean(1, keepdim=True)) * torch.rsqrt(x.var(1, unbiased=False, keepdim=True) + p["eps"])
    return x * w + p["b"].double()


def exact(case, seed):
    """run()'s outputs in 64 bits."""
    t = _tensors(case, seed)
    if case["op"] == "quantise":
        return _requantised_64(t["x"].double())
    if case["op"] == "linear":
        y = torch.matmul(_held_64(t["a"], case["k"]), _held_64(t["w"], case["k"]).t())
        if case["relu"]:
            y.clamp_(min=0)
        return y * t["scale"].double() + t["shift"].double() if case["affine"] else y
    v, r = _normed_64(t["post"], t["u"].double()), t["residual"].double()
    if t["row_off"] is not None:
        off = t["row_off"].tolist()
        for b in range(case["utts"]):
            v[off[b]:off[b + 1]] *= t["gate"][b].double()
    elif t["gate"] is not None:
        v = v * t["gate"].double()
    s = r + t["alpha"] * v
    z = _normed_64(t["pre"], s)
    if case["n"]:
        z = torch.matmul(_requantised_64(z), _held_64(t["w"], case["cols"]).t())
    return [r + s if case["dense"] else s, z]
