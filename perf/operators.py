"""The block-scaled 8-bit operators, case by case: what they are given, what they return in plain torch, and what one pass cannot do without.

The format ("blocks"): e4m3 values (4 exponent bits, 3 mantissa bits, no infinity, largest 448) in rows whose length is padded with zeros to a
multiple of 128, and one power of two for each block of 128 values along a row -- of ONE row (activations) or of 128 rows (weights) -- held as
its biased exponent in one byte: byte s stands for 2^(s - 127).  The power of a block is the smallest 2^e with max |x| <= 448 * 2^e over the block's
finite values (byte 127 for a block of zeros, never below byte 0); a value becomes the e4m3 nearest to x / 2^e, ties to even; what is not finite becomes NaN.
A row's scale bytes are padded with 127 to a multiple of four.

  quantize    x [rows][cols] f32 / f16 / bf16 -> values and scales, in blocks of 1 x 128 or 128 x 128
  dequantize  values and scales -> [rows][cols] f32 / f16 / bf16
  dense       y = epi(x . w^T + bias): x [rows][in] in blocks of 1 x 128 (or f32 / f16 / bf16, quantised within the call), w [out][in] in blocks
              of 128 x 128, epi nothing or the clipped ReLU min(max(y, 0), clip); y f32 / f16 / bf16
  stack       dense layers one behind the other, each but the last with the clipped ReLU and its result handed on in blocks

Where `own` is true, `run` calls stt_amd.blocks.
"""
import torch

own = False

BLOCK = 128
CLIP = 20.0         # the clipped ReLU of the acoustic model's dense layers
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
LARGEST = 32000 * 2048 * 8192       # multiply-adds of the largest dense case


def listed():
    return [
        # one hop of one live stream: 16 windows of 19 x 26 features on their way into layer 1
        {"name": "quantize hop", "op": "quantize", "rows": 16, "cols": 494, "type": "f32", "block_rows": 1},
        # layer outputs of two batches of 64 utterances of 5 s (250 frames each)
        {"name": "quantize batch", "op": "quantize", "rows": 32000, "cols": 2048, "type": "f16", "block_rows": 1},
        # the x half of the cell's kernel, once when a model is loaded
        {"name": "quantize weights", "op": "quantize", "rows": 8192, "cols": 2048, "type": "f32", "block_rows": 128},
        # a hop's rows read back
        {"name": "dequantize hop", "op": "dequantize", "rows": 16, "cols": 2048, "type": "f16", "block_rows": 1},
        {"name": "dequantize batch", "op": "dequantize", "rows": 32000, "cols": 2048, "type": "bf16", "block_rows": 1},
        # one frame through a hidden layer
        {"name": "dense frame", "op": "dense", "rows": 1, "inner": 2048, "out": 2048, "from": "f16", "to": "f16", "relu": True},
        # the x half of the cell for one stream's hop, for the hop of 128 live streams, and for two batches of 64 utterances at once
        {"name": "dense hop", "op": "dense", "rows": 16, "inner": 2048, "out": 8192, "from": "e4m3", "to": "f32", "relu": False},
        {"name": "dense live set", "op": "dense", "rows": 2048, "inner": 2048, "out": 8192, "from": "e4m3", "to": "f32", "relu": False},
        {"name": "dense batch", "op": "dense", "rows": 32000, "inner": 2048, "out": 8192, "from": "e4m3", "to": "f32", "relu": False},
        # the output layer over the frames of a long utterance
        {"name": "dense classes", "op": "dense", "rows": 1009, "inner": 2048, "out": 29, "from": "bf16", "to": "f32", "relu": False},
        # layers 1 - 3 of a hop; layers 1 - 3 and the x half of the cell for a time-chunk of 128 utterances (48 frames each)
        {"name": "stack hop", "op": "stack", "rows": 16, "inner": 494, "hidden": 2048, "layers": 3, "out": 2048, "from": "f32", "to": "f16"},
        {"name": "stack chunk", "op": "stack", "rows": 6144, "inner": 494, "hidden": 2048, "layers": 4, "out": 8192, "from": "f16", "to": "f16"},
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over its logarithm; every other one as it falls (odd ones among them), the others in 16s."""
    n = round(low * (high / low) ** rng.random())
    return n if n < 32 or rng.random() < 0.5 else n // 16 * 16


def draw(rng):
    op = rng.choice(("quantize", "dequantize", "dense", "dense", "stack"))
    rows = _spread(rng, 1, 32000)
    if op in ("quantize", "dequantize"):
        cols = _spread(rng, 26, 4096)
        rows = min(rows, 32000 * 2048 // cols)
        return {"op": op, "rows": rows, "cols": cols, "type": rng.choice(sorted(TYPES)), "block_rows": rng.choice((1, 1, BLOCK))}
    if op == "dense":
        inner, out = _spread(rng, 26, 4096), _spread(rng, 2, 8192)
        rows = min(rows, LARGEST // (inner * out), 32000 * 8192 // out)
        return {"op": op, "rows": rows, "inner": inner, "out": out, "from": rng.choice(("e4m3", "f32", "f16", "bf16")), "to": rng.choice(sorted(TYPES)),
                "relu": rng.random() < 0.5}
    hidden, out = _spread(rng, 128, 4096), _spread(rng, 29, 8192)
    layers = rng.choice((2, 3, 4))
    inner = _spread(rng, 26, 1024)
    rows = min(rows, LARGEST // (2 * hidden * (inner + hidden * (layers - 2) + out)))
    return {"op": op, "rows": rows, "inner": inner, "hidden": hidden, "layers": layers, "out": out, "from": rng.choice(sorted(TYPES)), "to": rng.choice(("f16", "bf16"))}


# ------------------------------------------------------------------------------------------------ inputs
def _features(rows, cols, gen):
    """Cepstral windows: the first coefficients much larger than the last."""
    x = torch.randn(rows, cols, device="cuda", generator=gen)
    return x * (30.0 / (1.0 + torch.arange(cols, device="cuda") % 26))


def _activations(rows, cols, gen):
    """What a clipped-ReLU layer leaves: about half zeros, rows of different loudness, some values at the clip."""
    x = torch.randn(rows, cols, device="cuda", generator=gen)
    x = x * torch.exp(1.5 * torch.randn(rows, 1, device="cuda", generator=gen))
    return x.clamp_(0.0, CLIP)


def _weights(out, inner, gen):
    w = torch.randn(out, inner, device="cuda", generator=gen) / inner ** 0.5
    return w * torch.exp(0.5 * torch.randn(out, 1, device="cuda", generator=gen))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = dict(case)
    if case["op"] == "quantize":
        x = _weights(case["rows"], case["cols"], gen) if case["block_rows"] == BLOCK else _activations(case["rows"], case["cols"], gen)
        s["x"] = x.to(TYPES[case["type"]])
    elif case["op"] == "dequantize":
        x = _weights(case["rows"], case["cols"], gen) if case["block_rows"] == BLOCK else _activations(case["rows"], case["cols"], gen)
        s["q"], s["scale"] = plain_quantize(x, case["block_rows"])
    else:
        if case["op"] == "dense":
            sizes = [case["inner"], case["out"]]
            x = _activations(case["rows"], case["inner"], gen)
        else:
            sizes = [case["inner"]] + [case["hidden"]] * (case["layers"] - 1) + [case["out"]]
            x = _features(case["rows"], case["inner"], gen)
        if case["from"] == "e4m3":
            s["q"], s["scale"] = plain_quantize(x, 1)
        else:
            s["x"] = x.to(TYPES[case["from"]])
        s["sizes"] = sizes
        s["w"] = [plain_quantize(_weights(o, i, gen), BLOCK) for i, o in zip(sizes, sizes[1:])]
        s["bias"] = [0.1 * torch.randn(o, device="cuda", generator=gen) for o in sizes[1:]]
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def _up(n, to):
    return -(-n // to) * to


def _power(byte):
    """2^(byte - 127) as the f32 with that exponent (a library's exp2 may be off in its last bit)."""
    b = byte.to(torch.int32)
    return torch.where(b > 0, b << 23, 1 << 22).view(torch.float32)


def plain_quantize(x, block_rows):
    """(values [rows][padded] e4m3, scales [rows of blocks][blocks padded to four] uint8)"""
    rows, cols = x.shape
    v = torch.nn.functional.pad(x.float(), (0, _up(cols, BLOCK) - cols, 0, _up(rows, block_rows) - rows))
    t = v.view(v.shape[0] // block_rows, block_rows, v.shape[1] // BLOCK, BLOCK)
    finite = torch.isfinite(t)
    top = torch.where(finite, t.abs(), 0.0).amax((1, 3), keepdim=True)
    m, e = torch.frexp(top)                                             # top = m 2^e, 1/2 <= m < 1; 448 = 0.875 * 2^9
    byte = torch.where(top == 0.0, 127, (e - 9 + (m > 0.875).to(e.dtype) + 127).clamp(0, 254))
    q = torch.where(finite, t * _power(254 - byte), float("nan")).view(v.shape)[:rows].to(torch.float8_e4m3fn)
    byte = byte[:, 0, :, 0].to(torch.uint8)
    return q, torch.nn.functional.pad(byte, (0, _up(byte.shape[1], 4) - byte.shape[1]), value=127)


def plain_values(q, scale, cols, block_rows):
    """[rows][cols] f32"""
    rows, blocks = q.shape[0], q.shape[1] // BLOCK
    s = _power(scale[:, :blocks]).repeat_interleave(block_rows, 0)[:rows]
    return (q.float().view(rows, blocks, BLOCK) * s[:, :, None]).view(rows, blocks * BLOCK)[:, :cols]


def plain_dense(x, w, bias, relu):
    y = x @ plain_values(w[0], w[1], x.shape[1], BLOCK).t() + bias
    return y.clamp(0.0, CLIP) if relu else y


def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "quantize":
        return plain_quantize(s["x"], s["block_rows"])
    if s["op"] == "dequantize":
        return plain_values(s["q"], s["scale"], s["cols"], s["block_rows"]).to(TYPES[s["type"]])
    q, scale = (s["q"], s["scale"]) if s["from"] == "e4m3" else plain_quantize(s["x"], 1)
    x = plain_values(q, scale, s["sizes"][0], 1)
    if s["op"] == "dense":
        return plain_dense(x, s["w"][0], s["bias"][0], s["relu"]).to(TYPES[s["to"]])
    for w, b in zip(s["w"][:-1], s["bias"][:-1]):
        y = plain_dense(x, w, b, True)
        x = plain_values(*plain_quantize(y, 1), y.shape[1], 1)
    return plain_dense(x, s["w"][-1], s["bias"][-1], False).to(TYPES[s["to"]])


# ------------------------------------------------------------------------------------------------ the framework's calls
def _run_own(s):
    from stt_amd import blocks
    if s["op"] == "quantize":
        b = blocks.quantize_blocks(s["x"], block_rows=s["block_rows"])
        return b.values, b.scale
    if s["op"] == "dequantize":
        return blocks.dequantize_blocks(blocks.BlockTensor(s["q"], s["scale"], s["cols"], s["block_rows"]), TYPES[s["type"]])
    x = blocks.BlockTensor(s["q"], s["scale"], s["sizes"][0], 1) if s["from"] == "e4m3" else s["x"]
    w = [blocks.BlockTensor(q, scale, inner, BLOCK) for (q, scale), inner in zip(s["w"], s["sizes"])]
    if s["op"] == "dense":
        return blocks.dense_blocks(x, w[0], s["bias"][0], relu_clip=CLIP if s["relu"] else None, dtype=TYPES[s["to"]])
    for v, b in zip(w[:-1], s["bias"][:-1]):
        x = blocks.dense_blocks(x, v, b, relu_clip=CLIP, dtype=torch.float8_e4m3fn)
    return blocks.dense_blocks(x, w[-1], s["bias"][-1], dtype=TYPES[s["to"]])


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def _held(rows, cols, block_rows):
    """Bytes of a matrix in blocks."""
    return rows * _up(cols, BLOCK) + _up(rows, block_rows) // block_rows * _up(_up(cols, BLOCK) // BLOCK, 4)


def work(case):
    if case["op"] in ("quantize", "dequantize"):
        n = case["rows"] * case["cols"]
        return {"bytes": n * BYTES[case["type"]] + _held(case["rows"], case["cols"], case["block_rows"]), "flops": 2 * n}
    rows = case["rows"]
    if case["op"] == "dense":
        sizes = [case["inner"], case["out"]]
    else:
        sizes = [case["inner"]] + [case["hidden"]] * (case["layers"] - 1) + [case["out"]]
    read = _held(rows, sizes[0], 1) if case["from"] == "e4m3" else rows * sizes[0] * BYTES[case["from"]]
    pairs = list(zip(sizes, sizes[1:]))
    return {"bytes": read + sum(_held(o, i, BLOCK) + 4 * o for i, o in pairs) + rows * sizes[-1] * BYTES[case["to"]],
            "flops": 2 * rows * sum(i * o for i, o in pairs)}


# ------------------------------------------------------------------------------------------------ 64 bits
def _two(e):
    """2^e in 64 bits for whole e, by its bits."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_power(top):
    """The smallest whole e >= -127 with top <= 448 * 2^e, top > 0."""
    e = torch.floor(torch.log2(top)) - 9
    for _ in range(2):
        e = torch.where(top > 448.0 * _two(e), e + 1, e)
    return e.clamp(min=-127)


def _exact_round(v):
    """The e4m3 nearest to v, ties to even: steps of 2^-9 below 2^-6, eight steps to each power of two from there on."""
    a = v.abs()
    step = _two(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.round(a / step) * step * torch.sign(v)


def _exact_quantize(x, block_rows):
    """(e4m3 values [rows][padded], bytes [rows of blocks][blocks]) of x in 64 bits"""
    rows, cols = x.shape
    big = torch.zeros(_up(rows, block_rows), _up(cols, BLOCK), dtype=torch.float64, device=x.device)
    big[:rows, :cols] = x
    of = [big[:, c:c + BLOCK].abs().amax(1).view(-1, block_rows).amax(1) for c in range(0, big.shape[1], BLOCK)]
    top = torch.stack(of, 1)
    e = torch.where(top > 0, _exact_power(torch.where(top > 0, top, 1.0)), 0.0)
    wide = e.repeat_interleave(block_rows, 0).repeat_interleave(BLOCK, 1)
    return _exact_round(big * _two(-wide))[:rows], e + 127


def _exact_values(v, byte, cols, block_rows):
    wide = _two(byte.double() - 127)
    return (v.double() * wide.repeat_interleave(block_rows, 0)[:v.shape[0]].repeat_interleave(BLOCK, 1)[:, :v.shape[1]])[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        v, byte = _exact_quantize(s["x"].double(), case["block_rows"])
        padded = torch.full((byte.shape[0], _up(byte.shape[1], 4)), 127, dtype=torch.uint8, device=byte.device)
        padded[:, :byte.shape[1]] = byte.to(torch.uint8)
        return v, padded
    if case["op"] == "dequantize":
        return _exact_values(s["q"], s["scale"], case["cols"], case["block_rows"])
    if case["from"] == "e4m3":
        v, byte = s["q"].double(), s["scale"]
    else:
        v, byte = _exact_quantize(s["x"].double(), 1)
    layers = list(zip(s["w"], s["bias"], s["sizes"]))
    for k, (w, b, inner) in enumerate(layers):
        if k:
            v, byte = _exact_quantize(y, 1)  # noqa: F821
        y = torch.addmm(b.double(), _exact_values(v, byte, inner, 1), _exact_values(w[0], w[1], inner, BLOCK).t())
        if k + 1 < len(layers) or case.get("relu"):
            y = y.clamp(0.0, CLIP)
    return y
