"""The block-scaled 8-bit operators against their definition in 64 bits (tests/blocks_ref.py), through stt_amd.blocks and the C entries.

Where operands are small whole numbers times powers of two, every sum below is exact in 32 bits in any order, and results have to be EQUAL.  With
real values a sum of n products (each exact: 4 x 4 significand bits) is off by at most n half steps of 32 bits of the sum of magnitudes, doubled
where an adder drops bits instead of rounding them: n * 2^-23 * sum |x w|, plus half a step of the result's own type."""
import ctypes as C

import numpy as np
import pytest
import torch

import blocks_ref as R
from stt_amd import blocks, native

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn


def host(t):
    return t.detach().double().cpu().numpy()


def bits(t):
    return t.view(torch.uint8).cpu().numpy()


def gpu_blocks(v, byte, cols, block_rows):
    """BlockTensor of reference values."""
    return blocks.BlockTensor(torch.from_numpy(np.asarray(v, np.float32)).to(E4M3).cuda(), torch.from_numpy(np.ascontiguousarray(byte)).cuda(), cols, block_rows)


def whole_blocks(rng, rows, cols, block_rows, spread=1):
    """A matrix in blocks whose values are whole numbers up to 4, its blocks' powers 2^-spread .. 2^spread: (BlockTensor, float64 matrix)."""
    v = np.zeros((rows, R.up(cols, 128)))
    v[:, :cols] = rng.integers(-4, 5, (rows, cols))
    nb = v.shape[1] // 128
    byte = np.full((-(-rows // block_rows), R.up(nb, 4)), 127, np.uint8)
    byte[:, :nb] = rng.integers(127 - spread, 128 + spread, (byte.shape[0], nb))
    return gpu_blocks(v, byte, cols, block_rows), R.values(v, byte, cols, block_rows)


def check_blocks(b, x, block_rows):
    v, byte = R.quantize(x, block_rows)
    np.testing.assert_array_equal(b.scale.cpu().numpy(), byte)
    np.testing.assert_array_equal(host(b.values), v)          # (NaN equals NaN)


def hard(rng, rows, cols, dtype):
    """Values that go wrong: ties, borders of powers, zeros, subnormals, the type's largest, infinities and NaN, rows that are all of one kind."""
    x = rng.standard_normal((rows, cols)) * np.exp(rng.uniform(-20 if dtype is torch.float16 else -60, 8, (rows, 1)))
    x[rng.random((rows, cols)) < 0.2] = 0.0
    kinds = [0.0, -0.0, 448.0, 448.5, 449.0, 1.75, -1.8125, 2.0 ** -9, 17.0, 19.0, 2.0 ** -24, np.inf, -np.inf, np.nan, torch.finfo(dtype).max, torch.finfo(dtype).tiny / 4]
    for r in range(rows):
        if r % 3 == 0:
            for k in range(r % 7):
                x[r, rng.integers(cols)] = kinds[rng.integers(len(kinds))]
        elif r % 11 == 5:
            x[r] = kinds[rng.integers(len(kinds))]
        elif r % 3 == 2:
            x[r] = rng.integers(-40, 41, cols) / 2.0           # ties: halves of a step between 8 and 20
    return torch.from_numpy(x).to(dtype)


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 127), (16, 494), (17, 513), (130, 129), (257, 1000), (64, 2048)])
def test_quantize(rows, cols, block_rows, t):
    x = hard(np.random.default_rng(rows * 1000 + cols), rows, cols, TYPES[t])
    check_blocks(blocks.quantize_blocks(x.cuda(), block_rows), host(x), block_rows)


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_strides(block_rows, t):
    """Rows of a wider matrix (aligned and not), every second row, one row for all."""
    x = hard(np.random.default_rng(5), 40, 700, TYPES[t]).cuda()
    for v in (x[:, 16:400], x[:, 3:390], x[1::2, 8:264], x[5:6, 1:300].expand(33, 299), x[7:7, :5]):
        check_blocks(blocks.quantize_blocks(v, block_rows), host(v), block_rows)


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("block_rows", [1, 128])
def test_dequantize_every_code(block_rows, t):
    """All 256 codes under powers from 2^-127 to 2^127 and the NaN byte; the one rounding is the type's own, so bits are equal."""
    bytes_ = [0, 1, 40, 100, 118, 127, 128, 140, 200, 254, 255]
    rows = len(bytes_) if block_rows == 1 else 128 * (len(bytes_) - 1) + 5
    codes = np.tile(np.arange(256, dtype=np.uint8), (rows, 2))[:, :384]
    scale = np.full((len(bytes_), 4), 127, np.uint8)
    scale[:, 0], scale[:, 1], scale[:, 2] = bytes_, bytes_[::-1], 130
    b = blocks.BlockTensor(torch.from_numpy(codes).view(E4M3).cuda(), torch.from_numpy(scale).cuda(), 383, block_rows)
    y = blocks.dequantize_blocks(b, TYPES[t])
    want = torch.from_numpy(R.values(R.e4m3_values()[codes], scale, 383, block_rows)).to(TYPES[t])       # (one rounding: 4 significand bits are exact in float32 and float64)
    np.testing.assert_array_equal(host(y), host(want))


@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 100), (33, 512), (200, 1001)])
def test_there_and_back(rows, cols):
    """A value comes back within half a step of three mantissa bits (2^-4 of it), or of 2^-9 of its block's power; a second pass changes nothing."""
    x = torch.randn(rows, cols, device="cuda") * torch.exp(3 * torch.randn(rows, 1, device="cuda"))
    b = blocks.quantize_blocks(x)
    y = blocks.dequantize_blocks(b)
    power = np.ldexp(1.0, b.scale.cpu().numpy().astype(int) - 127)[:, :-(-cols // 128)].repeat(128, 1)[:, :cols]
    assert (np.abs(host(y) - host(x)) <= np.maximum(np.abs(host(x)) / 16, power * 2.0 ** -10)).all()
    again = blocks.quantize_blocks(y)
    np.testing.assert_array_equal(host(blocks.dequantize_blocks(again)), host(y))


SHAPES = [(1, 1, 1), (1, 494, 2048), (3, 128, 16), (16, 494, 100), (17, 130, 129), (31, 2048, 29), (33, 1000, 257), (64, 256, 128), (65, 127, 130), (100, 640, 17), (129, 129, 127),
          (300, 385, 260), (128, 2048, 256), (513, 494, 385), (1009, 300, 29), (900, 130, 1400), (2000, 200, 2100), (4500, 128, 4100), (33000, 70, 30)]


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_dense_whole_numbers(m, k, n):
    """Equal in every bit: x in blocks and as f32 / f16 / bf16, y in every type, with and without bias and ReLU."""
    rng = np.random.default_rng(m + k + n)
    x, xd = whole_blocks(rng, m, k, 1)
    w, wd = whole_blocks(rng, n, k, 128)
    bias = rng.integers(-9, 10, n) / 4.0
    bg = torch.from_numpy(bias).float().cuda()
    for kind in ("blocks", "f32", "f16", "bf16"):
        xin = x if kind == "blocks" else torch.from_numpy(xd).to(TYPES[kind]).cuda()
        for b, bd, clip in ((None, None, None), (bg, bias, None), (bg, bias, 20.0)):
            want = R.dense(xd, wd, bd, clip)
            for t, dt in TYPES.items():
                y = blocks.dense_blocks(xin, w, b, relu_clip=clip, dtype=dt)
                np.testing.assert_array_equal(host(y), host(torch.from_numpy(want).float().to(dt)), err_msg="%s %s %s" % (kind, t, clip))
            check_blocks(blocks.dense_blocks(xin, w, b, relu_clip=clip, dtype=E4M3), want, 1)


@pytest.mark.parametrize("m,k,n", [(1, 2048, 300), (16, 4096, 128), (48, 494, 200), (200, 2048, 150), (700, 494, 300), (3000, 1000, 700), (2600, 2048, 3300)])
@pytest.mark.parametrize("kind", ["blocks", "f32", "f16", "bf16"])
def test_dense_real_values(m, k, n, kind):
    g = torch.Generator().manual_seed(m + n)
    x = torch.randn(m, k, generator=g) * torch.exp(2 * torch.randn(m, 1, generator=g))
    w = torch.randn(n, k, generator=g) * torch.exp(torch.randn(n, 1, generator=g)) / k ** 0.5
    bias = torch.randn(n, generator=g)
    x = x.to(TYPES.get(kind, torch.float32))
    xd = R.values(*R.quantize(host(x), 1), k, 1)
    wq = R.quantize(host(w), 128)
    wd = R.values(*wq, k, 128)
    xin = gpu_blocks(*R.quantize(host(x), 1), k, 1) if kind == "blocks" else x.cuda()
    want, size = R.dense(xd, wd, host(bias)), np.abs(xd) @ np.abs(wd).T + np.abs(host(bias))
    for dt in (torch.float32, torch.float16, torch.bfloat16):
        y = blocks.dense_blocks(xin, gpu_blocks(*wq, k, 128), bias.cuda(), dtype=dt)
        step, top = torch.finfo(dt).eps / 2, torch.finfo(dt).max
        room = (k + 1) * 2.0 ** -23 * size * (1 + step) + step * np.abs(want) + torch.finfo(dt).smallest_normal
        got = host(y)
        beyond = np.abs(want) + room > top                 # (what is above the type's largest value by half a step rounds to an infinity: 65520 and more in float16)
        assert (np.abs(got - want)[~beyond] <= room[~beyond]).all()
        assert beyond.sum() < 1e-3 * beyond.size + 1 and (np.sign(got[beyond]) * np.minimum(np.abs(got[beyond]), 2 * top) * np.sign(want[beyond]) >= top * (1 - 2 * step) - room[beyond]).all()


def test_dense_same_bits_every_time_and_fused():
    """Two calls, and rows quantised within the call or before it, give the same bits."""
    for m in (1, 16, 40, 64, 65, 500, 5000):
        x = torch.randn(m, 494, device="cuda")
        w = blocks.quantize_blocks(torch.randn(300, 494, device="cuda"), 128)
        a, b, c = blocks.dense_blocks(x, w, dtype=torch.float32), blocks.dense_blocks(x, w, dtype=torch.float32), blocks.dense_blocks(blocks.quantize_blocks(x), w, dtype=torch.float32)
        assert torch.equal(a, b) and torch.equal(a, c), m


@pytest.mark.parametrize("m", [2, 20, 150, 4000])
def test_dense_not_finite(m):
    """A NaN or infinity in a row makes that row NaN and no other, through the ReLU too; a NaN weight makes its column NaN; scale byte 255 its block."""
    rng = np.random.default_rng(m)
    x, xd = whole_blocks(rng, m, 300, 1)
    w, wd = whole_blocks(rng, 140, 300, 128)
    wd[7, 299] = np.nan
    w.values[7, 299] = float("nan")
    xd[1, 130] = np.nan
    for value in (np.nan, np.inf, -np.inf):
        for kind in ("f32", "f16", "bf16"):
            xin = torch.from_numpy(np.where(np.isnan(xd), value, xd)).to(TYPES[kind]).cuda()
            y = host(blocks.dense_blocks(xin, w, relu_clip=5.0, dtype=torch.float32))
            np.testing.assert_array_equal(y, R.dense(xd, wd, clip=5.0))
    x.scale[1, 2] = 255
    w.scale[1, 0] = 255
    y = host(blocks.dense_blocks(x, w, dtype=torch.bfloat16))
    want = R.dense(np.where(np.isnan(xd), 0, xd), wd)
    assert np.isnan(y[1]).all() and np.isnan(y[:, 128:]).all() and np.isnan(y[:, 7]).all()
    ok = np.isfinite(want)
    ok[1], ok[:, 128:] = False, False
    assert np.isfinite(y[ok]).all()


def test_dense_powers_far_apart():
    """Blocks whose powers are 2^100 apart, and sums beyond 32 bits.  Operands are the values in float32 (include/stt_amd.h): 5 * 2^(254 - 127) is above
    float32's largest, 2^128, and so an infinity, as is 3 * 2^(73 + 100) among the results."""
    v = np.zeros((4, 256))
    v[:, 0], v[:, 128] = 3, 5
    xs = np.array([[27, 227, 127, 127], [0, 254, 127, 127], [200, 54, 127, 127], [127, 127, 127, 127]], np.uint8)
    ws = np.array([[227, 27, 127, 127]], np.uint8)
    x, w = gpu_blocks(v, xs, 256, 1), gpu_blocks(v, ws, 256, 128)
    with np.errstate(over="ignore", invalid="ignore"):
        xd, wd = (R.values(v, a, 256, br).astype(np.float32) for a, br in ((xs, 1), (ws, 128)))
    assert np.isinf(xd[1, 128]) and wd[1, 0] == 3 * 2.0 ** 100
    y = host(blocks.dense_blocks(x, w, dtype=torch.float32))
    assert (y[1:3] == np.inf).all()
    want = R.dense(xd[[0, 3]].astype(np.float64), wd.astype(np.float64))
    small = gpu_blocks(v, np.array([[0, 1, 127, 127]] * 4, np.uint8), 256, 1)                      # 3 * 2^-127 and 5 * 2^-126, at and above 2^-126
    exact = 3 * 2.0 ** -127 * 3 * 2.0 ** 100 + 5 * 2.0 ** -126 * 5 * 2.0 ** -100
    assert (np.abs(host(blocks.dense_blocks(small, w, dtype=torch.float32)) - exact) <= 2.0 ** -22 * exact).all()
    assert (np.abs(y[[0, 3]] - want) <= 2.0 ** -22 * np.abs(want)).all(), (y, want)


@pytest.mark.parametrize("m", [5, 64, 200, 3000])
def test_nothing_is_written_behind_the_results(m):
    """Outputs in the middle of larger buffers: columns behind the last block and rows behind the last row stay as they were."""
    L, rng = native.lib(), np.random.default_rng(m)
    k, n = 200, 300
    x, xd = whole_blocks(rng, m, k, 1)
    w, wd = whole_blocks(rng, n, k, 128)
    want = R.dense(xd, wd)
    a = native.DenseBlocksArgs()
    a.x, a.x_scale, a.x_type, a.x_ld, a.x_scale_ld = x.values.data_ptr(), x.scale.data_ptr(), 3, 256, 4
    a.w, a.w_scale, a.w_ld, a.w_scale_ld = w.values.data_ptr(), w.scale.data_ptr(), 256, 4
    a.rows, a.inner, a.out = m, k, n
    y = torch.full((m + 2, n + 9), 77.0, device="cuda")
    a.y, a.y_ld, a.y_type = y.data_ptr() + 4, n + 9, 0
    assert L.STTX_DenseBlocks(C.byref(a)) == 0
    torch.cuda.synchronize()
    flat = host(y).reshape(-1)
    got = flat[1:1 + m * (n + 9)].reshape(m, n + 9)
    np.testing.assert_array_equal(got[:, :n], want)
    assert flat[0] == 77 and (got[:, n:] == 77).all() and (flat[1 + m * (n + 9):] == 77).all()
    q = torch.full((m + 3, 416), 0x55, dtype=torch.uint8, device="cuda")
    s = torch.full((m + 3, 12), 0x66, dtype=torch.uint8, device="cuda")
    for fill in ("dense", "quantize"):
        q.fill_(0x55), s.fill_(0x66)
        if fill == "dense":
            a.y, a.y_ld, a.y_type, a.y_scale, a.y_scale_ld = q.data_ptr(), 416, 3, s.data_ptr(), 12
            need = L.STTX_DenseBlocksWorkspace(3, 3, m, k, n)
            work = torch.full((need + 16,), 0x77, dtype=torch.uint8, device="cuda")
            a.workspace, a.workspace_bytes = work.data_ptr(), need
            assert L.STTX_DenseBlocks(C.byref(a)) == 0
        else:
            f = torch.from_numpy(want).float().cuda()
            assert L.STTX_QuantizeBlocks(f.data_ptr(), 0, m, n, n, 1, q.data_ptr(), 416, s.data_ptr(), 12, None) == 0
        torch.cuda.synchronize()
        assert (work[need:] == 0x77).all()
        assert (q[m:] == 0x55).all() and (q[:, 384:] == 0x55).all() and (s[m:] == 0x66).all() and (s[:, 4:] == 0x66).all()
        check_blocks(blocks.BlockTensor(q[:m, :384].contiguous().view(E4M3), s[:m, :4].contiguous(), n), want, 1)


def test_rows_far_apart():
    """Row offsets beyond 2^32 bytes, in and out."""
    rng = np.random.default_rng(3)
    for rows in (20, 70, 2900):
        ld = (6 << 30) // rows // 128 * 128
        big = torch.empty(rows * ld, dtype=torch.float16, device="cuda")
        x = big.as_strided((rows, 140), (ld, 1), 0)
        xd = rng.integers(-4, 5, (rows, 140)).astype(float)
        x.copy_(torch.from_numpy(xd).half())
        w, wd = whole_blocks(rng, 200, 140, 128)
        np.testing.assert_array_equal(host(blocks.dense_blocks(x, w, dtype=torch.float32)), R.dense(xd, wd))
        b = blocks.quantize_blocks(x)
        check_blocks(b, xd, 1)
        far = big.view(torch.uint8).as_strided((rows, 256), (2 * ld // 16 * 16, 1), 0)
        far.copy_(b.values.view(torch.uint8))
        fb = blocks.BlockTensor(far.view(E4M3), b.scale, 140)
        np.testing.assert_array_equal(host(blocks.dense_blocks(fb, w, dtype=torch.float32)), R.dense(xd, wd))
        np.testing.assert_array_equal(host(blocks.dequantize_blocks(fb)), xd)
        del big, x, far, fb


def test_more_rows_than_one_grid_dimension_has_threads():
    """2^26 + 5 rows (a wave each: 2^32 threads and more): every row quantised, read back and multiplied, the last ones too."""
    rows = (1 << 26) + 5
    x = (torch.arange(rows, device="cuda", dtype=torch.int32) % 15 + 1).to(torch.float16)[:, None]       # 1 .. 15: whole numbers e4m3 holds
    b = blocks.quantize_blocks(x)
    y = blocks.dequantize_blocks(b, torch.float16)
    assert torch.equal(x, y)
    del y
    w = blocks.quantize_blocks(torch.full((1, 1), 2.0, device="cuda"), 128)
    assert torch.equal(blocks.dense_blocks(b, w, dtype=torch.float16), 2 * x)


def _stack(x, layers, dtype):
    for w, b in layers[:-1]:
        x = blocks.dense_blocks(x, w, b, relu_clip=20.0, dtype=E4M3)
    return blocks.dense_blocks(x, layers[-1][0], layers[-1][1], dtype=dtype)


def _layers(rng, sizes):
    out = []
    for i, o in zip(sizes, sizes[1:]):
        w = torch.from_numpy(rng.integers(-1, 2, (o, i)) * 2.0 ** -3).float().cuda()
        out.append((blocks.quantize_blocks(w, 128), torch.from_numpy(rng.integers(-4, 5, o) / 8.0).float().cuda(), host(w)))
    return out


def _stack_ref(xd, layers):
    for _, b, wd in layers[:-1]:
        y = R.dense(R.values(*R.quantize(xd, 1), xd.shape[1], 1), wd, host(b), 20.0)
        xd = y
    _, b, wd = layers[-1]
    return R.dense(R.values(*R.quantize(xd, 1), xd.shape[1], 1), wd, host(b))


@pytest.mark.parametrize("m", [1, 16, 50, 300, 3000])
def test_stack(m):
    """Layers one behind the other, handed on in blocks, equal to the definition: sums of multiples of 2^-9 below 2^15 are exact in 32 bits."""
    rng = np.random.default_rng(m)
    layers = _layers(rng, [494, 300, 260, 140])
    xd = rng.integers(-8, 9, (m, 494)).astype(float)
    y = _stack(torch.from_numpy(xd).half().cuda(), [(w, b) for w, b, _ in layers], torch.float32)
    np.testing.assert_array_equal(host(y), _stack_ref(xd, layers))


def test_streams_and_graphs():
    """Work on another stream; two graphs of the same layers captured one behind the other, replayed in turn with eager work between."""
    rng = np.random.default_rng(11)
    layers = _layers(rng, [494, 256, 100])
    ops = [(w, b) for w, b, _ in layers]
    for m in (16, 200, 5000):
        side, static, graphs = torch.cuda.Stream(), [], []
        with torch.cuda.stream(side):
            xd = rng.integers(-8, 9, (m, 494)).astype(float)
            y = _stack(torch.from_numpy(xd).half().cuda(), ops, torch.float32)
        side.synchronize()
        np.testing.assert_array_equal(host(y), _stack_ref(xd, layers))
        for _ in range(2):
            x = torch.zeros(m, 494, dtype=torch.float16, device="cuda")
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = _stack(x, ops, torch.float32)
            static.append((x, out))
            graphs.append(g)
        for turn in range(3):
            wants = []
            for (x, _), g in zip(static, graphs):
                xd = rng.integers(-8, 9, (m, 494)).astype(float)
                x.copy_(torch.from_numpy(xd).half())
                wants.append((_stack(x, ops, torch.float32).clone(), xd))
                g.replay()
            torch.cuda.synchronize()
            for (_, out), (eager, xd) in zip(static, wants):
                assert torch.equal(out, eager)
                np.testing.assert_array_equal(host(out), _stack_ref(xd, layers))


def test_refuses_on_the_gpu():
    w = blocks.quantize_blocks(torch.randn(100, 300, device="cuda"), 128)
    x = torch.randn(5, 300, device="cuda")
    b = torch.randn(100, device="cuda")
    ok = blocks.dense_blocks(x, w, b)
    assert ok.shape == (5, 100) and ok.dtype is torch.float16
    for bad in (lambda: blocks.dense_blocks(x[:, :299], w), lambda: blocks.dense_blocks(x.t(), w), lambda: blocks.dense_blocks(x, blocks.quantize_blocks(x)),
                lambda: blocks.dense_blocks(w, w), lambda: blocks.dense_blocks(x, w, b.half()), lambda: blocks.dense_blocks(x, w, b[:99]), lambda: blocks.dense_blocks(x, w, b.cpu()),
                lambda: blocks.dense_blocks(x, w, relu_clip=0.0), lambda: blocks.dense_blocks(x, w, relu_clip=float("nan")), lambda: blocks.dense_blocks(x, w, dtype=torch.float64),
                lambda: blocks.dense_blocks(x.cpu(), w), lambda: blocks.quantize_blocks(x.t()), lambda: blocks.dequantize_blocks(w, E4M3)):
        with pytest.raises(ValueError):
            bad()
    assert blocks.dense_blocks(x[:0], w, b).shape == (0, 100) and blocks.quantize_blocks(x[:0]).shape == (0, 300)
    assert blocks.dequantize_blocks(blocks.quantize_blocks(x[:0])).shape == (0, 300)
    assert blocks.dense_blocks(x[:0], w, b, dtype=E4M3).shape == (0, 100)


def test_clip_has_to_be_a_float32():
    """A clip that float32 rounds to 0 would be no ReLU at all."""
    w = blocks.quantize_blocks(torch.eye(4, device="cuda"), 128)
    x = torch.tensor([[-4.0, 0.5, 8.0, 448.0]], device="cuda")
    for clip in (1e-50, 1e-39, 1e39, -1.0, -float("inf")):
        with pytest.raises(ValueError):
            blocks.dense_blocks(x, w, relu_clip=clip)
    assert host(blocks.dense_blocks(x, w, relu_clip=float("inf"), dtype=torch.float32)).tolist() == [[0.0, 0.5, 8.0, 448.0]]
    assert host(blocks.dense_blocks(x, w, relu_clip=torch.finfo(torch.float32).tiny, dtype=torch.float32)).tolist() == [[0.0] + 3 * [float(torch.finfo(torch.float32).tiny)]]


def test_threads():
    """Calls from four threads at once, each on a stream of its own, all forms: every thread has its own results."""
    import threading
    rng = np.random.default_rng(12)
    layers = _layers(rng, [494, 300, 100])
    ops = [(w, b) for w, b, _ in layers]
    sizes = (1, 16, 200, 5000)
    data = [rng.integers(-8, 9, (m, 494)).astype(float) for m in sizes]
    wants = [_stack_ref(xd, layers) for xd in data]
    torch.cuda.synchronize()
    got, errors = {}, []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                x = torch.from_numpy(data[i]).half().cuda()
                ys = [_stack(x, ops, torch.float32) for _ in range(20)]
            s.synchronize()
            got[i] = [host(y) for y in ys]
        except Exception as e:                    # told by the test's own thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sizes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for i, want in enumerate(wants):
        for y in got[i]:
            np.testing.assert_array_equal(y, want)


@pytest.mark.parametrize("m", [3, 40, 700])
def test_parts_of_block_tensors(m):
    """Rows out of the middle of a BlockTensor, features from a row of blocks on, fewer columns than the values have room for; results are detached."""
    rng = np.random.default_rng(m)
    xb, xd = whole_blocks(rng, m + 9, 300, 1)
    wb, wd = whole_blocks(rng, 400, 300, 128)
    x = blocks.BlockTensor(xb.values[4:4 + m], xb.scale[4:4 + m], 300)
    w = blocks.BlockTensor(wb.values[128:], wb.scale[1:], 300, 128)
    np.testing.assert_array_equal(host(blocks.dense_blocks(x, w, dtype=torch.float32)), R.dense(xd[4:4 + m], wd[128:]))
    np.testing.assert_array_equal(host(blocks.dequantize_blocks(x)), xd[4:4 + m])
    x1 = blocks.BlockTensor(x.values, x.scale, 256)                          # the first two blocks of a row
    w1 = blocks.BlockTensor(w.values, w.scale, 256, 128)
    np.testing.assert_array_equal(host(blocks.dense_blocks(x1, w1, dtype=torch.float32)), R.dense(xd[4:4 + m, :256], wd[128:, :256]))
    p = torch.ones(4, 300, device="cuda", requires_grad=True)
    assert not blocks.dense_blocks(p, w, dtype=torch.float32).requires_grad and not blocks.dequantize_blocks(blocks.quantize_blocks(p)).requires_grad


@pytest.mark.parametrize("k", [1, 128, 200, 300, 500, 640, 1025])
@pytest.mark.parametrize("m,n", [(300, 900), (999, 1100), (2500, 2100)])
def test_dense_blocks_along_k(m, n, k):
    """Tiles of 32, 64 and 128 rows over one block along k, fewer than they keep in flight, and more than one word of scale bytes; equal in every bit."""
    rng = np.random.default_rng(m + k)
    x, xd = whole_blocks(rng, m, k, 1)
    w, wd = whole_blocks(rng, n, k, 128)
    want = R.dense(xd, wd, None, None)
    for t, dt in TYPES.items():
        np.testing.assert_array_equal(host(blocks.dense_blocks(x, w, dtype=dt)), host(torch.from_numpy(want).float().to(dt)), err_msg=t)
    check_blocks(blocks.dense_blocks(x, w, dtype=E4M3), want, 1)


@pytest.mark.parametrize("k", [1, 100, 128, 129])
@pytest.mark.parametrize("m,n", [(300, 900), (999, 1100), (2500, 2100)])
def test_dense_bias_over_one_block(m, n, k):
    """The biases are in LDS before any wave adds them, also where a tile passes one barrier only: one block along k (and two, at 129), a bias, tiles of 32, 64
    and 128 rows, every type of result; equal in every bit."""
    rng = np.random.default_rng(m + k)
    x, xd = whole_blocks(rng, m, k, 1)
    w, wd = whole_blocks(rng, n, k, 128)
    bias = rng.integers(-900, 901, n) / 4.0
    bg = torch.from_numpy(bias).float().cuda()
    for clip in (None, 100.0):
        want = R.dense(xd, wd, bias, clip)
        for t, dt in TYPES.items():
            np.testing.assert_array_equal(host(blocks.dense_blocks(x, w, bg, relu_clip=clip, dtype=dt)), host(torch.from_numpy(want).float().to(dt)), err_msg="%s %s" % (t, clip))
        check_blocks(blocks.dense_blocks(x, w, bg, relu_clip=clip, dtype=E4M3), want, 1)


def test_block_tensors_of_one_row():
    """The stride of a single row means nothing: any will do, of values, of scales and of a plain x."""
    rng = np.random.default_rng(21)
    xb, xd = whole_blocks(rng, 1, 300, 1)
    wb, wd = whole_blocks(rng, 100, 300, 128)
    w1, w1d = whole_blocks(rng, 1, 300, 128)
    for ld, lds in ((1, 1), (0, 0), (7, 3), (385, 5)):
        x = blocks.BlockTensor(xb.values.as_strided((1, 384), (ld, 1)), xb.scale.as_strided((1, 4), (lds, 1)), 300)
        w = blocks.BlockTensor(wb.values, wb.scale.as_strided((1, 4), (lds, 1)), 300, 128)
        np.testing.assert_array_equal(host(blocks.dequantize_blocks(x)), xd)
        np.testing.assert_array_equal(host(blocks.dense_blocks(x, w, dtype=torch.float32)), R.dense(xd, wd))
        one = blocks.BlockTensor(w1.values.as_strided((1, 384), (ld, 1)), w1.scale.as_strided((1, 4), (lds, 1)), 300, 128)
        np.testing.assert_array_equal(host(blocks.dense_blocks(x, one, dtype=torch.float32)), R.dense(xd, w1d))
        np.testing.assert_array_equal(host(blocks.dense_blocks(torch.from_numpy(xd).half().cuda().as_strided((1, 300), (ld, 1)), w, dtype=torch.float32)), R.dense(xd, wd))


def test_block_tensors_whose_rows_are_refused():
    """Rows that overlap or start elsewhere than at 16 bytes (values) or 4 bytes (scales) are told as such, before the entry is called."""
    rng = np.random.default_rng(22)
    x, _ = whole_blocks(rng, 6, 600, 1)
    w, _ = whole_blocks(rng, 300, 600, 128)
    flat, marks = x.values.view(torch.uint8).reshape(-1), x.scale.reshape(-1)
    for v, s, cols in ((x.values[:1].expand(6, 640), x.scale, 600), (x.values, x.scale[:1].expand(6, 8), 600),
                       (flat.as_strided((4, 640), (512, 1)).view(E4M3), x.scale, 600), (flat.as_strided((4, 640), (648, 1)).view(E4M3), x.scale, 600),
                       (flat.as_strided((4, 640), (640, 1), 8).view(E4M3), x.scale, 600), (x.values, marks.as_strided((6, 8), (6, 1)), 600),
                       (x.values[:4], marks.as_strided((4, 8), (9, 1)), 600), (x.values[:, 128:], x.scale[:, 1:], 100), (x.values[:1], x.scale[:1, 2:], 100)):
        b = blocks.BlockTensor(v, s, cols)
        part = blocks.BlockTensor(w.values, w.scale, cols, 128)
        for call in (lambda: blocks.dequantize_blocks(b), lambda: blocks.dense_blocks(b, part)):
            with pytest.raises(ValueError, match="multiples of 16"):
                call()
    with pytest.raises(ValueError, match="multiples of 16"):
        blocks.dense_blocks(x, blocks.BlockTensor(w.values, w.scale[:1].expand(3, 8), 600, 128))


@pytest.mark.parametrize("k", [256, 300, 513, 1025, 2048])
def test_dense_256_row_tiles_along_k(k):
    """The tile of the largest products over two blocks along k and more, partial ones and several words of scale bytes; equal in every bit: sums of multiples of
    2^-2 below 2^18 are exact in 32 bits."""
    m, n = 4500, 4100
    rng = np.random.default_rng(k)
    x, xd = whole_blocks(rng, m, k, 1)
    w, wd = whole_blocks(rng, n, k, 128)
    bias = rng.integers(-900, 901, n) / 4.0
    want = R.dense(xd, wd, bias, None)
    bg = torch.from_numpy(bias).float().cuda()
    for t, dt in TYPES.items():
        np.testing.assert_array_equal(host(blocks.dense_blocks(x, w, bg, dtype=dt)), host(torch.from_numpy(want).float().to(dt)), err_msg=t)
    check_blocks(blocks.dense_blocks(x, w, bg, relu_clip=100.0, dtype=E4M3), R.dense(xd, wd, bias, 100.0), 1)


@pytest.mark.parametrize("kind", ["blocks", "f16"])
def test_dense_256_row_tiles_real_values(kind):
    """As test_dense_real_values (its tolerance), in the tile of the largest products."""
    m, k, n = 4500, 2048, 4100
    g = torch.Generator().manual_seed(6)
    x = (torch.randn(m, k, generator=g) * torch.exp(torch.randn(m, 1, generator=g))).half()
    w = torch.randn(n, k, generator=g) * torch.exp(torch.randn(n, 1, generator=g)) / k ** 0.5
    bias = torch.randn(n, generator=g)
    xd, wd = (R.values(*R.quantize(host(v), br), k, br) for v, br in ((x, 1), (w, 128)))
    xin = gpu_blocks(*R.quantize(host(x), 1), k, 1) if kind == "blocks" else x.cuda()
    want, size = R.dense(xd, wd, host(bias)), np.abs(xd) @ np.abs(wd).T + np.abs(host(bias))
    got = host(blocks.dense_blocks(xin, blocks.quantize_blocks(w.cuda(), 128), bias.cuda(), dtype=torch.float32))
    assert (np.abs(got - want) <= (k + 1) * 2.0 ** -23 * size * (1 + 2.0 ** -24) + 2.0 ** -24 * np.abs(want)).all()


@pytest.mark.parametrize("k", [100, 494, 2048])
def test_tiles_of_every_height_give_the_same_bits(k):
    """Real rows in batches that take tiles of 32, 64, 128 and 256 rows, from the batch's start and from within a tile: a row's sums run in one order, so its f32
    bits and its blocks are the same in all of them."""
    n = 4100
    x = torch.randn(4500, k, device="cuda") * torch.exp(torch.randn(4500, 1, device="cuda"))
    xb = blocks.quantize_blocks(x)
    w = blocks.quantize_blocks(torch.randn(n, k, device="cuda"), 128)
    b = torch.randn(n, device="cuda")
    whole, held = blocks.dense_blocks(xb, w, b, dtype=torch.float32), blocks.dense_blocks(xb, w, b, relu_clip=20.0, dtype=E4M3)
    for first, rows in ((0, 200), (37, 224), (0, 600), (101, 896), (0, 2000), (333, 3800)):
        part = blocks.BlockTensor(xb.values[first:first + rows], xb.scale[first:first + rows], k)
        assert torch.equal(blocks.dense_blocks(part, w, b, dtype=torch.float32).view(torch.int32), whole[first:first + rows].view(torch.int32)), (first, rows)
        h = blocks.dense_blocks(part, w, b, relu_clip=20.0, dtype=E4M3)
        assert torch.equal(h.values.view(torch.uint8), held.values[first:first + rows].view(torch.uint8)) and torch.equal(h.scale, held.scale[first:first + rows]), (first, rows)
