"""The block-scaled 8-bit operators without a GPU: the reference's own format against torch's e4m3, and what the entries refuse before any GPU work."""
import ctypes as C

import numpy as np
import pytest
import torch

import blocks_ref as R
from stt_amd import blocks, native

INVALID_SHAPE = 0x2001


@pytest.fixture(scope="module")
def L():
    return native.lib()


def test_reference_codes_are_torchs_e4m3():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(codes, R.e4m3_values())
    x = np.concatenate([np.linspace(-448, 448, 4001), np.float64(np.random.RandomState(0).randn(4000).astype(np.float32)), np.arange(-512, 513) / 2.0 ** 11])
    np.testing.assert_array_equal(torch.from_numpy(x).float().to(torch.float8_e4m3fn).double().numpy(), R.round_e4m3(np.float64(np.float32(x))))


def test_reference_powers():
    for top, byte in ((448.0, 127), (448.0 + 2.0 ** -15, 128), (1.0, 119), (1.75, 119), (1.7500001, 120), (0.0, 127), (2.0 ** -140, 0), (3.0e38, 247), (448 * 2.0 ** -127, 0)):
        x = np.zeros((1, 130))
        x[0, 5] = -np.float64(np.float32(top))
        assert R.quantize(x, 1)[1][0].tolist() == [byte, 127, 127, 127], top
    rng = np.random.RandomState(1)
    for top in np.float64(np.float32(np.concatenate([np.ldexp(rng.uniform(0.5, 1, 200), rng.randint(-148, 129, 200)), np.ldexp(448.0, rng.randint(-127, 119, 40))]))):
        p = -127
        while top > np.ldexp(448.0, p):
            p += 1
        assert R.quantize(np.full((1, 1), top), 1)[1][0, 0] == p + 127, top


def _quant(L, x=0x10000, type=0, rows=4, cols=200, ldx=200, block_rows=1, q=0x20000, ldq=256, scale=0x30000, lds=4):
    return L.STTX_QuantizeBlocks(x, type, rows, cols, ldx, block_rows, q, ldq, scale, lds, None)


def test_quantize_refuses(L, capfd):
    for bad in (dict(x=None), dict(x=0x10002), dict(type=3), dict(type=-1), dict(rows=-1), dict(rows=1 << 31), dict(cols=0), dict(cols=-5), dict(cols=1 << 31), dict(ldx=-200),
                dict(block_rows=2), dict(block_rows=0), dict(block_rows=128, rows=128 * 65535 + 1), dict(q=None), dict(q=0x20008), dict(ldq=200), dict(ldq=264), dict(ldq=240),
                dict(scale=None), dict(scale=0x30002), dict(lds=2), dict(lds=3), dict(cols=600, ldx=600, ldq=640, lds=4), dict(ldx=1 << 50)):
        assert _quant(L, **bad) == INVALID_SHAPE, bad
        assert "STTX_QuantizeBlocks" in capfd.readouterr().err, bad
    assert _quant(L, rows=0) == 0                       # nothing to do, no GPU needed
    assert _quant(L, rows=0, x=None, q=None, scale=None) == 0


def _dequant(L, q=0x20000, ldq=256, scale=0x30000, lds=4, rows=4, cols=200, block_rows=128, y=0x10000, type=1, ldy=200):
    return L.STTX_DequantizeBlocks(q, ldq, scale, lds, rows, cols, block_rows, y, type, ldy, None)


def test_dequantize_refuses(L, capfd):
    for bad in (dict(q=None), dict(q=0x20001), dict(ldq=128), dict(scale=None), dict(lds=0), dict(rows=-1), dict(cols=0), dict(block_rows=64), dict(y=None), dict(y=0x10001), dict(type=3),
                dict(type=7), dict(ldy=199), dict(ldy=0)):
        assert _dequant(L, **bad) == INVALID_SHAPE, bad
        assert "STTX_DequantizeBlocks" in capfd.readouterr().err, bad
    assert _dequant(L, rows=0) == 0


def _dense(L, **change):
    a = native.DenseBlocksArgs()
    a.x, a.x_scale, a.x_type, a.x_ld, a.x_scale_ld = 0x10000, 0x20000, 3, 256, 4
    a.w, a.w_scale, a.w_ld, a.w_scale_ld = 0x30000, 0x40000, 256, 4
    a.bias, a.y, a.y_ld, a.y_type = 0x50000, 0x60000, 300, 0
    a.rows, a.inner, a.out = 70, 200, 300
    for k, v in change.items():
        setattr(a, k, v)
    return L.STTX_DenseBlocks(C.byref(a))


def test_dense_refuses(L, capfd):
    for bad in (dict(rows=-1), dict(rows=1 << 31), dict(inner=0), dict(out=0), dict(inner=1 << 31), dict(x=None), dict(x_scale=None), dict(x_type=4), dict(x=0x10008), dict(x_ld=200), dict(x_ld=128),
                dict(x_scale_ld=2), dict(w=None), dict(w_scale=None), dict(w=0x30004), dict(w_ld=250), dict(w_scale_ld=1), dict(bias=0x50002), dict(y=None), dict(y=0x60002), dict(y_ld=299),
                dict(y_type=5), dict(y_type=3, y_ld=384), dict(y_type=3, y_ld=300, y_scale=0x70000, y_scale_ld=4), dict(y_type=3, y_ld=384, y_scale=0x70000, y_scale_ld=3),
                dict(relu_clip=-1.0), dict(relu_clip=float("nan")),
                dict(x_type=1, x_ld=200, rows=7000),                                       # 7000 rows of f16 need a workspace
                dict(x_type=1, x_ld=200, rows=7000, workspace=0x80000, workspace_bytes=7000 * 260 - 1), dict(x_type=1, x_ld=200, rows=7000, workspace=0x80004, workspace_bytes=1 << 30),
                dict(y_type=3, y_ld=384, y_scale=0x70000, y_scale_ld=4, workspace=0x80000, workspace_bytes=70 * 300 * 4 - 1)):
        assert _dense(L, **bad) == INVALID_SHAPE, bad
        assert "STTX_DenseBlocks" in capfd.readouterr().err, bad
    assert L.STTX_DenseBlocks(None) == INVALID_SHAPE
    assert _dense(L, rows=0) == 0


def test_workspace(L):
    W = L.STTX_DenseBlocksWorkspace
    assert W(3, 0, 1 << 20, 2048, 8192) == 0                  # already in blocks
    assert W(0, 1, 1, 2048, 2048) == 0                        # few rows are quantised on the way
    assert W(3, 3, 16, 2048, 2046) == 16 * 2048 * 4           # ... and their results, where those go on in blocks
    assert W(1, 3, 100, 494, 2046) == (100 * (512 + 4) + 15) // 16 * 16 + 100 * 2048 * 4       # ... of a few more, both
    assert W(1, 0, 6144, 494, 2048) == 6144 * (512 + 4) == W(1, 3, 6144, 494, 2048)
    assert W(2, 2, 1 << 20, 130, 2048) == (1 << 20) * (256 + 4)
    assert W(9, 0, 100, 100, 100) == 0 and W(0, 0, -1, 100, 100) == 0 and W(0, -1, 5000, 100, 9000) == 0 and W(0, 0, 5000, 0, 9000) == 0


def test_argument_block_is_the_structure():
    v = tuple(range(1, 10)) + tuple(range(-6, 0)) + (77,) + (8, 9, 10) + (2, 3, 20.0)
    assert blocks._ARGS(*v) == bytes(native.DenseBlocksArgs(*v)) and C.sizeof(native.DenseBlocksArgs) == len(blocks._ARGS(*v))


def test_python_refuses():
    x = torch.zeros(4, 200)
    w = blocks.BlockTensor(torch.zeros(300, 256).to(torch.float8_e4m3fn), torch.zeros(3, 4, dtype=torch.uint8), 200, 128)
    for bad in (x, x.double(), x[0], x.to(torch.int8), x.t()):
        with pytest.raises(ValueError):
            blocks.quantize_blocks(bad)
    with pytest.raises(ValueError):
        blocks.quantize_blocks(x, block_rows=64)
    with pytest.raises(ValueError):
        blocks.dequantize_blocks(w)                                      # not in GPU memory
    with pytest.raises(ValueError):
        blocks.dense_blocks(x, w)
    for v, s, cols, br in ((torch.zeros(3, 256), torch.zeros(3, 4, dtype=torch.uint8), 200, 1), (w.values, w.scale, 300, 128), (w.values, w.scale, 0, 128), (w.values, w.scale[:2], 200, 128),
                           (w.values, w.scale[:, :2], 200, 128), (w.values, w.scale, 200, 1), (w.values, w.scale, 200, 16), (w.values, w.scale.to(torch.int8), 200, 128)):
        with pytest.raises(ValueError):
            blocks.dequantize_blocks(blocks.BlockTensor(v, s, cols, br))
    assert repr(w) == "BlockTensor(300 x 200, blocks of 128 x 128)" and w.shape == (300, 200)


def test_more_rows_than_a_launch_holds(L, capfd):
    """Refused with the other arguments, before anything is enqueued: 2^39 groups of four blocks there and back; 2^24 tiles of 256 x 128 of a dense layer, with x
    in blocks and with an x that a quantising launch would go in front of."""
    many, wide = (1 << 31) - 1, 1 << 17
    assert _quant(L, rows=many, cols=wide, ldx=0, ldq=wide, lds=wide // 128) == INVALID_SHAPE
    assert "too many rows" in capfd.readouterr().err
    assert _dequant(L, rows=many, cols=wide, ldq=wide, lds=wide // 128, ldy=wide) == INVALID_SHAPE
    assert "too many rows" in capfd.readouterr().err
    assert _dense(L, rows=many, out=129, y_ld=129) == INVALID_SHAPE
    assert "too many rows" in capfd.readouterr().err
    assert _dense(L, rows=many, out=129, y_ld=129, x_type=1, x_ld=0, workspace=0x80000, workspace_bytes=1 << 60) == INVALID_SHAPE
    assert "too many rows" in capfd.readouterr().err
