"""stt_amd/blocks.py -- the block-scaled 8-bit operators of include/stt_amd.h (STTX_QuantizeBlocks, STTX_DequantizeBlocks, STTX_DenseBlocks) on torch
tensors in HBM: 8-bit floating point (e4m3) with one power of two per block of 128 values along a row.

    w = quantize_blocks(weight, block_rows=128)                     # [out][in], once: blocks of 128 x 128
    h = dense_blocks(x, w, bias, relu_clip=20.0, dtype=torch.float8_e4m3fn)   # x f32 / f16 / bf16 or a BlockTensor; h handed on in blocks
    y = dense_blocks(h, v, c, dtype=torch.float16)
    f = dequantize_blocks(h, torch.float32)                         # a hidden layer's rows read back

Calls enqueue on torch's current stream of the tensors' device and allocate with torch, so they can be captured into a graph like any torch
call.  No compute happens in Python; there is no fallback for tensors elsewhere, and there are no gradients: results are detached.

A call on a few rows is over in less time than a careless caller needs to make it, so the checks below are one expression each on the way that
succeeds, and the messages are put together on the way that fails.
"""
import struct

import torch

from . import native

BLOCK = 128
E4M3 = torch.float8_e4m3fn
_PLAIN = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}            # STTX_ElementType
_E4M3 = 3
_CLIP_MIN, _CLIP_MAX = torch.finfo(torch.float32).tiny, torch.finfo(torch.float32).max   # (as a float32 nothing below it may become 0: no ReLU)
_UINT8 = torch.uint8
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_ARGS = struct.Struct("9Q6q1Q3q2if4x").pack                                  # native.DenseBlocksArgs as bytes: a third of the time of filling one in
_lib = None


def _entry():
    """The library and the number of devices, looked up on first use."""
    global _lib, _devices
    _devices = torch.cuda.device_count()
    _lib = native.lib()
    return _lib


class BlockTensor(object):
    """A matrix in blocks: `values` float8_e4m3fn [rows][cols rounded up to 128], `scale` uint8 [rows or row blocks][blocks rounded up to 4] (byte s
    stands for 2^(s - 127)), `cols` columns that count, blocks of `block_rows` (1 or 128) x 128.  The padding of `values` is zeros.  Parts of larger
    matrices will do whose rows do not overlap and start at multiples of 16 (values) and 4 bytes (scale)."""
    __slots__ = ("values", "scale", "cols", "block_rows")

    def __init__(self, values, scale, cols, block_rows=1):
        self.values, self.scale, self.cols, self.block_rows = values, scale, cols, block_rows

    @property
    def shape(self):
        return (self.values.shape[0], self.cols)

    def __repr__(self):
        return "BlockTensor(%d x %d, blocks of %d x %d)" % (self.values.shape[0], self.cols, self.block_rows, BLOCK)


def _bad_plain(t, what):
    if t.dim() != 2 or t.dtype not in _PLAIN:
        return ValueError("%s: a two-dimensional float32, float16 or bfloat16 tensor is wanted, got %s %s" % (what, t.dtype, tuple(t.shape)))
    if t.shape[1] < 1:
        return ValueError("%s: at least one column is wanted" % what)
    if not t.is_cuda:
        return ValueError("%s: has to be in GPU memory, got a tensor on %s" % (what, t.device))
    return ValueError("%s: columns have to be contiguous (stride 1), got stride %d" % (what, t.stride(1)))


def _plain(t, what):
    """(type, rows, cols, row stride, device index)"""
    shape, kind = t.shape, _PLAIN.get(t.dtype, -1)
    if kind < 0 or len(shape) != 2 or shape[1] < 1 or not t.is_cuda or (t.stride(1) != 1 and shape[1] > 1):
        raise _bad_plain(t, what)
    return kind, shape[0], shape[1], t.stride(0), t.get_device()


def _bad_blocks(b, what, block_rows):
    v, s = b.values, b.scale
    if v.dtype is not E4M3 or v.dim() != 2 or s.dtype is not _UINT8 or s.dim() != 2:
        return ValueError("%s: values are a float8_e4m3fn matrix and scales a uint8 matrix, got %s %s and %s %s" % (what, v.dtype, tuple(v.shape), s.dtype, tuple(s.shape)))
    if b.block_rows not in block_rows:
        return ValueError("%s: blocks of %s rows are wanted, got %r" % (what, " or ".join(map(str, block_rows)), b.block_rows))
    if b.cols < 1 or v.shape[1] < -(-b.cols // BLOCK) * BLOCK:
        return ValueError("%s: %d columns of values do not hold %d columns rounded up to 128" % (what, v.shape[1], b.cols))
    if s.shape[0] < -(-v.shape[0] // b.block_rows) or s.shape[1] < -(-b.cols // 512) * 4:
        return ValueError("%s: scales %s do not cover the blocks of %d x %d values" % (what, tuple(s.shape), v.shape[0], b.cols))
    if not v.is_cuda or v.device != s.device:
        return ValueError("%s: values and scales have to be in one GPU's memory, got %s and %s" % (what, v.device, s.device))
    if v.stride(1) != 1 or s.stride(1) != 1:
        return ValueError("%s: columns have to be contiguous (stride 1)" % what)
    return ValueError("%s: rows must not overlap and have to start at multiples of 16 bytes (values) and 4 bytes (scale), got strides of %d and %d from 0x%x and 0x%x" %
                      (what, v.stride(0), s.stride(0), v.data_ptr(), s.data_ptr()))


def _blocks(b, what, block_rows):
    """(rows, cols, values' address and row stride, scales' address and row stride, device index); block_rows: the ones that may be"""
    v, s, cols, br = b.values, b.scale, b.cols, b.block_rows
    vs, ss = v.shape, s.shape
    if (v.dtype is not E4M3 or s.dtype is not _UINT8 or len(vs) != 2 or len(ss) != 2 or br not in block_rows or cols < 1 or vs[1] < (wide := -(-cols // BLOCK) * BLOCK) or
            ss[0] * br < vs[0] or ss[1] < (words := -(-cols // 512) * 4) or not v.is_cuda or v.get_device() != s.get_device()):
        raise _bad_blocks(b, what, block_rows)
    (ldq, one), (lds, unit), q, scale = v.stride(), s.stride(), v.data_ptr(), s.data_ptr()
    if one != 1 or unit != 1 or ldq < wide or lds < words or (ldq | q) & 15 or (lds | scale) & 3:
        if vs[0] < 2:                       # (torch leaves the stride of a single row open)
            ldq = wide
        if ss[0] < 2:
            lds = words
        if one != 1 or unit != 1 or ldq < wide or lds < words or (ldq | q) & 15 or (lds | scale) & 3:
            raise _bad_blocks(b, what, block_rows)
    return vs[0], cols, q, ldq, scale, lds, v.get_device()


def _call(index, fn, *args):
    """The entry with the tensors' device current: a torch stream number of 0 is the CURRENT device's default stream."""
    if _devices == 1 or index == torch.cuda.current_device():
        status = fn(*args)
    else:
        with torch.cuda.device(index):
            status = fn(*args)
    if status != 0:
        raise RuntimeError("block operator failed with '%s' (0x%X)" % (native.error_message(status), status))


def quantize_blocks(x, block_rows=1):
    """x [rows][cols] float32 / float16 / bfloat16 -> BlockTensor in blocks of block_rows (1: activations, 128: weights) x 128."""
    kind, rows, cols, ld, index = _plain(x, "x")
    if block_rows != 1 and block_rows != BLOCK:
        raise ValueError("blocks have 1 or 128 rows, got %r" % (block_rows,))
    ldq, lds = -(-cols // BLOCK) * BLOCK, -(-cols // 512) * 4
    values = x.new_empty((rows, ldq), dtype=E4M3)
    scale = x.new_empty((-(-rows // block_rows), lds), dtype=_UINT8)
    _call(index, (_lib or _entry()).STTX_QuantizeBlocks, x.data_ptr(), kind, rows, cols, ld, block_rows, values.data_ptr(), ldq, scale.data_ptr(), lds, _raw_stream(index))
    return BlockTensor(values, scale, cols, block_rows)


def dequantize_blocks(b, dtype=torch.float32):
    """BlockTensor -> [rows][cols] of `dtype` (float32, float16, bfloat16), one rounding."""
    rows, cols, q, ldq, scale, lds, index = _blocks(b, "b", (1, BLOCK))
    kind = _PLAIN.get(dtype, -1)
    if kind < 0:
        raise ValueError("dtype: float32, float16 or bfloat16 is wanted, got %s" % (dtype,))
    y = b.scale.new_empty((rows, cols), dtype=dtype)
    _call(index, (_lib or _entry()).STTX_DequantizeBlocks, q, ldq, scale, lds, rows, cols, b.block_rows, y.data_ptr(), kind, cols, _raw_stream(index))
    return y


def dense_blocks(x, w, bias=None, relu_clip=None, dtype=torch.float16):
    """A dense layer: x . w^T + bias, with the clipped ReLU min(max(y, 0), relu_clip) if one is given.

    x: [rows][in] float32 / float16 / bfloat16 (quantised within the call) or a BlockTensor in blocks of 1 x 128; w: BlockTensor [out][in] in blocks of
    128 x 128; bias: float32 [out].  Returns [rows][out] of `dtype`, or for dtype float8_e4m3fn a BlockTensor in blocks of 1 x 128."""
    out, inner, w_ptr, w_ld, w_scale, w_scale_ld, index = _blocks(w, "w", (BLOCK,))
    if isinstance(x, BlockTensor):
        rows, cols, x_ptr, x_ld, x_scale, x_scale_ld, at = _blocks(x, "x", (1,))
        kind = _E4M3
    else:
        kind, rows, cols, x_ld, at = _plain(x, "x")
        x_ptr, x_scale, x_scale_ld = x.data_ptr(), 0, 0
    if cols != inner or out < 1:
        raise ValueError("x has %d columns, w is %d x %d" % (cols, out, inner))
    if at != index:
        raise ValueError("x is on device %d, w on device %d" % (at, index))
    b_ptr = 0
    if bias is not None:
        if bias.dtype is not torch.float32 or bias.dim() != 1 or bias.shape[0] != out or bias.get_device() != index or (bias.stride(0) != 1 and out > 1):
            raise ValueError("bias: a contiguous float32 vector of %d on device %d is wanted, got %s %s on %s" % (out, index, bias.dtype, tuple(bias.shape), bias.device))
        b_ptr = bias.data_ptr()
    clip = 0.0
    if relu_clip is not None:
        if not _CLIP_MIN <= relu_clip <= _CLIP_MAX and relu_clip != float("inf"):
            raise ValueError("relu_clip: a positive number of float32's normal range, inf or None is wanted, got %r" % (relu_clip,))
        clip = relu_clip
    L = _lib or _entry()
    if dtype is E4M3:
        y_ld, y_scale_ld = -(-out // BLOCK) * BLOCK, -(-out // 512) * 4
        y = BlockTensor(w.scale.new_empty((rows, y_ld), dtype=E4M3), w.scale.new_empty((rows, y_scale_ld), dtype=_UINT8), out)
        y_kind, y_ptr, y_scale = _E4M3, y.values.data_ptr(), y.scale.data_ptr()
    else:
        y_kind = _PLAIN.get(dtype, -1)
        if y_kind < 0:
            raise ValueError("dtype: float32, float16, bfloat16 or float8_e4m3fn is wanted, got %s" % (dtype,))
        y = w.scale.new_empty((rows, out), dtype=dtype)
        y_ptr, y_ld, y_scale, y_scale_ld = y.data_ptr(), out, 0, 0
    need = L.STTX_DenseBlocksWorkspace(kind, y_kind, rows, inner, out) if kind != _E4M3 or y_kind == _E4M3 else 0
    work = w.scale.new_empty(need) if need else None         # torch's allocator: this stream's, or the capturing graph's own
    args = _ARGS(x_ptr, x_scale, w_ptr, w_scale, b_ptr, y_ptr, y_scale, work.data_ptr() if need else 0, _raw_stream(index),
                                  x_ld, x_scale_ld, w_ld, w_scale_ld, y_ld, y_scale_ld, need, rows, inner, out, kind, y_kind, clip)
    _call(index, L.STTX_DenseBlocks, args)
    return y
