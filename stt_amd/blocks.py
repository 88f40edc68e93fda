"""stt_amd/blocks.py -- the block-scaled 8-bit operators of include/stt_amd.h (STTX_QuantizeBlocks, STTX_DequantizeBlocks, STTX_DenseBlocks) on torch
tensors in HBM: 8-bit floating point (e4m3) with one power of two per block of 128 values along a row.

    w = quantize_blocks(weight, block_rows=128)                     # [out][in], once: blocks of 128 x 128
    h = dense_blocks(x, w, bias, relu_clip=20.0, dtype=torch.float8_e4m3fn)   # x f32 / f16 / bf16 or a BlockTensor; h handed on in blocks
    y = dense_blocks(h, v, c, dtype=torch.float16)
    f = dequantize_blocks(h, torch.float32)                         # a hidden layer's rows read back

Calls enqueue on torch's current stream of the tensors' device and allocate with torch, so they can be captured into a graph like any torch
call.  No compute happens in Python; there is no fallback for tensors elsewhere.
"""
import ctypes as C

import torch

from . import native

BLOCK = 128
E4M3 = torch.float8_e4m3fn
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, E4M3: 3}   # STTX_ElementType


def _up(n, to):
    return -(-n // to) * to


class BlockTensor(object):
    """A matrix in blocks: `values` float8_e4m3fn [rows][cols rounded up to 128], `scale` uint8 [rows or row blocks][blocks rounded up to 4] (byte s
    stands for 2^(s - 127)), `cols` columns that count, blocks of `block_rows` (1 or 128) x 128.  The padding of `values` is zeros."""
    __slots__ = ("values", "scale", "cols", "block_rows")

    def __init__(self, values, scale, cols, block_rows=1):
        self.values, self.scale, self.cols, self.block_rows = values, scale, cols, block_rows

    @property
    def shape(self):
        return (self.values.shape[0], self.cols)

    def __repr__(self):
        return "BlockTensor(%d x %d, blocks of %d x %d)" % (self.values.shape[0], self.cols, self.block_rows, BLOCK)


def _plain(t, what):
    if t.dim() != 2 or t.dtype not in _TYPES or t.dtype is E4M3:
        raise ValueError("%s: a two-dimensional float32, float16 or bfloat16 tensor is wanted, got %s %s" % (what, t.dtype, tuple(t.shape)))
    if t.stride(1) != 1 and t.shape[1] > 1:
        raise ValueError("%s: columns have to be contiguous (stride 1), got stride %d" % (what, t.stride(1)))
    if not t.is_cuda:
        raise ValueError("%s: has to be in GPU memory, got a tensor on %s" % (what, t.device))


def _blocks(b, what, block_rows=None):
    v, s = b.values, b.scale
    if v.dtype is not E4M3 or v.dim() != 2 or s.dtype is not torch.uint8 or s.dim() != 2:
        raise ValueError("%s: values are a float8_e4m3fn matrix and scales a uint8 matrix, got %s %s and %s %s" % (what, v.dtype, tuple(v.shape), s.dtype, tuple(s.shape)))
    if b.block_rows not in (1, BLOCK) or (block_rows is not None and b.block_rows != block_rows):
        raise ValueError("%s: blocks of %s rows are wanted, got %r" % (what, "1 or 128" if block_rows is None else block_rows, b.block_rows))
    rows, cols = v.shape
    if b.cols < 1 or cols < _up(b.cols, BLOCK):
        raise ValueError("%s: %d columns of values do not hold %d columns rounded up to 128" % (what, cols, b.cols))
    if s.shape[0] < -(-rows // b.block_rows) or s.shape[1] < _up(-(-b.cols // BLOCK), 4):
        raise ValueError("%s: scales %s do not cover the blocks of %d x %d values" % (what, tuple(s.shape), rows, b.cols))
    if v.stride(1) != 1 or s.stride(1) != 1:
        raise ValueError("%s: columns have to be contiguous (stride 1)" % what)
    if not v.is_cuda or v.device != s.device:
        raise ValueError("%s: values and scales have to be in one GPU's memory, got %s and %s" % (what, v.device, s.device))


def _call(device, status_of):
    """Runs `status_of` with the device current (a torch stream number of 0 is the CURRENT device's default stream) and raises what it reports."""
    if device.index == torch.cuda.current_device():
        status = status_of()
    else:
        with torch.cuda.device(device):
            status = status_of()
    if status != 0:
        raise RuntimeError("block operator failed with '%s' (0x%X)" % (native.error_message(status), status))


def _empty(rows, cols, block_rows, device):
    values = torch.empty((rows, _up(cols, BLOCK)), dtype=E4M3, device=device)
    scale = torch.empty((-(-rows // block_rows), _up(-(-cols // BLOCK), 4)), dtype=torch.uint8, device=device)
    return BlockTensor(values, scale, cols, block_rows)


def quantize_blocks(x, block_rows=1):
    """x [rows][cols] float32 / float16 / bfloat16 -> BlockTensor in blocks of block_rows (1: activations, 128: weights) x 128."""
    _plain(x, "x")
    if block_rows not in (1, BLOCK):
        raise ValueError("blocks have 1 or 128 rows, got %r" % (block_rows,))
    rows, cols = x.shape
    if cols < 1:
        raise ValueError("x: at least one column is wanted")
    b = _empty(rows, cols, block_rows, x.device)
    L = native.lib()
    _call(x.device, lambda: L.STTX_QuantizeBlocks(x.data_ptr(), _TYPES[x.dtype], rows, cols, x.stride(0), block_rows, b.values.data_ptr(), b.values.stride(0),
                                                  b.scale.data_ptr(), b.scale.stride(0), torch.cuda.current_stream(x.device).cuda_stream))
    return b


def dequantize_blocks(b, dtype=torch.float32):
    """BlockTensor -> [rows][cols] of `dtype` (float32, float16, bfloat16), one rounding."""
    _blocks(b, "b")
    if dtype not in _TYPES or dtype is E4M3:
        raise ValueError("dtype: float32, float16 or bfloat16 is wanted, got %s" % (dtype,))
    rows, cols = b.shape
    y = torch.empty((rows, cols), dtype=dtype, device=b.values.device)
    L = native.lib()
    _call(y.device, lambda: L.STTX_DequantizeBlocks(b.values.data_ptr(), b.values.stride(0), b.scale.data_ptr(), b.scale.stride(0), rows, cols, b.block_rows, y.data_ptr(),
                                                    _TYPES[dtype], y.stride(0), torch.cuda.current_stream(y.device).cuda_stream))
    return y


def dense_blocks(x, w, bias=None, relu_clip=None, dtype=torch.float16):
    """A dense layer: x . w^T + bias, with the clipped ReLU min(max(y, 0), relu_clip) if one is given.

    x: [rows][in] float32 / float16 / bfloat16 (quantised within the call) or a BlockTensor in blocks of 1 x 128; w: BlockTensor [out][in] in blocks of
    128 x 128; bias: float32 [out].  Returns [rows][out] of `dtype`, or for dtype float8_e4m3fn a BlockTensor in blocks of 1 x 128."""
    _blocks(w, "w", BLOCK)
    out, inner = w.shape
    if out < 1:
        raise ValueError("w: at least one row is wanted")
    device = w.values.device
    a = native.DenseBlocksArgs()
    if isinstance(x, BlockTensor):
        _blocks(x, "x", 1)
        a.x, a.x_scale, a.x_type = x.values.data_ptr(), x.scale.data_ptr(), 3
        a.x_ld, a.x_scale_ld = x.values.stride(0), x.scale.stride(0)
        at = x.values.device
    else:
        _plain(x, "x")
        a.x, a.x_type, a.x_ld = x.data_ptr(), _TYPES[x.dtype], x.stride(0)
        at = x.device
    rows = x.shape[0]
    if x.shape[1] != inner:
        raise ValueError("x has %d columns, w has %d" % (x.shape[1], inner))
    if at != device:
        raise ValueError("x is on %s, w on %s" % (at, device))
    if bias is not None:
        if bias.dtype is not torch.float32 or bias.dim() != 1 or bias.shape[0] != out or (bias.stride(0) != 1 and out > 1) or bias.device != device:
            raise ValueError("bias: a contiguous float32 vector of %d on %s is wanted, got %s %s on %s" % (out, device, bias.dtype, tuple(bias.shape), bias.device))
        a.bias = bias.data_ptr()
    if relu_clip is not None:
        if not relu_clip > 0.0:
            raise ValueError("relu_clip: a positive number or None is wanted, got %r" % (relu_clip,))
        a.relu_clip = relu_clip
    if dtype not in _TYPES:
        raise ValueError("dtype: float32, float16, bfloat16 or float8_e4m3fn is wanted, got %s" % (dtype,))
    if dtype is E4M3:
        y = _empty(rows, out, 1, device)
        a.y, a.y_ld, a.y_scale, a.y_scale_ld = y.values.data_ptr(), y.values.stride(0), y.scale.data_ptr(), y.scale.stride(0)
    else:
        y = torch.empty((rows, out), dtype=dtype, device=device)
        a.y, a.y_ld = y.data_ptr(), out
    a.y_type = _TYPES[dtype]
    a.w, a.w_ld, a.w_scale, a.w_scale_ld = w.values.data_ptr(), w.values.stride(0), w.scale.data_ptr(), w.scale.stride(0)
    a.rows, a.inner, a.out = rows, inner, out
    L = native.lib()
    need = L.STTX_DenseBlocksWorkspace(a.x_type, rows, inner)
    if need:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)     # torch's allocator: this stream's, or the capturing graph's own
        a.workspace, a.workspace_bytes = workspace.data_ptr(), need
    a.stream = torch.cuda.current_stream(device).cuda_stream
    _call(device, lambda: L.STTX_DenseBlocks(C.byref(a)))
    return y
