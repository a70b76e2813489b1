"""Norms before and after a block, with its gate, its scale and the residual stream (l2_block_norm of include/llama2_b200.h) on torch CUDA tensors."""
import ctypes as C
import struct

from . import paged
from ._lib import BlockNormArgs, check, lib

_call = lib.l2_block_norm
_ARGS = struct.Struct("@" + "Pqi0q" * 5 + "PPffii")  # l2_block_norm_args
assert _ARGS.size == C.sizeof(BlockNormArgs)
_NONE = (0, 0, 0)
_types = paged._types


def _rows(t, what, device, shape, one_for_all):
    """The fields of an l2_rows for t [rows, dim], or [dim] for all rows."""
    strides = t.stride()
    if t.shape != shape:
        if not one_for_all or t.shape != shape[1:]:
            raise ValueError("%s: [%d, %d] expected, got %s" % (what, *shape, tuple(t.shape)))
        strides = (0, *strides)
    if (strides[1] != 1 and shape[1] > 1) or t.get_device() != device:
        raise ValueError("%s: on device %d with its last dimension contiguous expected" % (what, device))
    return t.data_ptr(), strides[0], _types[t.dtype] if t.dtype in _types else paged._type(t)


def block_norm(block, residual=None, out=None, *, residual_out=None, post_weight=None, pre_weight=None, gate=None, scale=1.0, eps=1e-5, stream=None):
    """For rows [rows, dim] in f32, f16 or bf16, with norm(x) = x / sqrt(mean(x^2) + eps):

        t = norm(block) * post_weight               (without a post_weight: block)
        residual_out = residual + scale * gate * t  (gate: [rows, dim], or [dim] for all rows)
        out = norm(residual_out) * pre_weight

    in f32, rounded once.  The weights are f32 [dim].  block, residual and gate may be None (1 for a gate, else 0), and one of residual_out and out; residual_out may be
    residual, out may be block.  Enqueued on the current stream unless `stream` (a cudaStream_t) is given.  Returns (residual_out, out)."""
    first = block if block is not None else residual
    if first is None or first.dim() != 2:
        raise ValueError("block or residual: [rows, dim] expected")
    shape, device = first.shape, first.get_device()
    rows, dim = shape
    if rows >> 31 or dim >> 31:
        paged._int32(rows=rows, dim=dim)
    if device < 0:
        raise ValueError("tensors on a CUDA device expected")
    record = _ARGS.pack(
        *(_rows(block, "block", device, shape, False) if block is not None else _NONE),
        *(_rows(residual, "residual", device, shape, False) if residual is not None else _NONE),
        *(_rows(gate, "gate", device, shape, True) if gate is not None else _NONE),
        *(_rows(residual_out, "residual_out", device, shape, False) if residual_out is not None else _NONE),
        *(_rows(out, "out", device, shape, False) if out is not None else _NONE),
        paged._packed(post_weight, "post_weight", device, (dim,), paged.F32) if post_weight is not None else 0,
        paged._packed(pre_weight, "pre_weight", device, (dim,), paged.F32) if pre_weight is not None else 0,
        scale, eps, rows, dim)
    rc = _call(record, paged._stream_on(device, stream))
    if rc:
        check(rc)
    return residual_out, out
