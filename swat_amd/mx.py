"""Microscaled matrices: blocks of 32 columns of a row share a power of two, elements are e4m3 (8 bits) or e2m1 (4 bits).

8 bits are the checkpoint form of activations — a linear layer's input, an MLP's pre-activation — that the backward pass reads as
they are (linear_wgrad, act_bwd); 4 bits halve that again for weights of frozen towers and large collections of rows; matmul
multiplies any two of them without unpacking.  Thin wrappers over the C ABI (include/swat_hip.h) on torch's current stream; no
PyTorch fallback.
"""
import functools
from collections import namedtuple

import torch

from . import _lib
from .ops import ACT

_BF, _F32, _U8 = torch.bfloat16, torch.float32, torch.uint8
_COLS = 1 << 24  # columns of a matrix at most (the C entries take them as 32-bit numbers)


class MX(namedtuple("MX", "codes scale cols bits")):
    """A packed [rows, cols] matrix: codes uint8 [rows, ceil(cols / 32) * 32 * bits / 8] (4 bits: the even column in the low half, zeros
    behind the last column), scale uint8 [rows, ceil(cols / 32)] (exponent + 127; 255: the block is NaN).  Packing takes the smallest power
    of two that keeps a block within the format (other software may take the largest element's and cut off what is past the end) and
    writes bytes of 17 or more; in a matrix put together by hand, values under smaller bytes are rounded where they become bf16."""
    __slots__ = ()

    @property
    def rows(self):
        return self.codes.shape[0]

    @property
    def shape(self):
        return (self.codes.shape[0], self.cols)


def _empty(like, rows, cols, bits):
    blocks = (cols + 31) // 32
    return MX(like.new_empty((rows, blocks * 4 * bits), dtype=_U8), like.new_empty((rows, blocks), dtype=_U8), cols, bits)


def _check(m, what, bits=(4, 8)):
    """The pointers of an MX matrix whose parts fit together, on the current device."""
    if not isinstance(m, MX) or m.bits not in bits or not isinstance(m.cols, int) or not 1 <= m.cols <= _COLS:
        raise _lib.SwatHipError(f"{what}: an MX matrix of {' or '.join(map(str, bits))} bits and 1 to {_COLS} columns is wanted, got {m!r:.80}")
    codes, scale, cols, nbits = m
    if not isinstance(codes, torch.Tensor) or not isinstance(scale, torch.Tensor) or codes.dim() != 2:
        raise _lib.SwatHipError(f"{what}: codes {codes!r:.60} and scale {scale!r:.60} are not the parts of an MX matrix")
    rows, blocks, device = codes.shape[0], (cols + 31) // 32, codes.get_device()
    if (device < 0 or device != scale.get_device() or device != _lib._current() or codes.dtype != _U8 or scale.dtype != _U8
            or codes.shape != (rows, blocks * 4 * nbits) or scale.shape != (rows, blocks)
            or not codes.is_contiguous() or not scale.is_contiguous()):
        raise _lib.SwatHipError(f"{what}: codes {tuple(codes.shape)} {codes.dtype} on {codes.device}, scale {tuple(scale.shape)} {scale.dtype} on "
                                f"{scale.device} are not the contiguous parts of {m.cols} columns in {m.bits} bits on the current device "
                                "(no CPU fallback)")
    return codes.data_ptr(), scale.data_ptr()


def _act(act, what):
    if not isinstance(act, str) or ACT.get(act, 0) == 0:
        raise _lib.SwatHipError(f"{what}: activation {act!r} ('gelu' or 'quick_gelu')")
    return ACT[act]


def quantize(x, bits=8):
    """x [rows, cols] bf16 or fp32 (rows may be strided) -> MX."""
    px, ld = _lib.rows_ptr(x, "mx.quantize", (_BF, _F32))
    if bits not in (4, 8) or not 1 <= x.shape[1] <= _COLS:
        raise _lib.SwatHipError(f"mx.quantize: {bits} bits (4 or 8) of {x.shape[1]} columns (1 to {_COLS})")
    m = _empty(x, x.shape[0], x.shape[1], bits)
    _lib.check(_lib.lib().swat_mx_quantize(px, ld, x.dtype == _BF, bits, m.codes.data_ptr(), m.scale.data_ptr(), x.shape[0], x.shape[1],
                                           _lib.stream()), "swat_mx_quantize")
    return m


def dequantize(m, dtype=_BF):
    """The values an MX matrix stands for, [rows, cols] in bf16 or fp32 (exact in both; in bf16 from scale byte 17 on)."""
    codes, scale = _check(m, "mx.dequantize")
    if dtype not in (_BF, _F32):
        raise _lib.SwatHipError(f"mx.dequantize: {dtype} (bfloat16 or float32)")
    out = m.codes.new_empty(m.shape, dtype=dtype)
    _lib.check(_lib.lib().swat_mx_dequantize(codes, scale, m.bits, out.data_ptr(), dtype == _BF, m.rows, m.cols, _lib.stream()),
               "swat_mx_dequantize")
    return out


def act_fwd(f, act="gelu"):
    """f bf16 [rows, n] -> (act(f) bf16, the 8-bit checkpoint of f), f read once."""
    pf, ld = _lib.rows_ptr(f, "mx.act_fwd", (_BF,))
    a = _act(act, "mx.act_fwd")
    if not 1 <= f.shape[1] <= _COLS:
        raise _lib.SwatHipError(f"mx.act_fwd: {f.shape[1]} columns (1 to {_COLS})")
    m = _empty(f, f.shape[0], f.shape[1], 8)
    g = f.new_empty(f.shape)
    _lib.check(_lib.lib().swat_mx_act_fwd(pf, ld, a, g.data_ptr(), m.codes.data_ptr(), m.scale.data_ptr(), f.shape[0], f.shape[1],
                                          _lib.stream()), "swat_mx_act_fwd")
    return g, m


def act_bwd(dg, m, act="gelu", want_act=True):
    """dg bf16 [rows, n] and the checkpoint of f -> (df = dg act'(f8) bf16, act(f8) bf16 or None)."""
    codes, scale = _check(m, "mx.act_bwd", (8,))
    pg, ld = _lib.rows_ptr(dg, "mx.act_bwd: dg", (_BF,), m.cols)
    a = _act(act, "mx.act_bwd")
    if dg.shape[0] != m.rows:
        raise _lib.SwatHipError(f"mx.act_bwd: {dg.shape[0]} rows of dg, {m.rows} of the checkpoint")
    df = dg.new_empty(m.shape)
    g = dg.new_empty(m.shape) if want_act else None
    _lib.check(_lib.lib().swat_mx_act_bwd(pg, ld, codes, scale, a, df.data_ptr(), g.data_ptr() if want_act else None, m.rows, m.cols,
                                          _lib.stream()), "swat_mx_act_bwd")
    return df, g


@functools.lru_cache(maxsize=256)
def _wgrad_workspace(rows, n, cols):
    return _lib.lib().swat_mx_linear_wgrad_workspace_bytes(rows, n, cols)


def linear_wgrad(dy, m, want_bias=False, out=None):
    """Weight gradient from the 8-bit checkpoint of a linear layer's input: dy bf16 [rows, n] -> dW fp32 [n, cols] (, column sums of dy)."""
    codes, scale = _check(m, "mx.linear_wgrad", (8,))
    py, ld = _lib.rows_ptr(dy, "mx.linear_wgrad: dy", (_BF,))
    rows, n = dy.shape
    if rows != m.rows or n > _COLS:
        raise _lib.SwatHipError(f"mx.linear_wgrad: {rows} rows of {n} columns of dy, {m.rows} rows of the checkpoint")
    if out is None:
        out = dy.new_empty((n, m.cols), dtype=_F32)
    pw = _lib.vec_ptr(out, "mx.linear_wgrad: out", n, m.cols)
    db = dy.new_empty(n, dtype=_F32) if want_bias else None
    nbytes = _wgrad_workspace(rows, n, m.cols)
    ws = dy.new_empty(nbytes, dtype=_U8) if nbytes > 0 else None
    _lib.check(_lib.lib().swat_mx_linear_wgrad(py, ld, codes, scale, pw, db.data_ptr() if want_bias else None, rows, n, m.cols,
                                      ws.data_ptr() if nbytes > 0 else None, nbytes, _lib.stream()), "swat_mx_linear_wgrad")
    return (out, db) if want_bias else out


def matmul(a, b, bias=None, out_dtype=_BF):
    """a [M, K] @ b [N, K].T (+ bias fp32 [N]) -> [M, N]; 4 or 8 bits each, nothing is unpacked.  bf16, or fp32 where both have 4 bits
    (with an 8-bit operand the matrix instruction keeps 13 binary places below the largest of eight neighbouring products: beside plain
    32-bit sums, 0.7 % of the results are the next bfloat16 number or, where a sum cancels, off by 2^-13 of its terms).  Sums in 32 bits
    with 8-bit operands: ops.linear_fwd on dequantize(a), dequantize(b), which are exact (K a multiple of 8, N of 4)."""
    ca, sa = _check(a, "mx.matmul: a")
    cb, sb = _check(b, "mx.matmul: b")
    if a.cols != b.cols or not (out_dtype == _BF or (out_dtype == _F32 and a.bits == b.bits == 4)):
        raise _lib.SwatHipError(f"mx.matmul: {a.shape} in {a.bits} bits by {b.shape} in {b.bits} bits (the same columns) into {out_dtype} "
                                "(bfloat16; float32 where both have 4 bits)")
    pb = _lib.vec_ptr(bias, "mx.matmul: bias", b.codes.shape[0])
    c = a.codes.new_empty((a.rows, b.rows), dtype=out_dtype)
    _lib.check(_lib.lib().swat_mx_matmul(ca, sa, a.bits, cb, sb, b.bits, pb, c.data_ptr(), out_dtype == _BF, a.rows, b.rows, a.cols, _lib.stream()),
               "swat_mx_matmul")
    return c
