"""Microscaled 4-bit floats (the OCP MXFP4 format): quantisation, its inverse
and the product of two such matrices, as HIP kernels (``nibble_mx_quantize``,
``nibble_mx_dequantize`` and ``nibble_mx_matmul`` of the C ABI).

The second 4-bit format of this package, beside the grouped INT4 weights of
:mod:`nibblegemm_amd.quant`: the one the matrix cores of gfx950 multiply as it
is, four times as fast as fp16, which pays where a product is bound by
arithmetic.  Both operands are 4-bit, so activations are quantised too.

Layout
------
A matrix is ``[rows, K]``, K a multiple of 32, and is quantised along K: an
activation ``X [M, K]`` as it is, a weight as ``[N, K]`` -- a ``torch.nn.Linear``
weight as it is, this package's dense ``[K, N]`` weights as ``W.t()``.  The 32
values of a block share one power of two,

    e = max(floor(log2(max|v|)) - 2, -127),

and each is stored as the 4-bit float (sign, two exponent bits, one mantissa
bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6) nearest to ``v / 2^e``, ties to the even code,
values beyond 6 as 6.  A block that holds an infinity or a NaN is stored as
NaN.  ``codes`` is uint8 ``[rows, K / 2]``, the even k in the low half of a
byte; ``scales`` is uint8 ``[ceil(K / 128), rows, 4]``: ``e + 127`` (255 is NaN)
of four neighbouring blocks to a word, the words of one k group side by side,
as the kernels load them; it is zero behind the last block.
:func:`mx_from_blocks` makes one from scales ``[rows, K / 32]``, the order of
other tools.

No operator here has a backward: a call whose inputs autograd follows raises.
"""
from __future__ import annotations

import dataclasses
from dataclasses import dataclass
from typing import Optional, Union

import torch

from . import _native
from .ops import _call, _check_no_backward, _stream, _workspace

#: Values that share a scale, and blocks whose scales share a word.
MX_BLOCK = 32
MX_GROUP = 128

#: The values of the 16 codes.
MX_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)

#: Bytes of quantised activations that a stream's calls keep between them; a
#: larger x gets a buffer of its own.
_KEPT_BYTES = 16 << 20

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


@dataclass(frozen=True)
class MXMatrix:
    """One microscaled ``[rows, K]`` matrix (the module's docstring has the
    layout)."""

    codes: torch.Tensor  # uint8 [rows, K // 2]
    scales: torch.Tensor  # uint8 [ceil(K / 128), rows, 4]
    rows: int
    K: int

    def to(self, device) -> "MXMatrix":
        """The same matrix with both tensors moved to ``device``."""
        return dataclasses.replace(self, codes=self.codes.to(device), scales=self.scales.to(device))

    @property
    def nbytes(self) -> int:
        """Bytes a product must read for this matrix: codes and scales."""
        return self.codes.numel() + self.scales.numel()

    def block_scales(self) -> torch.Tensor:
        """The biased exponents as ``[rows, K / 32]`` (a copy)."""
        flat = self.scales.transpose(0, 1).reshape(self.rows, -1)
        return flat[:, :self.K // MX_BLOCK].contiguous()


def _groups(K: int) -> int:
    return -(-K // MX_GROUP)


def _check_k(K: int) -> None:
    if K % MX_BLOCK:
        raise ValueError(f"K={K} must be divisible by {MX_BLOCK}")


def _check_mx(name: str, m: MXMatrix) -> None:
    _check_k(m.K)
    codes, scales = m.codes, m.scales
    if (codes.dtype is torch.uint8 and scales.dtype is torch.uint8
            and codes.shape == (m.rows, m.K // 2) and scales.shape == (_groups(m.K), m.rows, 4)
            and codes.is_contiguous() and scales.is_contiguous()
            and codes.get_device() == scales.get_device()):
        return
    for what, t, shape in (("codes", m.codes, (m.rows, m.K // 2)),
                           ("scales", m.scales, (_groups(m.K), m.rows, 4))):
        if t.dtype != torch.uint8:
            raise RuntimeError(f"{name}: {what} must be uint8, got {t.dtype}")
        if tuple(t.shape) != shape:
            raise ValueError(f"{name}: {what} must be {list(shape)}, got {list(t.shape)}")
        if not t.is_contiguous():
            raise RuntimeError(f"{name}: {what} must be contiguous")
    if m.codes.device != m.scales.device:
        raise RuntimeError(f"{name}: codes and scales must live on the same device")


def _check_values(name: str, x: torch.Tensor) -> None:
    if x.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got shape {tuple(x.shape)}")
    if x.dtype not in _DTYPES:
        raise RuntimeError(f"{name} must be fp16, bf16 or fp32, got {x.dtype}")
    _check_no_backward(name, x)
    _check_k(x.shape[1])


def mx_from_blocks(codes: torch.Tensor, scales: torch.Tensor) -> MXMatrix:
    """A matrix from ``codes`` uint8 ``[rows, K / 2]`` and one biased exponent a
    block, ``scales`` uint8 ``[rows, K / 32]``, on their device."""
    if codes.dim() != 2 or scales.dim() != 2 or codes.shape[0] != scales.shape[0] or \
            codes.shape[1] != scales.shape[1] * (MX_BLOCK // 2):
        raise ValueError(f"expected codes [rows, K / 2] and scales [rows, K / {MX_BLOCK}], got "
                         f"{tuple(codes.shape)} and {tuple(scales.shape)}")
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise RuntimeError(f"codes and scales must be uint8, got {codes.dtype} and {scales.dtype}")
    rows, blocks = scales.shape
    words = _groups(blocks * MX_BLOCK)
    padded = torch.zeros((rows, words * 4), dtype=torch.uint8, device=scales.device)
    padded[:, :blocks] = scales
    return MXMatrix(codes.contiguous(), padded.view(rows, words, 4).transpose(0, 1).contiguous(),
                    rows, blocks * MX_BLOCK)


def quantize_mx(x: torch.Tensor) -> MXMatrix:
    """``x`` ``[rows, K]`` (fp16, bf16 or fp32) quantised along K, on its device.
    On a GPU one kernel reads ``x`` once, whether the k or (a transposed view)
    the rows are adjacent in memory; other strides are copied first.  Elsewhere
    the same arithmetic runs as tensor operations."""
    _check_values("x", x)
    rows, K = x.shape
    if not x.is_cuda:
        return _quantize_ops(x)
    if x.is_neg():  # a view whose values are its memory's, negated
        x = x.resolve_neg()
    row_stride, k_stride = x.stride()
    if rows == 1 and k_stride == 1:  # (whatever a single row's stride is)
        row_stride = K
    if not (row_stride == 1 and k_stride > 1 or k_stride == 1 and row_stride > 0):
        x = x.contiguous()
        row_stride, k_stride = x.stride()
    ext = _native.binding()
    codes = torch.empty((rows, K // 2), dtype=torch.uint8, device=x.device)
    scales = torch.empty((_groups(K), rows, 4), dtype=torch.uint8, device=x.device)
    _call(ext.mx_quantize, x.device, x.data_ptr(), rows, K, row_stride, k_stride,
            _DTYPES[x.dtype], codes.data_ptr(), scales.data_ptr())
    return MXMatrix(codes, scales, rows, K)


def _quantize_ops(x: torch.Tensor) -> MXMatrix:
    """:func:`quantize_mx` as tensor operations on x's device."""
    rows, K = x.shape
    v = x.detach().double().reshape(rows, K // MX_BLOCK, MX_BLOCK)
    top = v.abs().amax(-1)
    finite = torch.isfinite(top)
    _, ex = torch.frexp(torch.where(finite & (top > 0), top, 2.0 ** -125))  # f 2^ex, f in [1/2, 1)
    e = (ex - 3).clamp(min=-127)
    u = torch.where(finite[..., None], v * torch.exp2(-e.double())[..., None], 0.0)
    a = u.abs()
    half = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))  # distance of the neighbours
    a = (torch.round(a / half) * half).clamp(max=6.0)
    code = torch.bucketize(a, torch.tensor(MX_VALUES[1:8], dtype=torch.float64, device=x.device),
                           right=True)
    code = (code + 8 * torch.signbit(u)).to(torch.uint8).reshape(rows, K)
    biased = torch.where(finite, e + 127, 255).to(torch.uint8)
    return mx_from_blocks(code[:, 0::2] | code[:, 1::2] << 4, biased)


def dequantize_mx(m: MXMatrix, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The ``[rows, K]`` values ``m`` stands for, on its device: exact in bf16 and
    fp32 (what those types cannot hold becomes infinite), rounded once in fp16.
    Elsewhere than on a GPU the same values from tensor operations."""
    _check_mx("m", m)
    if dtype not in _DTYPES:
        raise RuntimeError(f"dtype must be fp16, bf16 or fp32, got {dtype}")
    dev = m.codes.device
    if not m.codes.is_cuda:
        pairs = torch.stack([m.codes & 15, m.codes >> 4], -1).reshape(m.rows, m.K)
        v = torch.tensor(MX_VALUES, dtype=torch.float64)[pairs.long()]
        e = m.block_scales().repeat_interleave(MX_BLOCK, 1)
        v = v * torch.exp2(e.double() - 127)
        return torch.where(e == 255, float("nan"), v).float().to(dtype)
    ext = _native.binding()
    out = torch.empty((m.rows, m.K), dtype=dtype, device=dev)
    _call(ext.mx_dequantize, dev, m.codes.data_ptr(), m.scales.data_ptr(), m.rows, m.K,
            _DTYPES[dtype], out.data_ptr())
    return out


def matmul_mx(x: Union[torch.Tensor, MXMatrix], w: MXMatrix,
              out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``x w^T`` ``[M, N]`` of ``x`` ``[M, K]`` and the weight ``w`` ``[N, K]``:
    the products of the 4-bit values summed in fp32 and rounded once to
    ``out_dtype`` (fp16, bf16 or fp32).  A dense ``x`` (fp16, bf16 or fp32) is
    quantised first, with :func:`quantize_mx`'s values, and gives its own dtype
    by default; an :class:`MXMatrix` fp16.  A NaN block makes the outputs of its
    row of ``x`` or of ``w`` NaN."""
    _check_mx("w", w)
    if not w.codes.is_cuda:
        raise RuntimeError("all tensors must live on the GPU")
    dense = isinstance(x, torch.Tensor)
    if dense:
        _check_values("x", x)
        M, K = x.shape
    else:
        _check_mx("x", x)
        M, K = x.rows, x.K
    if (x if dense else x.codes).get_device() != w.codes.get_device():
        raise RuntimeError("all tensors must live on the same device")
    dev = w.codes.device
    if K != w.K:
        raise RuntimeError(f"x has K={K}, the weight K={w.K}")
    if out_dtype is None:
        out_dtype = x.dtype if dense else torch.float16
    if out_dtype not in _DTYPES:
        raise RuntimeError(f"out_dtype must be fp16, bf16 or fp32, got {out_dtype}")
    ext = _native.binding()
    N = w.rows
    y = torch.empty((M, N), dtype=out_dtype, device=dev)
    if dense and (x.stride(1) != 1 or x.is_neg() or (M > 1 and x.stride(0) < 1)):
        x, dense = quantize_mx(x), False
    if dense:
        need = ext.mx_matmul_dense_workspace_bytes(M, N, K, M <= 16 and _rows_on_16_bytes(x))
        if need <= _KEPT_BYTES:
            ws, ws_bytes = _workspace((need, -1), dev, _stream(dev))
        else:
            ws, ws_bytes = torch.empty(need, dtype=torch.uint8, device=dev), need
        _call(ext.mx_matmul_dense, dev, x.data_ptr(), M, x.stride(0) if M > 1 else K,
              _DTYPES[x.dtype], w.codes.data_ptr(), w.scales.data_ptr(), N, K, _DTYPES[out_dtype],
              y.data_ptr(), ws.data_ptr() if ws is not None else None, ws_bytes)
        return y
    _call(ext.mx_matmul, dev, x.codes.data_ptr(), x.scales.data_ptr(), M, w.codes.data_ptr(),
          w.scales.data_ptr(), N, K, _DTYPES[out_dtype], y.data_ptr())
    return y


def _rows_on_16_bytes(x: torch.Tensor) -> bool:
    """Whether a kernel may read the rows of ``x`` in pieces of 16 bytes."""
    size = x.element_size()
    return (x.data_ptr() % 16 == 0 and (x.shape[0] == 1 or x.stride(0) * size % 16 == 0)
            and ((x.shape[0] - 1) * x.stride(0) + x.shape[1]) * size < 1 << 31)


__all__ = ["MX_BLOCK", "MX_GROUP", "MX_VALUES", "MXMatrix", "dequantize_mx", "matmul_mx",
           "mx_from_blocks", "quantize_mx"]
