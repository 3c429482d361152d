"""Products in 8-bit integers with a scale per token and one per output channel.

``Int8QTensor`` keeps a matrix of 8-bit codes with a scale per row in HBM, in
the layout that the products read: weights (rows = output channels) and
quantized activations (rows = tokens) alike.  ``int8_gemm`` multiplies tokens,
quantized in the call or by ``quantize_tokens`` before it, by such weights:

    y[t, n] = s_x[t] * s_w[n] * sum_k q_x[t, k] * q_w[n, k]  (+ bias[n])

The sums are exact 32-bit integers.  Weights of GGUF types stay with
``tensor.QTensor``, 4-bit group weights with ``group4``.
"""
from __future__ import annotations

import torch

from . import _lib
from .tensor import _as_f32_dev, _dev, _ELEM, _elem, _gpu_tensor, _launch, _rows_meet, _rows_of, _workspace_bytes

__all__ = ["Int8QTensor", "quantize_tokens", "int8_gemm", "K_MAX"]

K_MAX = 131071  # sums of products stay within 32 bits

_PACKED = 3


class Int8QTensor:
    """A matrix (rows x k) of 8-bit codes with a scale per row, resident on one GPU."""

    def __init__(self, data: torch.Tensor, rows: int, k: int):
        if not isinstance(data, torch.Tensor) or data.dtype != torch.uint8 or data.device.type != "cuda":
            raise ValueError("Int8QTensor data must be a cuda uint8 tensor")
        nbytes = _lib.load().vb_int8_bytes(rows, k)
        if nbytes < 0 or data.numel() != nbytes or not data.is_contiguous():
            raise ValueError(f"Int8QTensor: {data.numel()} bytes, {nbytes} expected for {rows} x {k}")
        self.data = data
        self.rows, self.k = int(rows), int(k)

    @property
    def shape(self) -> tuple:
        return (self.rows, self.k)

    @property
    def nbytes(self) -> int:
        return self.data.numel()

    @property
    def device(self) -> torch.device:
        return self.data.device

    @property
    def scales(self) -> torch.Tensor:
        """The rows' scales, (rows,) float32: a view."""
        at = self.data.numel() - (self.rows + 15) // 16 * 64
        return self.data[at:].view(torch.float32)[:self.rows]

    def ptr(self) -> int:
        return self.data.data_ptr()

    def __repr__(self) -> str:
        return f"Int8QTensor(rows={self.rows}, k={self.k}, {self.device})"

    @classmethod
    def _empty(cls, rows: int, k: int, device) -> "Int8QTensor":
        nbytes = _lib.load().vb_int8_bytes(rows, k)
        if nbytes < 0:
            raise ValueError(f"Int8QTensor: no layout for {rows} x {k} (k at most {K_MAX})")
        return cls(torch.empty(nbytes, dtype=torch.uint8, device=device), rows, k)

    @classmethod
    def from_int8(cls, codes: torch.Tensor, scales: torch.Tensor) -> "Int8QTensor":
        """From device tensors: codes (rows, k) int8, scales (rows,) or (rows, 1) float32 / float16 / bfloat16.
        The parts are not kept."""
        dev = _gpu_tensor(codes, "Int8QTensor: codes")
        if codes.dim() != 2 or codes.dtype != torch.int8 or 0 in codes.shape:
            raise ValueError(f"Int8QTensor: codes must be (rows, k) int8, got {tuple(codes.shape)} {codes.dtype}")
        rows, k = codes.shape
        _elem(scales, "Int8QTensor: scales")
        if _gpu_tensor(scales, "Int8QTensor: scales") != dev or tuple(scales.shape) not in ((rows,), (rows, 1)):
            raise ValueError(f"Int8QTensor: scales must be ({rows},) or ({rows}, 1) on {dev}, got "
                             f"{tuple(scales.shape)} on {scales.device}")
        out = cls._empty(rows, k, dev)
        codes, scales = _rows_of(codes, k), scales.reshape(rows).to(torch.float32).contiguous()
        _launch(dev, "vb_int8_pack", codes.data_ptr(), codes.stride(0), scales.data_ptr(), out.ptr(), rows, k)
        return out

    @classmethod
    def quantize(cls, w, device=None) -> "Int8QTensor":
        """Quantize a (rows, k) matrix on the device, a scale per row (vb_int8_quantize): s = max |w| / 127, at least
        2^-126 (0 for a row of zeros), codes w / s to the nearest, ties to even.  A row that holds a NaN or an
        infinity gets the scale NaN."""
        if isinstance(w, torch.Tensor) and w.is_cuda and device is None:
            dev, src = w.device, w
        else:
            dev = _dev(device)
            src = _as_f32_dev(w, dev)
        kind = _elem(src, "Int8QTensor.quantize: w")
        if src.dim() != 2 or 0 in src.shape:
            raise ValueError(f"Int8QTensor.quantize expects a 2-D (rows, k) matrix, got {tuple(src.shape)}")
        rows, k = src.shape
        src = _rows_of(src, k)
        out = cls._empty(rows, k, dev)
        _launch(dev, "vb_int8_quantize", src.data_ptr(), kind, src.stride(0), rows, k, out.ptr())
        return out

    def dequantize(self) -> torch.Tensor:
        """codes * scale in fp32 (rows, k) (vb_int8_dequant_rows)."""
        out = torch.empty((self.rows, self.k), dtype=torch.float32, device=self.device)
        _launch(self.device, "vb_int8_dequant_rows", self.ptr(), out.data_ptr(), self.rows, self.k)
        return out


def quantize_tokens(x: torch.Tensor) -> Int8QTensor:
    """Activations (m, k) (or one token, (k,)) as 8-bit codes with a scale per token, for products that share them."""
    _gpu_tensor(x, "quantize_tokens: x")
    return Int8QTensor.quantize(x.reshape(1, -1) if x.dim() == 1 else x)


def int8_gemm(w: Int8QTensor, x, bias: torch.Tensor | None = None, out: torch.Tensor | None = None,
              out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Y = X W^T (+ bias) in 8-bit integers (vb_int8_gemm): x (m, k) -> (m, rows), or one token (k,) -> (rows,).

    x: float32 / float16 / bfloat16 on w's device, rows of any stride, quantized in the call as ``quantize_tokens``
    does; or its result, which several products may share.  bias: (rows,) float32.  The result is float32, or of
    ``out_dtype`` (or ``out``: contiguous, of the result's shape, apart from the operands).  Sums of products are
    exact; they are rounded to fp32, scaled, and the result is rounded once to its type.  A NaN or an infinity makes
    its own token's results NaN."""
    if not isinstance(w, Int8QTensor):  # (other weights hold fewer bytes than the products read)
        raise ValueError(f"int8_gemm: W must be an Int8QTensor, got {type(w).__name__}")
    packed = isinstance(x, Int8QTensor)
    dev = x.device if packed else _gpu_tensor(x, "int8_gemm: x")
    if dev != w.device:
        raise ValueError(f"int8_gemm: x is on {dev}, W on {w.device}")
    if packed:
        if x.k != w.k:
            raise ValueError(f"int8_gemm: x has k={x.k}, W has k={w.k}")
        m, kind, x_ptr, x_ld, shape = x.rows, _PACKED, x.ptr(), 0, (x.rows, w.rows)
    else:
        if x.dim() not in (1, 2) or x.shape[-1] != w.k:
            raise ValueError(f"int8_gemm: x must be ({w.k},) or (m, {w.k}), got {tuple(x.shape)}")
        kind = _elem(x, "int8_gemm: x")
        xr = _rows_of(x, w.k)
        m, x_ptr, x_ld = xr.shape[0], xr.data_ptr(), xr.stride(0)
        shape = (w.rows,) if x.dim() == 1 else (m, w.rows)
    if bias is not None:
        if _gpu_tensor(bias, "int8_gemm: bias") != dev or bias.dtype != torch.float32 or bias.numel() != w.rows:
            raise ValueError(f"int8_gemm: bias must be ({w.rows},) float32 on {dev}, got {tuple(bias.shape)} "
                             f"{bias.dtype} on {bias.device}")
        bias = bias.contiguous()
    if out is None:
        out = torch.empty(shape, dtype=torch.float32 if out_dtype is None else out_dtype, device=dev)
        y_type = _elem(out, "int8_gemm: out_dtype")
    else:
        if not isinstance(out, torch.Tensor) or out.device != dev or not out.is_contiguous() \
                or tuple(out.shape) != shape or out.dtype not in _ELEM or out_dtype not in (None, out.dtype):
            raise ValueError(f"int8_gemm: out must be a contiguous {shape} tensor on {dev}"
                             f"{'' if out_dtype is None else f' of {out_dtype}'}")
        y_type = _ELEM[out.dtype]
        first, nbytes = out.data_ptr(), out.numel() * out.element_size()
        for what, at, ld, width, count in (
                ("W", w.ptr(), 0, w.nbytes, 1),
                ("x", x_ptr, 0 if packed else x_ld * xr.element_size(), x.nbytes if packed else w.k * xr.element_size(),
                 1 if packed else m),
                ("bias", 0 if bias is None else bias.data_ptr(), 0, 4 * w.rows, 0 if bias is None else 1)):
            if nbytes and count and _rows_meet(first, 0, nbytes, 1, at, ld, width, count):
                raise ValueError(f"int8_gemm: out overlaps {what}, which is read until the call's end")
    nbytes = _workspace_bytes(dev, "vb_int8_workspace", m, w.rows, w.k, kind)
    ws = w.data.new_empty(nbytes) if nbytes > 0 else None
    _launch(dev, "vb_int8_gemm", w.ptr(), w.rows, w.k, x_ptr, kind, x_ld, m, None if bias is None else bias.data_ptr(),
            out.data_ptr(), y_type, None if ws is None else ws.data_ptr(), max(nbytes, 0))
    return out
