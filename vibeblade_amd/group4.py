"""4-bit weights with one scale (and zero point) per group of a row.

``W[n, k] = (q[n, k] - z[n, g]) * s[n, g]`` with ``g = k // group``: the form in
which post-training quantizers other than GGUF's leave their weights (codes,
fp16 scales and zero points in tensors of their own).  ``GroupQTensor`` keeps
such a matrix in HBM in the layout that the products read; ``group_gemv``
multiplies one or a few tokens by it.  The K-quants of ``ggml`` stay with
``QTensor``.
"""
from __future__ import annotations

import torch

from . import _lib
from .tensor import (_as_f32_dev, _check_out, _dev, _elem, _gpu_tensor, _launch, _rows_meet, _rows_of,
                     _workspace_bytes)

__all__ = ["GroupQTensor", "group_gemv"]


def _groups(k: int, group: int) -> int:
    if group not in (32, 64) and (group <= 0 or group % 128 or group >= 1 << 31):
        raise ValueError(f"group must be 32, 64 or a multiple of 128 below 2^31, got {group}")
    return -(-k // group)


class GroupQTensor:
    """A 4-bit weight matrix (rows outputs x k inputs) with group scales, resident on one GPU."""

    def __init__(self, data: torch.Tensor, rows: int, k: int, group: int, zeros: bool):
        _groups(k, group)
        if not isinstance(data, torch.Tensor) or data.dtype != torch.uint8 or data.device.type != "cuda":
            raise ValueError("GroupQTensor data must be a cuda uint8 tensor")
        nbytes = _lib.load().vb_group4_bytes(rows, k, group, int(zeros))
        if nbytes < 0 or data.numel() != nbytes or not data.is_contiguous():
            raise ValueError(f"GroupQTensor: {data.numel()} bytes, {nbytes} expected for {rows} x {k} in groups of {group}")
        self.data = data
        self.rows, self.k, self.group, self.zeros = int(rows), int(k), int(group), bool(zeros)

    @property
    def shape(self) -> tuple:
        return (self.rows, self.k)

    @property
    def nbytes(self) -> int:
        return self.data.numel()

    @property
    def device(self) -> torch.device:
        return self.data.device

    def ptr(self) -> int:
        return self.data.data_ptr()

    def __repr__(self) -> str:
        return (f"GroupQTensor(rows={self.rows}, k={self.k}, group={self.group}, "
                f"{'zero points' if self.zeros else 'symmetric'}, {self.device})")

    @classmethod
    def from_packed(cls, packed: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, *, k: int,
                    group: int = 128) -> "GroupQTensor":
        """From device tensors: packed (rows, ceil(k / 2)) uint8 with code 2i of a row in the low half of its byte
        i (``quant.pack_nibbles`` order), scales (rows, ceil(k / group)) float16, zeros of that shape, uint8 in
        0..15 (None: 8 everywhere; the check of these values waits for the device).  The parts are not kept."""
        dev = _gpu_tensor(packed, "GroupQTensor: packed")
        k, group = int(k), int(group)
        if packed.dim() != 2 or packed.dtype != torch.uint8 or packed.shape[0] == 0 or k <= 0 \
                or packed.shape[1] != (k + 1) // 2:
            raise ValueError(f"GroupQTensor: packed must be (rows, {(k + 1) // 2}) uint8 for k={k}, got "
                             f"{tuple(packed.shape)} {packed.dtype}")
        rows = packed.shape[0]
        want = (rows, _groups(k, group))
        for t, name, dtype in ((scales, "scales", torch.float16), (zeros, "zeros", torch.uint8)):
            if t is None and name == "zeros":
                continue
            if _gpu_tensor(t, f"GroupQTensor: {name}") != dev or t.dtype != dtype or tuple(t.shape) != want:
                raise ValueError(f"GroupQTensor: {name} must be {want} {dtype} on {dev}, got {tuple(t.shape)} "
                                 f"{t.dtype} on {t.device}")
        if zeros is not None and bool((zeros > 15).any()):
            raise ValueError("GroupQTensor: zero points must be 0 to 15")
        return cls._pack(packed, scales, zeros, k, group)

    @classmethod
    def _pack(cls, packed, scales, zeros, k: int, group: int) -> "GroupQTensor":
        rows, dev = packed.shape[0], packed.device
        packed, scales = packed.contiguous(), scales.contiguous()
        zeros = None if zeros is None else zeros.contiguous()
        nbytes = _lib.load().vb_group4_bytes(rows, k, group, int(zeros is not None))
        if nbytes < 0:
            raise ValueError(f"GroupQTensor: no layout for {rows} x {k} in groups of {group}")
        data = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        _launch(dev, "vb_group4_pack", packed.data_ptr(), scales.data_ptr(), None if zeros is None else zeros.data_ptr(),
                data.data_ptr(), rows, k, group)
        return cls(data, rows, k, group, zeros is not None)

    @classmethod
    def quantize(cls, w, group: int = 128, zeros: bool = True, device=None) -> "GroupQTensor":
        """Quantize a (rows, k) matrix on the device (vb_group4_quantize).  A group that holds a NaN or an infinity
        becomes NaN."""
        if isinstance(w, torch.Tensor) and w.is_cuda and device is None:
            dev, src = w.device, w
            _elem(src, "GroupQTensor.quantize: w")
        else:
            dev = _dev(device)
            src = _as_f32_dev(w, dev)
        if src.dim() != 2 or 0 in src.shape:
            raise ValueError(f"GroupQTensor.quantize expects a 2-D (rows, k) matrix, got {tuple(src.shape)}")
        rows, k = src.shape
        src = _rows_of(src, k)
        groups = _groups(k, int(group))
        packed = torch.empty((rows, (k + 1) // 2), dtype=torch.uint8, device=dev)
        scales = torch.empty((rows, groups), dtype=torch.float16, device=dev)
        z = torch.empty((rows, groups), dtype=torch.uint8, device=dev) if zeros else None
        _launch(dev, "vb_group4_quantize", src.data_ptr(), _elem(src, "GroupQTensor.quantize: w"), src.stride(0), rows, k,
                int(group), packed.data_ptr(), scales.data_ptr(), None if z is None else z.data_ptr())
        return cls._pack(packed, scales, z, k, int(group))

    def dequantize(self) -> torch.Tensor:
        """The weights in fp32 (rows, k), exact (vb_group4_dequant_rows)."""
        out = torch.empty((self.rows, self.k), dtype=torch.float32, device=self.device)
        _launch(self.device, "vb_group4_dequant_rows", self.ptr(), out.data_ptr(), self.rows, self.k, self.group,
                int(self.zeros))
        return out


def group_gemv(w: GroupQTensor, x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """y = W x for one activation vector (k,) -> (rows,) or a few of them (m, k) -> (m, rows), fp32
    (vb_group4_gemv).  x: float32, float16 or bfloat16 on w's device, rows of any stride.  out: contiguous
    float32, apart from x and w.

    Products with the codes are exact and summed in fp32 or wider, but of an activation much smaller than the
    largest of its 128 neighbours (blocks of 128 along k) the last bits are dropped: fp32 keeps all of them from
    2^-6 of that largest on and loses at most 2^-30 of it below; 16-bit types from 2^-14 (bfloat16) or 2^-11
    (float16) on and at most 2^-22; with more than a few tokens float16 goes in as it is and bfloat16 loses at most
    2^-38.  Which of the two forms 16-bit tokens take, and in which order groups are summed, depends on their number
    and the number of rows: the same token in another batch may differ in its last bits.  The same call gives the
    same bits.  A NaN or an infinity makes its own token's results NaN or infinite."""
    dev = _gpu_tensor(x, "group_gemv: x")
    if dev != w.device:
        raise ValueError(f"group_gemv: x is on {dev}, W on {w.device}")
    if x.dim() not in (1, 2) or x.shape[-1] != w.k:
        raise ValueError(f"group_gemv: x must be ({w.k},) or (m, {w.k}), got {tuple(x.shape)}")
    kind = _elem(x, "group_gemv: x")
    xr = _rows_of(x, w.k)
    m = xr.shape[0]
    if out is None:
        out = x.new_empty((w.rows,) if x.dim() == 1 else (m, w.rows), dtype=torch.float32)
    else:
        _check_out(out, m * w.rows, dev, "group_gemv")
        each = xr.element_size()
        if _rows_meet(out.data_ptr(), 0, out.numel() * 4, 1, xr.data_ptr(), xr.stride(0) * each, w.k * each, m):
            raise ValueError("group_gemv: out overlaps x, which is read until the call's end")
        if m > 0 and w.ptr() - out.numel() * 4 < out.data_ptr() < w.ptr() + w.nbytes:
            raise ValueError("group_gemv: out overlaps the weights")
    nbytes = _workspace_bytes(dev, "vb_group4_workspace", m, w.rows, w.k, w.group, int(w.zeros), kind)
    ws = w.data.new_empty(nbytes) if nbytes > 0 else None
    _launch(dev, "vb_group4_gemv", w.ptr(), w.rows, w.k, w.group, int(w.zeros), xr.data_ptr(), kind, xr.stride(0), m,
            out.data_ptr(), None if ws is None else ws.data_ptr(), nbytes)
    return out
