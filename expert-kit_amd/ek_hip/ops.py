"""Operators beside a layer, over the C ABI: the RMS norm that adds the residual and quantises
(ek_norm), and one int8 matrix on 8-bit activations (ek_linear).

An 8-bit row is ``q`` (int8) with one fp32 ``scale`` and stands for ``q * scale``:
``q = rint(127 v / max|v|)``, ``scale = max|v| / 127``.  As in ``backend``, torch supplies buffers and
streams and all arithmetic happens inside libek_hip.so.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _capi as C
from .backend import _DT, _alloc_on, _desc, _mem, _stream_ptr


def _check_device(t: torch.Tensor, device_id: int) -> None:
    if t.is_cuda and t.device.index != device_id:
        raise C.EKError(C.EK_INVALID_INPUT, f"tensors are on {t.device}, the handle on device {device_id}")


def _addr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


class NormOut(NamedTuple):
    """What HipNorm.forward returns: x + residual, the normed rows, and their 8-bit form (None: not asked for)."""
    sum: Optional[torch.Tensor]
    y: Optional[torch.Tensor]
    q: Optional[torch.Tensor]
    scale: Optional[torch.Tensor]


class HipNorm:
    """RMS norm of the residual stream with a 16-bit and an 8-bit output (ek_norm)."""

    def __init__(self, gain: torch.Tensor, eps: float = 1e-6, device_id: int = 0):
        """gain [H], bf16 or fp16: the type of every 16-bit tensor of the calls."""
        if gain.dim() != 1 or gain.dtype not in (torch.bfloat16, torch.float16):
            raise C.EKError(C.EK_INVALID_INPUT, f"gain must be a bf16 or fp16 vector (got {tuple(gain.shape)} {gain.dtype})")
        self._lib = C.load()
        self._forward = self._lib.ek_norm_forward
        self.hidden, self.dtype, self.device_id = gain.numel(), gain.dtype, device_id
        _check_device(gain, device_id)
        gain = gain.contiguous()
        cfg = C.ek_norm_cfg(hidden=self.hidden, act_dtype=_DT[gain.dtype], eps=eps, device_id=device_id, flags=0)
        self._h = ctypes.c_void_p()
        C.check(self._lib.ek_norm_create(ctypes.byref(cfg), gain.data_ptr(), _mem(gain), ctypes.byref(self._h)))

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None, norm: bool = True, quantize: bool = True,
                stream=None, out: Optional[NormOut] = None) -> NormOut:
        """x, residual [n, H] -> NormOut.  norm / quantize: which outputs to make (the sum is made when there is a
        residual).  out: the tensors to write, in place of the three switches; its sum may be x or residual."""
        H, dev = self.hidden, x.device
        if x.dim() != 2 or x.shape[1] != H or x.dtype != self.dtype:
            raise C.EKError(C.EK_INVALID_INPUT, f"x must be [n, {H}] {self.dtype} (got {tuple(x.shape)} {x.dtype})")
        on_gpu = dev.type == "cuda"
        if on_gpu and dev.index != self.device_id:
            _check_device(x, self.device_id)
        if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != dev):
            raise C.EKError(C.EK_INVALID_INPUT, "residual must be like x")
        n = x.shape[0]
        if out is None or not x.is_contiguous() or (residual is not None and not residual.is_contiguous()):
            with _alloc_on(stream):
                x = x.contiguous()
                residual = residual.contiguous() if residual is not None else None
                if out is None:
                    out = NormOut(torch.empty_like(x) if residual is not None else None, torch.empty_like(x) if norm else None,
                                  torch.empty(n, H, dtype=torch.int8, device=dev) if quantize else None,
                                  torch.empty(n, dtype=torch.float32, device=dev) if quantize else None)
        total, y, q, scale = out
        for t, name, shape, dt in ((total, "sum", (n, H), x.dtype), (y, "y", (n, H), x.dtype), (q, "q", (n, H), torch.int8),
                                   (scale, "scale", (n,), torch.float32)):
            if t is not None and (t.shape != shape or t.dtype != dt or t.device != dev or not t.is_contiguous()):
                raise C.EKError(C.EK_INVALID_INPUT, f"out.{name} must be a contiguous {shape} {dt} tensor beside x")
        status = self._forward(self._h, x.data_ptr(), _addr(residual), n, _addr(total), _addr(y), _addr(q), _addr(scale),
                               C.EK_DEVICE if on_gpu else C.EK_HOST, _stream_ptr(stream))
        if status:
            C.check(status)
        return out

    def shape(self):
        hidden, dt = ctypes.c_int64(), ctypes.c_int32()
        C.check(self._lib.ek_norm_shape(self._h, ctypes.byref(hidden), ctypes.byref(dt)))
        return hidden.value

    def close(self) -> None:
        if getattr(self, "_h", None) is not None and self._h.value:
            self._lib.ek_norm_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class HipLinear:
    """One int8 matrix with a scale per output channel on 8-bit activations (ek_linear)."""

    def __init__(self, weight: torch.Tensor, scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                 act_dtype=torch.bfloat16, max_rows: int = 1024, device_id: int = 0):
        """weight [N, K] int8, scale [N], bias [N] or None."""
        if weight.dim() != 2 or scale.dim() != 1 or scale.numel() != weight.shape[0] or (bias is not None and tuple(bias.shape) != (weight.shape[0],)):
            raise C.EKError(C.EK_INVALID_INPUT, "weight must be [N, K], scale [N] and bias [N]")
        if weight.dtype not in _DT or scale.dtype not in _DT or act_dtype not in _DT or (bias is not None and bias.dtype not in _DT):
            raise C.EKError(C.EK_INVALID_INPUT, "unsupported dtype")
        self._lib = C.load()
        self.out_features, self.in_features = weight.shape
        self.act_dtype, self.device_id = act_dtype, device_id
        _check_device(weight, device_id)
        d, keep = _desc(weight, scale)
        if bias is not None:
            bias = bias.to(weight.device).contiguous()
        cfg = C.ek_linear_cfg(in_features=self.in_features, out_features=self.out_features, max_rows=max_rows,
                              act_dtype=_DT[act_dtype], device_id=device_id, flags=0)
        self._h = ctypes.c_void_p()
        C.check(self._lib.ek_linear_create(ctypes.byref(cfg), ctypes.byref(d), _addr(bias), _DT[bias.dtype] if bias is not None else C.EK_F32,
                                           ctypes.byref(self._h)))
        del keep

    def forward(self, x: torch.Tensor, scale: Optional[torch.Tensor] = None, stream=None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x [n, K]: int8 with scale [n] fp32, or of the activation dtype without (quantised by the library) -> [n, N]."""
        want = self.act_dtype if scale is None else torch.int8
        if x.dim() != 2 or x.shape[1] != self.in_features or x.dtype != want:
            raise C.EKError(C.EK_INVALID_INPUT, f"x must be [n, {self.in_features}] {want} (got {tuple(x.shape)} {x.dtype})")
        _check_device(x, self.device_id)
        n = x.shape[0]
        if scale is not None and (tuple(scale.shape) != (n,) or scale.dtype != torch.float32 or scale.device != x.device):
            raise C.EKError(C.EK_INVALID_INPUT, "scale must be [n] fp32 beside x")
        if out is not None and (tuple(out.shape) != (n, self.out_features) or out.dtype != self.act_dtype or out.device != x.device
                                or not out.is_contiguous()):
            raise C.EKError(C.EK_INVALID_INPUT, "out must be a contiguous [n, N] tensor of the activation dtype beside x")
        if out is None or not x.is_contiguous() or (scale is not None and not scale.is_contiguous()):
            with _alloc_on(stream):
                x = x.contiguous()
                scale = scale.contiguous() if scale is not None else None
                if out is None:
                    out = torch.empty(n, self.out_features, dtype=self.act_dtype, device=x.device)
        C.check(self._lib.ek_linear_forward(self._h, _addr(x), _addr(scale), n, _addr(out), _mem(x), _stream_ptr(stream)))
        return out

    def shape(self):
        k, n = ctypes.c_int64(), ctypes.c_int64()
        C.check(self._lib.ek_linear_shape(self._h, ctypes.byref(k), ctypes.byref(n)))
        return k.value, n.value

    def close(self) -> None:
        if getattr(self, "_h", None) is not None and self._h.value:
            self._lib.ek_linear_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
