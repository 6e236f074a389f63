"""RMSNorm and LayerNorm on B200 — the norms whose output is the tied head's input.

Mirrors NimbleML/layers/rms_norm.py:9-90 (``RMSNorm(normalized_shape,
epsilon)`` with a learnable ``gamma``) over ``nimble_rmsnorm_forward /
_backward``: fp32 row statistics, one read and one write per element, and a
deterministic grad_gamma (per-block partial sums reduced in a fixed order).

``LayerNorm(normalized_shape, epsilon)`` with learnable ``gamma`` and ``beta``
stands beside it over ``nimble_layernorm_forward / _backward``, with the same
guarantees.
"""
from __future__ import annotations

import contextlib

import torch
from torch.autograd.function import once_differentiable

from nimbleml_b200.kernels.fused_tied_crossentropy import _TORCH_TO_NIMBLE, _stream_ptr, compute_dtype_of, native


class _RMSNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, eps):
        d = x.shape[-1]
        x2d = x.reshape(-1, d).contiguous()
        g = gamma.to(x.dtype).contiguous()
        y, ms, rms = rmsnorm_forward(x2d, g, eps)
        ctx.save_for_backward(x2d, g, ms, rms)
        ctx.eps = float(eps)
        ctx.gamma_dtype = gamma.dtype
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, grad):
        x2d, g, ms, rms = ctx.saved_tensors
        n, d = x2d.shape
        gx, gg = rmsnorm_backward(grad.reshape(n, d), x2d, g, ms, rms, ctx.eps)
        return gx.view(grad.shape), gg.to(ctx.gamma_dtype), None


def rmsnorm_forward(x2d: torch.Tensor, gamma: torch.Tensor, eps: float):
    """(y, ms, rms) of nimble_rmsnorm_forward for a contiguous (n, d) input; gamma in x's dtype."""
    n, d = x2d.shape
    y = torch.empty_like(x2d)
    ms = torch.empty(n, dtype=torch.float32, device=x2d.device)
    rms = torch.empty(n, dtype=torch.float32, device=x2d.device)
    native.call("nimble_rmsnorm_forward", x2d.data_ptr(), gamma.data_ptr(), n, d, float(eps),
                _TORCH_TO_NIMBLE[x2d.dtype], y.data_ptr(), ms.data_ptr(), rms.data_ptr(), _stream_ptr(x2d.device))
    return y, ms, rms


def rmsnorm_backward(grad2d: torch.Tensor, x2d: torch.Tensor, gamma: torch.Tensor, ms: torch.Tensor,
                     rms: torch.Tensor, eps: float):
    """(grad_x in x's dtype, grad_gamma fp32). An fp32 ``grad2d`` is read as is
    (the tied head's fp32 grad_hidden); other dtypes are cast to x's dtype."""
    n, d = x2d.shape
    if grad2d.dtype != torch.float32 and grad2d.dtype != x2d.dtype:
        grad2d = grad2d.to(x2d.dtype)
    gy = grad2d.contiguous()
    gx = torch.empty_like(x2d)
    gg = torch.empty(d, dtype=torch.float32, device=x2d.device)
    ws_bytes = native.rmsnorm_backward_workspace_size(n, d)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=x2d.device)
    native.call("nimble_rmsnorm_backward", gy.data_ptr(), x2d.data_ptr(), gamma.data_ptr(), ms.data_ptr(),
                rms.data_ptr(), n, d, float(eps), _TORCH_TO_NIMBLE[x2d.dtype], _TORCH_TO_NIMBLE[gy.dtype],
                gx.data_ptr(), gg.data_ptr(), 0, ws.data_ptr(), ws_bytes, _stream_ptr(x2d.device))
    return gx, gg


def rms_norm(x: torch.Tensor, gamma: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    """y = x / sqrt(mean(x^2, -1) + eps) * gamma."""
    if x.shape[-1] != gamma.shape[-1]:
        raise ValueError(f"Expected last dim {gamma.shape[-1]}, got {x.shape[-1]}")
    compute_dtype_of(x)
    return _RMSNormFn.apply(x, gamma, eps)


class RMSNorm(torch.nn.Module):
    """``RMSNorm(normalized_shape, epsilon=1e-5)`` with ``gamma`` initialised to ones."""

    def __init__(self, normalized_shape: int, epsilon: float = 1e-5, device=None, dtype=torch.float32):
        super().__init__()
        self.normalized_shape = int(normalized_shape)
        self.epsilon = float(epsilon)
        self.gamma = torch.nn.Parameter(torch.ones(self.normalized_shape, device=device, dtype=dtype))

    def forward(self, inputs: torch.Tensor) -> torch.Tensor:
        if inputs.shape[-1] != self.normalized_shape:
            raise ValueError(f"Expected last dim {self.normalized_shape}, got {inputs.shape[-1]}")
        return rms_norm(inputs, self.gamma, self.epsilon)


MAX_D = 8192


def _on(device: torch.device):
    """Makes ``device`` current for the native calls when it is not."""
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _rows_view(x: torch.Tensor) -> torch.Tensor:
    """(n, d) rows of ``x``: a view where its rows are contiguous and in order, else a copy."""
    x2d = x.reshape(-1, x.shape[-1])
    n, d = x2d.shape
    if x2d.stride(1) != 1 or (n > 1 and x2d.stride(0) < d):
        x2d = x2d.contiguous()
    return x2d


def _params_for(x: torch.Tensor, gamma: torch.Tensor, beta):
    """gamma and beta in one dtype the kernels read: x's own, else fp32 (never rounded)."""
    dt = x.dtype if gamma.dtype == x.dtype and (beta is None or beta.dtype == x.dtype) else torch.float32
    return gamma.to(dt).contiguous(), None if beta is None else beta.to(dt).contiguous()


def layernorm_forward(x2d: torch.Tensor, gamma: torch.Tensor, beta, eps: float, *, stats: bool = True):
    """(y, mean, rstd) of nimble_layernorm_forward for (n, d) rows; gamma and beta in x's dtype or fp32.

    Without ``stats`` the row statistics are not written (None)."""
    n, d = x2d.shape
    dev = x2d.device
    y = torch.empty((n, d), dtype=x2d.dtype, device=dev)
    mean, rstd = torch.empty((2, n), dtype=torch.float32, device=dev).unbind(0) if stats else (None, None)
    with _on(dev):
        native.call("nimble_layernorm_forward", x2d.data_ptr(), max(x2d.stride(0), d), gamma.data_ptr(),
                    beta.data_ptr() if beta is not None else None, n, d, float(eps), _TORCH_TO_NIMBLE[x2d.dtype],
                    _TORCH_TO_NIMBLE[gamma.dtype], y.data_ptr(), mean.data_ptr() if stats else None,
                    rstd.data_ptr() if stats else None, _stream_ptr(dev))
    return y, mean, rstd


def layernorm_backward(grad2d: torch.Tensor, x2d: torch.Tensor, gamma: torch.Tensor, mean: torch.Tensor,
                       rstd: torch.Tensor):
    """(grad_x in x's dtype, grad_gamma fp32, grad_beta fp32); the row sums are in a fixed order."""
    n, d = x2d.shape
    dev = x2d.device
    gy = grad2d.to(x2d.dtype).contiguous()
    gx = torch.empty((n, d), dtype=x2d.dtype, device=dev)
    gg, gb = torch.empty((2, d), dtype=torch.float32, device=dev).unbind(0)
    ws_bytes = native.layernorm_backward_workspace_size(n, d)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    with _on(dev):
        native.call("nimble_layernorm_backward", gy.data_ptr(), x2d.data_ptr(), max(x2d.stride(0), d),
                    gamma.data_ptr(), mean.data_ptr(), rstd.data_ptr(), n, d, _TORCH_TO_NIMBLE[x2d.dtype],
                    _TORCH_TO_NIMBLE[gamma.dtype], gx.data_ptr(), gg.data_ptr(), gb.data_ptr(), ws.data_ptr(),
                    ws_bytes, _stream_ptr(dev))
    return gx, gg, gb


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, eps):
        x2d = _rows_view(x)
        g, b = _params_for(x, gamma, beta)
        y, mean, rstd = layernorm_forward(x2d, g, b, eps)
        ctx.save_for_backward(x2d, g, mean, rstd)
        ctx.dtypes = (gamma.dtype, None if beta is None else beta.dtype)
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x2d, g, mean, rstd = ctx.saved_tensors
        gx, gg, gb = layernorm_backward(grad.reshape(x2d.shape), x2d, g, mean, rstd)
        gamma_dtype, beta_dtype = ctx.dtypes
        return gx.view(grad.shape), gg.to(gamma_dtype), None if beta_dtype is None else gb.to(beta_dtype), None


def layer_norm(x: torch.Tensor, gamma: torch.Tensor, beta=None, eps: float = 1e-5) -> torch.Tensor:
    """y = (x - mean(x)) / sqrt(var(x) + eps) * gamma + beta over the last dimension (at most 8192).

    ``x`` is float32, float16 or bfloat16; ``gamma`` and ``beta`` (None: no
    bias) have the last dimension's size and any of these dtypes. Statistics
    are fp32, the variance is the biased one of centred values.
    """
    if not x.is_cuda:
        raise RuntimeError("layer_norm on B200 needs CUDA tensors; there is no CPU path")
    compute_dtype_of(x)
    d = x.shape[-1] if x.ndim else 0
    for name, p in (("gamma", gamma), ("beta", beta)):
        if p is None and name == "beta":
            continue
        if tuple(p.shape) != (d,):
            raise ValueError(f"Expected {name} of shape ({d},), got {tuple(p.shape)}")
        if p.device != x.device:
            raise ValueError(f"{name} is on {p.device}, x on {x.device}")
        compute_dtype_of(p)
    if not 0 < d <= MAX_D:
        raise ValueError(f"layer_norm takes rows of 1 to {MAX_D} elements, got {d}")
    if torch.is_grad_enabled() and (x.requires_grad or gamma.requires_grad or
                                    (beta is not None and beta.requires_grad)):
        return _LayerNormFn.apply(x, gamma, beta, float(eps))
    g, b = _params_for(x, gamma, beta)
    return layernorm_forward(_rows_view(x), g, b, eps, stats=False)[0].view(x.shape)


class LayerNorm(torch.nn.Module):
    """``LayerNorm(normalized_shape, epsilon=1e-5)`` with ``gamma`` ones and ``beta`` zeros (``bias=False``: none)."""

    def __init__(self, normalized_shape: int, epsilon: float = 1e-5, bias: bool = True, device=None,
                 dtype=torch.float32):
        super().__init__()
        self.normalized_shape = int(normalized_shape)
        self.epsilon = float(epsilon)
        self.gamma = torch.nn.Parameter(torch.ones(self.normalized_shape, device=device, dtype=dtype))
        self.beta = torch.nn.Parameter(torch.zeros(self.normalized_shape, device=device, dtype=dtype)) if bias else None

    def forward(self, inputs: torch.Tensor) -> torch.Tensor:
        if inputs.shape[-1] != self.normalized_shape:
            raise ValueError(f"Expected last dim {self.normalized_shape}, got {inputs.shape[-1]}")
        return layer_norm(inputs, self.gamma, self.beta, self.epsilon)


__all__ = ["RMSNorm", "rms_norm", "rmsnorm_forward", "rmsnorm_backward", "LayerNorm", "layer_norm",
           "layernorm_forward", "layernorm_backward"]
