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

import torch

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
    """Makes ``device`` current for the native calls."""
    return torch.cuda.device(device)


def _rows_view(x: torch.Tensor) -> torch.Tensor:
    """(n, d) rows of ``x``: a view where its rows are contiguous and in order, else a copy."""
    x2d = x if x.ndim == 2 else x.reshape(-1, x.shape[-1])
    if x2d.is_contiguous():
        return x2d
    n, d = x2d.shape
    if x2d.stride(1) != 1 or (n > 1 and x2d.stride(0) < d):
        x2d = x2d.contiguous()
    return x2d


def _params_for(x: torch.Tensor, gamma: torch.Tensor, beta):
    """gamma and beta in one dtype the kernels read: x's own, else fp32 (never rounded)."""
    dt = x.dtype if gamma.dtype == x.dtype and (beta is None or beta.dtype == x.dtype) else torch.float32
    if gamma.dtype != dt or not gamma.is_contiguous():
        gamma = gamma.to(dt).contiguous()
    if beta is not None and (beta.dtype != dt or not beta.is_contiguous()):
        beta = beta.to(dt).contiguous()
    return gamma, beta


def layernorm_forward(x2d: torch.Tensor, gamma: torch.Tensor, beta, eps: float, *, stats: bool = True):
    """(y, stats) of nimble_layernorm_forward for (n, d) rows; gamma and beta in x's dtype or fp32.

    ``stats`` (2, n) fp32 holds each row's mean and 1 / sqrt(var + eps); without
    it they are not written (None)."""
    dev = x2d.device
    if dev.index != torch.cuda.current_device():
        with _on(dev):
            return layernorm_forward(x2d, gamma, beta, eps, stats=stats)
    n, d = x2d.shape
    y = torch.empty((n, d), dtype=x2d.dtype, device=dev)
    st = torch.empty((2, n), dtype=torch.float32, device=dev) if stats else None
    mean = st.data_ptr() if stats else None
    native.call("nimble_layernorm_forward", x2d.data_ptr(), max(x2d.stride(0), d), gamma.data_ptr(),
                beta.data_ptr() if beta is not None else None, n, d, eps, _TORCH_TO_NIMBLE[x2d.dtype],
                _TORCH_TO_NIMBLE[gamma.dtype], y.data_ptr(), mean, mean + 4 * n if stats else None, _stream_ptr(dev))
    return y, st


def layernorm_backward(grad2d: torch.Tensor, x2d: torch.Tensor, gamma: torch.Tensor, stats: torch.Tensor, *,
                       bias: bool = True):
    """(grad_x in x's dtype, grad_gamma fp32, grad_beta fp32 or None); the row sums are in a fixed order."""
    dev = x2d.device
    if dev.index != torch.cuda.current_device():
        with _on(dev):
            return layernorm_backward(grad2d, x2d, gamma, stats, bias=bias)
    n, d = x2d.shape
    gy = grad2d if grad2d.dtype == x2d.dtype else grad2d.to(x2d.dtype)
    gy = gy.contiguous()
    gx = torch.empty((n, d), dtype=x2d.dtype, device=dev)
    gg = torch.empty(d, dtype=torch.float32, device=dev)
    gb = torch.empty(d, dtype=torch.float32, device=dev) if bias else None
    ws_bytes = native.layernorm_backward_workspace_size(n, d)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    mean = stats.data_ptr()
    native.call("nimble_layernorm_backward", gy.data_ptr(), x2d.data_ptr(), max(x2d.stride(0), d), gamma.data_ptr(),
                mean, mean + 4 * n, n, d, _TORCH_TO_NIMBLE[x2d.dtype], _TORCH_TO_NIMBLE[gamma.dtype], gx.data_ptr(),
                gg.data_ptr(), gb.data_ptr() if bias else None, ws.data_ptr(), ws_bytes, _stream_ptr(dev))
    return gx, gg, gb


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, eps):
        x2d = _rows_view(x)
        g, b = _params_for(x, gamma, beta)
        y, stats = layernorm_forward(x2d, g, b, eps)
        ctx.save_for_backward(x2d, g, stats)
        ctx.dtypes = (gamma.dtype, None if beta is None else beta.dtype)
        return y if x.ndim == 2 else y.view(x.shape)

    @staticmethod
    def backward(ctx, grad):
        if torch.is_grad_enabled():
            raise RuntimeError("layer_norm's backward is not differentiable itself")
        x2d, g, stats = ctx.saved_tensors
        gamma_dtype, beta_dtype = ctx.dtypes
        gx, gg, gb = layernorm_backward(grad if grad.ndim == 2 else grad.reshape(x2d.shape), x2d, g, stats,
                                        bias=beta_dtype is not None)
        if gamma_dtype != torch.float32:
            gg = gg.to(gamma_dtype)
        if gb is not None and beta_dtype != torch.float32:
            gb = gb.to(beta_dtype)
        return gx if grad.ndim == 2 else gx.view(grad.shape), gg, gb, None


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
    wants_grad = x.requires_grad
    for name, p in (("gamma", gamma), ("beta", beta)):
        if p is None and name == "beta":
            continue
        if p.ndim != 1 or p.shape[0] != d:
            raise ValueError(f"Expected {name} of shape ({d},), got {tuple(p.shape)}")
        if p.get_device() != x.get_device():
            raise ValueError(f"{name} is on {p.device}, x on {x.device}")
        compute_dtype_of(p)
        wants_grad = wants_grad or p.requires_grad
    if not 0 < d <= MAX_D:
        raise ValueError(f"layer_norm takes rows of 1 to {MAX_D} elements, got {d}")
    eps = float(eps)
    if wants_grad and torch.is_grad_enabled():
        return _LayerNormFn.apply(x, gamma, beta, eps)
    g, b = _params_for(x, gamma, beta)
    y = layernorm_forward(_rows_view(x), g, b, eps, stats=False)[0]
    return y if x.ndim == 2 else y.view(x.shape)


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
