"""The tied matrix's other grad and its update: embedding scatter-add and AdamW.

* ``embedding_scatter_add`` — grad_weights[ids] += grad_out, the input
  embedding's share of the tied matrix's grad
  (NimbleML/kernels/embedding_scatter.py:39-81), into an fp32 grad buffer,
  deterministically and for one vocab shard.
* ``AdamW`` — the reference's fused AdamW update (NimbleML/optimizers/adam.py:20-43,
  85-131, 295-312) over fp32 master weights, e.g. one rank's vocab shard of E,
  with an optional low-precision copy written in the same pass. A step
  updates all tensors in one launch, with the moments in 32 or in 8 bits.
* ``adamw_step_many`` — that step as a function over lists of tensors.
"""
from __future__ import annotations

import contextlib
from typing import Iterable, NamedTuple, Optional, Sequence, Union

import torch

from nimbleml_b200._host import host
from nimbleml_b200.kernels.fused_tied_crossentropy import _TORCH_TO_NIMBLE, _stream_ptr, native, status_word


def embedding_scatter_add(grad_weights: torch.Tensor, ids: torch.Tensor, grad_out: torch.Tensor, *,
                          vocab_offset: int = 0, vocab_size: Optional[int] = None) -> torch.Tensor:
    """In-place ``grad_weights[ids[i] - vocab_offset] += grad_out[i]`` into an fp32 grad.

    ``grad_weights`` holds rows [vocab_offset, vocab_offset + rows) of a
    ``vocab_size`` vocabulary (default: all of it); ids of other rows are
    skipped, ids outside [0, vocab_size) set the status word's bad-label bit.
    Deterministic: each id's rows are added in ascending row order, the loop
    order of the reference's CPU scatter (native/src/scatter.cpp:6-15).
    """
    if grad_weights.dtype != torch.float32 or not grad_weights.is_contiguous():
        raise ValueError("grad_weights must be a contiguous float32 (vocab, d) tensor")
    v, d = grad_weights.shape
    vocab_size = v if vocab_size is None else int(vocab_size)
    flat_ids = ids.reshape(-1).to(torch.int64).contiguous()
    go = grad_out.reshape(-1, d).contiguous()
    n = go.shape[0]
    if n != flat_ids.numel():
        raise ValueError(f"ids length ({flat_ids.numel()}) must match grad_out rows ({n}).")
    if n == 0:
        return grad_weights
    ws_bytes = native.scatter_add_workspace_size(n, v)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=go.device)
    native.call("nimble_embedding_scatter_add", grad_weights.data_ptr(), flat_ids.data_ptr(), go.data_ptr(), n,
                int(vocab_offset), v, vocab_size, d, _TORCH_TO_NIMBLE[go.dtype], ws.data_ptr(), ws_bytes,
                status_word(go.device).data_ptr(), _stream_ptr(go.device))
    return grad_weights


QUANT_BLOCK = 128  # elements that share a scale


class QuantizedMoment(NamedTuple):
    """An AdamW moment in 8 bits: e4m3 codes of the tensor's shape and one fp32
    scale for each run of 128 elements. The second moment holds its root."""

    codes: torch.Tensor
    scales: torch.Tensor


def _on(device: torch.device):
    """Makes ``device`` current for the native calls when it is not."""
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _check_quantized(codes: torch.Tensor, scales: torch.Tensor) -> None:
    if codes.dtype != torch.float8_e4m3fn or not codes.is_contiguous():
        raise ValueError("8-bit moments are contiguous float8_e4m3fn codes")
    if (scales.dtype != torch.float32 or not scales.is_contiguous() or
            scales.numel() != -(-codes.numel() // QUANT_BLOCK)):
        raise ValueError(f"8-bit moments need one contiguous float32 scale per {QUANT_BLOCK} elements")
    if not codes.is_cuda or scales.device != codes.device:
        raise ValueError("8-bit moments live on one CUDA device")


def quantize_moment(x: torch.Tensor, *, root: bool = False) -> QuantizedMoment:
    """An fp32 moment in 8 bits; ``root`` for the second moment, which is held as its root."""
    host.begin_quantize(x)
    if x.dtype != torch.float32 or not x.is_cuda:
        raise ValueError("moments are float32 CUDA tensors")
    x = x.contiguous()
    codes = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scales = torch.empty(-(-x.numel() // QUANT_BLOCK), dtype=torch.float32, device=x.device)
    with _on(x.device):
        native.call("nimble_adamw_quantize", x.data_ptr(), x.numel(), int(root), codes.data_ptr(), scales.data_ptr(),
                    _stream_ptr(x.device))
    return QuantizedMoment(codes, scales)


def dequantize_moment(codes: torch.Tensor, scales: torch.Tensor, *, root: bool = False) -> torch.Tensor:
    """The fp32 values that 8-bit codes stand for (``root``: their squares, the second moment)."""
    host.begin_dequantize(codes, scales)
    _check_quantized(codes, scales)
    out = torch.empty(codes.shape, dtype=torch.float32, device=codes.device)
    with _on(codes.device):
        native.call("nimble_adamw_dequantize", codes.data_ptr(), scales.data_ptr(), codes.numel(), int(root),
                    out.data_ptr(), _stream_ptr(codes.device))
    return out


Moment = Union[torch.Tensor, QuantizedMoment]


def adamw_step_many(params: Sequence[torch.Tensor], grads: Sequence[Optional[torch.Tensor]],
                    exp_avgs: Sequence[Moment], exp_avg_sqs: Sequence[Moment], *, step: int,
                    learning_rate: float = 0.001, beta1: float = 0.9, beta2: float = 0.999, epsilon: float = 1e-8,
                    weight_decay: float = 0.01, copies: Optional[Sequence[Optional[torch.Tensor]]] = None) -> None:
    """One in-place AdamW step over many tensors, in one launch for up to 400 of them.

    Args:
        params: contiguous fp32 master weights of any sizes. Two that overlap in part must
            not be in one step; one that is listed twice is updated twice, in order.
        grads: gradients of the same sizes (float32, float16 or bfloat16);
            tensors whose gradient is None are left as they are.
        exp_avgs, exp_avg_sqs: all fp32 tensors, or all 8-bit pairs (codes,
            scales) as :class:`QuantizedMoment` describes them.
        step: the step's number, from 1 (bias correction).
        copies: tensors (or None) that receive the new weights in their dtype.

    The update is that of the reference's AdamW (NimbleML/optimizers/adam.py:20-43).
    With 8-bit moments the weights are updated from the new moments before
    these are rounded. A gradient that is not finite spoils its own weight and,
    with 8-bit moments, the block of 128 it lies in. A captured step keeps the
    scalars it was captured with. All tensors are checked first: a step that is
    refused changes none of them. It counts as an in-place write: a backward
    pass that has kept an updated tensor raises.
    """
    host.adamw_step_many(params, grads, exp_avgs, exp_avg_sqs, copies, int(step), float(learning_rate), float(beta1),
                         float(beta2), float(epsilon), float(weight_decay), False)


class AdamW:
    """AdamW over fp32 master tensors (learning_rate, beta1, beta2, epsilon, weight_decay
    as in the reference's ``AdamW``); ``copies`` optionally receive the updated
    weights in their own dtype (e.g. the fp16 E used by the GEMMs).

    ``state_bits``: 32 keeps the moments ``m`` and ``v`` as fp32 tensors (8
    bytes a weight), 8 as :class:`QuantizedMoment` pairs (2.06 bytes); ``v``
    then holds the second moment's root, and ``moments()`` gives both in fp32.
    """

    def __init__(self, params: Iterable[torch.Tensor], learning_rate=0.001, beta1=0.9, beta2=0.999,
                 epsilon=1e-8, weight_decay=0.01, copies: Optional[Iterable[Optional[torch.Tensor]]] = None,
                 state_bits: int = 32):
        self.params = list(params)
        for p in self.params:
            if p.dtype != torch.float32 or not p.is_contiguous():
                raise ValueError("AdamW master weights must be contiguous float32 tensors")
        if state_bits not in (32, 8):
            raise ValueError("state_bits must be 32 or 8")
        self.state_bits = int(state_bits)
        self.copies = list(copies) if copies is not None else [None] * len(self.params)
        if len(self.copies) != len(self.params):
            raise ValueError(f"copies must have one entry per tensor: {len(self.copies)} for {len(self.params)}")
        self.lr, self.beta1, self.beta2 = float(learning_rate), float(beta1), float(beta2)
        self.epsilon, self.weight_decay = float(epsilon), float(weight_decay)
        self.m = [self._zero_moment(p) for p in self.params]
        self.v = [self._zero_moment(p) for p in self.params]
        self.t = 0

    def _zero_moment(self, p: torch.Tensor) -> Moment:
        if self.state_bits == 32:
            return torch.zeros_like(p)
        return QuantizedMoment(torch.zeros(p.shape, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn),
                               torch.zeros(-(-p.numel() // QUANT_BLOCK), dtype=torch.float32, device=p.device))

    def moments(self):
        """(first moments, second moments) as lists of fp32 tensors: the state itself in 32 bits, else its values."""
        if self.state_bits == 32:
            return self.m, self.v
        return [dequantize_moment(*q) for q in self.m], [dequantize_moment(*q, root=True) for q in self.v]

    @torch.no_grad()
    def step(self):
        """One step over all tensors with a gradient; a refused one changes neither them nor ``t``.

        With fp32 moments, tensors that are not whole eights on 16-byte
        boundaries keep a launch of their own (``nimble_adamw_step``), whose
        scalar kernel rounds in another order than the list's.
        """
        host.adamw_step_many(self.params, [p.grad for p in self.params], self.m, self.v, self.copies, self.t + 1,
                             self.lr, self.beta1, self.beta2, self.epsilon, self.weight_decay, True)
        self.t += 1

    def zero_grad(self, set_to_none: bool = True):
        for p in self.params:
            p.grad = None if set_to_none else (torch.zeros_like(p) if p.grad is None else p.grad.zero_())


__all__ = ["embedding_scatter_add", "AdamW", "QuantizedMoment", "adamw_step_many", "quantize_moment",
           "dequantize_moment"]
