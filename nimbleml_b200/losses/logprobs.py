"""Log probabilities of given tokens, with entropy and top alternatives.

The reference's losses return one mean (NimbleML/losses/cross_entropy.py:31-192).
Policy gradients, preference losses, distillation checks and scoring need the
terms of every token instead:

* ``token_logprobs(logits, tokens, top_k=k)`` over logits that exist (what
  ``lm_head.tied_logits`` and ``last_token_logits`` return): one pass for the
  log-sum-exp, the token's log probability, the entropy and the ``k`` best
  classes.
* ``tied_token_logprobs(hidden, weights, tokens)`` straight from the hidden
  states and the tied matrix. As in ``CrossEntropyLoss.forward_tied`` the logits
  are not kept: the forward keeps the lse and the entropy of each token, the
  backward recomputes the logits slab by slab (a slab holds at most half of them,
  or all where they take 256 MiB or less).

Both are differentiable in the log probabilities and in the entropies:
d/dx_j (a logp_t + b H) = a [j = t] - p_j (a + b (H + log p_j)).
Reverse mode only, once; inputs with a tangent and calls under a tracer raise.
"""
from __future__ import annotations

import contextlib
import math
from typing import NamedTuple, Optional

import torch

from nimbleml_b200 import vocab_parallel
from nimbleml_b200._host import host
from nimbleml_b200.kernels.fused_tied_crossentropy import (
    _NO_IGNORE,
    CHECK_BOUNDS,
    SLAB_BYTES,
    _monitor,
    _monitors,
    _status_words,
    _stream_ptr,
    as_label_indices,
    check_status,
    compute_dtype_of,
    native,
    poll_status,
    snapshot_status,
    status_word,
)

MAX_TOP_K = 64


class TokenLogProbs(NamedTuple):
    """Per-token results, all fp32 in the shape of ``tokens`` (alternatives: one more dimension of k).

    Tokens equal to ``ignore_index`` get 0, 0 and alternatives -inf, -1.
    """

    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: Optional[torch.Tensor] = None
    top_ids: Optional[torch.Tensor] = None


def _on(device: torch.device):
    """Makes ``device`` current where it is not."""
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _token_ids(tokens, n: int, device: torch.device) -> torch.Tensor:
    if (isinstance(tokens, torch.Tensor) and tokens.dtype == torch.int64 and tokens.device == device and
            tokens.numel() == n and tokens.is_contiguous()):
        return tokens  # the kernels read n ids in order, whatever the shape
    return as_label_indices(tokens, batch_size=n, device=device)


def _status_ptr(device: torch.device) -> int:
    """Address of the device's status word, which a captured launch must find in place, as the monitor's
    pinned memory: made by the first call on a device, it would otherwise lie in the graph's own memory."""
    if device.index not in _status_words or device.index not in _monitors:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("call the operator once on this device before capturing it into a CUDA graph")
        _monitor(device)
    return status_word(device).data_ptr()


def _refuse_double_backward() -> None:
    if torch.is_grad_enabled():
        raise RuntimeError("the log probabilities' backward is not differentiable itself")


def token_logprobs(logits: torch.Tensor, tokens, ignore_index: Optional[int] = None, *, top_k: int = 0) -> TokenLogProbs:
    """Log probability of ``tokens`` under ``logits`` (..., classes), the entropy of each
    row and, with ``top_k`` (at most 64), its best classes.

    Args:
        logits: float32, float16 or bfloat16 CUDA tensor; -inf marks classes
            that are ruled out. A row of -inf only gives -inf, entropy 0 and no
            gradient; NaN or +inf makes the row's numbers NaN.
        tokens: class ids, one per row of ``logits``.
        ignore_index: rows with this token are not read (results 0, 0).
        top_k: alternatives per row, by logit, equal ones by the lowest class
            id; not differentiable.

    A token outside the classes gives a NaN log probability and sets the
    status word's bad-label bit.
    """
    host.begin_token_logprobs(logits)
    if not logits.is_cuda:
        raise RuntimeError("token_logprobs on B200 needs CUDA tensors; there is no CPU path")
    compute_dtype_of(logits)
    shape = logits.shape
    if not shape or shape[-1] == 0:
        raise ValueError("logits must be (..., classes) with at least one class")
    v = shape[-1]
    top_k = int(top_k)
    if not 0 <= top_k <= min(MAX_TOP_K, v):
        raise ValueError(f"top_k must lie in [0, {min(MAX_TOP_K, v)}], got {top_k}")
    dev = logits.device
    ids = _token_ids(tokens, math.prod(shape[:-1]), dev)
    ign = _NO_IGNORE if ignore_index is None else int(ignore_index)
    out = TokenLogProbs(*host.token_logprobs(logits, ids, ign, top_k, _status_ptr(dev)))
    if CHECK_BOUNDS and not torch.cuda.is_current_stream_capturing():
        check_status(dev)
    return out


def shard_logprob_stats(h: torch.Tensor, w: torch.Tensor, tokens: torch.Tensor, vocab_offset: int = 0) -> torch.Tensor:
    """(4, N) statistics of one weight shard: a reference logit, sum 2^d, sum d 2^d (d = (s - reference) log2 e) and the
    token's logit (0 where the shard does not hold it)."""
    return host.tied_shard_stats(h, w, tokens, vocab_offset, _NO_IGNORE, _status_ptr(h.device))


def combine_logprob_stats(stats: torch.Tensor, tokens: torch.Tensor, vocab_size: int, ignore_index: int):
    """Merges (P, 4, N) shard statistics into (3, N): log probabilities, entropies, lse."""
    p, _, n = stats.shape
    dev = stats.device
    out = torch.empty((3, n), dtype=torch.float32, device=dev)
    at = out.data_ptr()
    native.call("nimble_tied_logprobs_combine", stats.data_ptr(), p, tokens.data_ptr(), n, vocab_size, ignore_index,
                at, at + 4 * n, at + 8 * n, status_word(dev).data_ptr(), _stream_ptr(dev))
    return out


def shard_logprob_backward(g_lp, g_ent, h, w, tokens, lse, ent, *, vocab_offset=0, vocab_size=None, ignore_index,
                           grad_hidden=None, grad_weights=None, accumulate=False):
    """Fills ``grad_hidden`` (this shard's partial) and fills or adds to ``grad_weights``, those that are given."""
    host.tied_backward(g_lp, g_ent, h, w, tokens, lse, ent, vocab_offset, w.shape[0] if vocab_size is None else vocab_size,
                       ignore_index, grad_hidden, grad_weights, accumulate, SLAB_BYTES,
                       _status_ptr(h.device))


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """Contiguous and on a 16-byte boundary, as the TMA loads need it."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _after_call(device: torch.device) -> None:
    snapshot_status(device)
    if CHECK_BOUNDS:
        check_status(device)


host.set_status_hooks(lambda index: poll_status(torch.device("cuda", index)),
                      lambda index: check_status(torch.device("cuda", index)))


def _shard_forward(hidden, weights, tokens, ignore_index, vocab_offset, vocab_size, group):
    """(h, w as the kernels read them, (3, n) log probability, entropy, lse) with the vocabulary in shards."""
    dev = hidden.device
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return _shard_forward(hidden, weights, tokens, ignore_index, vocab_offset, vocab_size, group)
    # 16-bit operands for the tensor cores; fp32 master weights still get an fp32 grad.
    w = _aligned(weights if weights.dtype == hidden.dtype else weights.to(hidden.dtype))
    h = _aligned(hidden if hidden.ndim == 2 else hidden.reshape(-1, hidden.shape[-1]))
    # A captured launch must not be joined by event queries and host copies.
    watch = not torch.cuda.is_current_stream_capturing()
    if watch:
        poll_status(dev)
    part = shard_logprob_stats(h, w, tokens, vocab_offset)
    if vocab_parallel.world_size(group) > 1:
        part = vocab_parallel.gather_shard_stats(part, group).transpose(0, 1).contiguous()
    else:
        part = part.unsqueeze(0)
    out = combine_logprob_stats(part, tokens, vocab_size, ignore_index)
    if watch:
        _after_call(dev)
    return h, w, out


class _ShardTokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weights, tokens, ignore_index, vocab_offset, vocab_size, group, grad_buffer):
        h, w, out = _shard_forward(hidden, weights, tokens, ignore_index, vocab_offset, vocab_size, group)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(h, w, tokens, out)
        ctx.meta = (ignore_index, vocab_offset, vocab_size, group, weights.dtype, hidden.shape)
        ctx.grad_buffer = grad_buffer
        return out[0], out[1]

    @staticmethod
    def backward(ctx, g_lp, g_ent):
        _refuse_double_backward()
        none = (None,) * 6
        if g_lp is None and g_ent is None:
            return (None, None, *none)
        h, w, tokens, out = ctx.saved_tensors
        ignore_index, vocab_offset, vocab_size, group, w_dtype, shape = ctx.meta
        buf = ctx.grad_buffer
        dev = h.device
        world = vocab_parallel.world_size(group)
        with _on(dev):
            gh = gw = None
            if ctx.needs_input_grad[0]:
                gh = torch.empty(h.shape, dtype=vocab_parallel.dh_reduce_dtype(h.dtype) if world > 1 else h.dtype,
                                 device=dev)
            if buf is not None:
                gw = buf
            elif ctx.needs_input_grad[1]:
                gw = torch.empty(w.shape, dtype=w_dtype, device=dev)
            watch = not torch.cuda.is_current_stream_capturing()
            if watch:
                poll_status(dev)
            shard_logprob_backward(g_lp, g_ent, h, w, tokens, out[2], out[1],
                                   vocab_offset=vocab_offset, vocab_size=vocab_size, ignore_index=ignore_index,
                                   grad_hidden=gh, grad_weights=gw, accumulate=buf is not None)
            if watch:
                _after_call(dev)
            if gh is not None and world > 1:
                gh = vocab_parallel.reduce_grad_hidden(gh, group).to(h.dtype)
        if gh is not None and len(shape) != 2:
            gh = gh.view(shape)
        return (gh, None if buf is not None else gw, *none)


def tied_token_logprobs(hidden: torch.Tensor, weights: torch.Tensor, tokens, ignore_index: Optional[int] = None, *,
                        vocab_offset: int = 0, vocab_size: Optional[int] = None, group=None,
                        grad_weights_buffer: Optional[torch.Tensor] = None) -> TokenLogProbs:
    """Log probability of ``tokens`` under ``hidden @ weights.T`` and the entropy of each row.

    Args:
        hidden: (..., d) float16 or bfloat16, d a multiple of 8. Rows of
            ignored tokens must be finite (they meet zero gradients).
        weights: (classes, d); cast to the hidden's dtype, its grad comes in its own.
        tokens: class ids, one per row of ``hidden``.
        ignore_index: rows with this token give 0, 0 and no gradient.
        vocab_offset, vocab_size, group: ``weights`` is this rank's vocab shard,
            as in :func:`tied_cross_entropy`.
        grad_weights_buffer: fp32 tensor of the weights' shape that the backward
            adds the weight grad into; autograd then gets none for ``weights``.

    The gradient of the logits is formed in the compute dtype, so gradients
    carry one 16-bit rounding more than their own. It averages out over many
    tokens; with a handful of them each term of the weight grad has it whole.
    Upstream gradients may have any size, and any sizes beside each other.
    """
    host.begin_tied_token_logprobs(hidden, weights)
    if not hidden.is_cuda:
        raise RuntimeError("tied_token_logprobs on B200 needs CUDA tensors; there is no CPU path")
    if hidden.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("tied log probabilities run in float16 or bfloat16")
    if weights.ndim != 2 or hidden.ndim == 0 or hidden.shape[-1] != weights.shape[1]:
        raise ValueError("hidden must be (..., d_model) and weights (vocab, d_model)")
    if weights.device != hidden.device:
        raise ValueError(f"weights are on {weights.device}, hidden on {hidden.device}")
    compute_dtype_of(weights)
    v, d = weights.shape
    if v == 0 or d == 0 or d % 8 != 0:
        raise ValueError(f"weights must be (vocab, d_model) with d_model a multiple of 8, got {tuple(weights.shape)}")
    vocab_size = v if vocab_size is None else int(vocab_size)
    if vocab_offset < 0 or vocab_offset + v > vocab_size:
        raise ValueError("the shard must lie inside the vocabulary")
    if grad_weights_buffer is not None and (grad_weights_buffer.dtype != torch.float32 or
                                            grad_weights_buffer.shape != weights.shape or
                                            grad_weights_buffer.device != weights.device or
                                            not grad_weights_buffer.is_contiguous()):
        raise ValueError("grad_weights_buffer must be a contiguous float32 tensor of the weights' shape")
    shape = hidden.shape[:-1]
    ids = _token_ids(tokens, math.prod(shape), hidden.device)
    ign = _NO_IGNORE if ignore_index is None else int(ignore_index)
    if v == vocab_size and vocab_parallel.world_size(group) == 1:
        dev = hidden.device
        return TokenLogProbs(*host.tied_token_logprobs(hidden, weights, ids, ign, grad_weights_buffer, SLAB_BYTES,
                                                       _status_ptr(dev), _monitor(dev).flag_ptr, CHECK_BOUNDS))
    args = (hidden, weights, ids, ign, int(vocab_offset), vocab_size, group)
    if (hidden.requires_grad or weights.requires_grad) and torch.is_grad_enabled():
        lp, ent = _ShardTokenLogProbs.apply(*args, grad_weights_buffer)
    else:
        out = _shard_forward(*args)[2]
        lp, ent = out[0], out[1]
    if len(shape) != 1:
        lp, ent = lp.view(shape), ent.view(shape)
    return TokenLogProbs(lp, ent)


__all__ = ["TokenLogProbs", "token_logprobs", "tied_token_logprobs", "MAX_TOP_K"]
