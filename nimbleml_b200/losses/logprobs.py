"""Log probabilities of given tokens, with entropy and top alternatives.

The reference's losses return one mean (NimbleML/losses/cross_entropy.py:31-192).
Policy gradients, preference losses, distillation checks and scoring need the
terms of every token instead:

* ``token_logprobs(logits, tokens, top_k=k)`` over logits that exist (what
  ``lm_head.tied_logits`` and ``last_token_logits`` return): one pass for the
  log-sum-exp, the token's log probability, the entropy and the ``k`` best
  classes.
* ``tied_token_logprobs(hidden, weights, tokens)`` straight from the hidden
  states and the tied matrix. As in ``CrossEntropyLoss.forward_tied`` no N x V
  buffer exists: the forward keeps the lse and the entropy of each token, the
  backward recomputes the logits slab by slab.

Both are differentiable in the log probabilities and in the entropies:
d/dx_j (a logp_t + b H) = a [j = t] - p_j (a + b (H + log p_j)).
"""
from __future__ import annotations

import contextlib
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from nimbleml_b200.kernels.fused_tied_crossentropy import (
    _NO_IGNORE,
    _TORCH_TO_NIMBLE,
    CHECK_BOUNDS,
    SLAB_BYTES,
    _stream_ptr,
    _workspace,
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
    """Makes ``device`` current for the native calls when it is not."""
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _grad_rows(grad: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if grad is None else grad.reshape(-1).float().contiguous()


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x2d, tokens, ignore_index, top_k):
        n, v = x2d.shape
        dev = x2d.device
        # Rows may be a view of wider ones; a broadcast or a transposed matrix is copied.
        if x2d.stride(1) != 1 or (n > 1 and x2d.stride(0) < v):
            x2d = x2d.contiguous()
        out = torch.empty((4, n), dtype=torch.float32, device=dev)
        top_lp = torch.empty((n, top_k), dtype=torch.float32, device=dev) if top_k else None
        top_id = torch.empty((n, top_k), dtype=torch.int64, device=dev) if top_k else None
        with _on(dev):
            native.call("nimble_token_logprobs_forward", x2d.data_ptr(), max(x2d.stride(0), v), tokens.data_ptr(), n,
                        v, _TORCH_TO_NIMBLE[x2d.dtype], ignore_index, top_k, out[0].data_ptr(), out[1].data_ptr(),
                        out[2].data_ptr(), out[3].data_ptr(), _ptr(top_lp), _ptr(top_id), status_word(dev).data_ptr(), _stream_ptr(dev))
        if CHECK_BOUNDS:
            check_status(dev)
        lp, ent, row_max, logsum = out.unbind(0)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x2d, tokens, row_max, logsum, ent)
        ctx.ignore_index = ignore_index
        if top_k:
            ctx.mark_non_differentiable(top_lp, top_id)
        return lp, ent, top_lp, top_id

    @staticmethod
    @once_differentiable
    def backward(ctx, g_lp, g_ent, *_):
        x2d, tokens, row_max, logsum, ent = ctx.saved_tensors
        if g_lp is None and g_ent is None:
            return None, None, None, None
        n, v = x2d.shape
        ld = max(x2d.stride(0), v)
        # Rows of whole 16 bytes where the logits have them, so that both sides use vectors.
        per16 = 16 // x2d.element_size()
        pitch = -(-v // per16) * per16 if ld % per16 == 0 else v
        g = torch.empty((n, pitch), dtype=x2d.dtype, device=x2d.device)
        a, b = _grad_rows(g_lp), _grad_rows(g_ent)
        with _on(x2d.device):
            native.call("nimble_token_logprobs_backward", _ptr(a), _ptr(b), x2d.data_ptr(), ld, tokens.data_ptr(),
                        row_max.data_ptr(), logsum.data_ptr(), ent.data_ptr(), n, v, _TORCH_TO_NIMBLE[x2d.dtype], ctx.ignore_index,
                        g.data_ptr(), pitch, _stream_ptr(x2d.device))
        return g[:, :v], None, None, None


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
    if not logits.is_cuda:
        raise RuntimeError("token_logprobs on B200 needs CUDA tensors; there is no CPU path")
    compute_dtype_of(logits)
    if logits.ndim == 0 or logits.shape[-1] == 0:
        raise ValueError("logits must be (..., classes) with at least one class")
    v = logits.shape[-1]
    top_k = int(top_k)
    if not 0 <= top_k <= min(MAX_TOP_K, v):
        raise ValueError(f"top_k must lie in [0, {min(MAX_TOP_K, v)}], got {top_k}")
    shape = logits.shape[:-1]
    x2d = logits.reshape(-1, v)
    ids = as_label_indices(tokens, batch_size=x2d.shape[0], device=logits.device)
    ign = _NO_IGNORE if ignore_index is None else int(ignore_index)
    lp, ent, top_lp, top_id = _TokenLogProbs.apply(x2d, ids, ign, top_k)
    if not top_k:
        return TokenLogProbs(lp.reshape(shape), ent.reshape(shape))
    return TokenLogProbs(lp.reshape(shape), ent.reshape(shape), top_lp.reshape(*shape, top_k),
                         top_id.reshape(*shape, top_k))


def shard_logprob_stats(h: torch.Tensor, w: torch.Tensor, tokens: torch.Tensor, vocab_offset: int = 0) -> torch.Tensor:
    """(4, N) statistics of one weight shard: max, sum 2^d, sum d 2^d (d = (s - max) log2 e)
    and the token's logit (0 where the shard does not hold it)."""
    n, d = h.shape
    v_local = w.shape[0]
    dt = compute_dtype_of(h)
    dev = h.device
    out = torch.empty((4, n), dtype=torch.float32, device=dev)
    ws = _workspace(native.tied_logprobs_forward_workspace_size(n, d, v_local, dt), dev)
    native.call("nimble_tied_logprobs_forward", h.data_ptr(), w.data_ptr(), tokens.data_ptr(), n, d, v_local,
                vocab_offset, dt, out.data_ptr(), ws.data_ptr(), ws.numel(), status_word(dev).data_ptr(),
                _stream_ptr(dev))
    return out


def combine_logprob_stats(stats: torch.Tensor, tokens: torch.Tensor, vocab_size: int, ignore_index: int):
    """Merges (P, 4, N) shard statistics into (logprobs, entropy, lse), each (N,)."""
    p, _, n = stats.shape
    dev = stats.device
    out = torch.empty((3, n), dtype=torch.float32, device=dev)
    native.call("nimble_tied_logprobs_combine", stats.data_ptr(), p, tokens.data_ptr(), n, vocab_size, ignore_index,
                out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), status_word(dev).data_ptr(),
                _stream_ptr(dev))
    return out.unbind(0)


def shard_logprob_backward(g_lp, g_ent, h, w, tokens, lse, ent, *, vocab_offset=0, vocab_size=None, ignore_index,
                           grad_hidden=None, grad_weights=None, accumulate=False):
    """Adds nothing to None: fills ``grad_hidden`` (this shard's partial) and ``grad_weights`` where given."""
    n, d = h.shape
    v_local = w.shape[0]
    dt = compute_dtype_of(h)
    dev = h.device
    ws = _workspace(native.tied_logprobs_backward_workspace_size(n, d, v_local, dt, SLAB_BYTES), dev)
    native.call("nimble_tied_logprobs_backward", _ptr(g_lp), _ptr(g_ent), h.data_ptr(), w.data_ptr(),
                tokens.data_ptr(), lse.data_ptr(), ent.data_ptr(), n, d, v_local, vocab_offset,
                v_local if vocab_size is None else vocab_size, ignore_index, dt, _ptr(grad_hidden),
                _TORCH_TO_NIMBLE[grad_hidden.dtype] if grad_hidden is not None else dt, _ptr(grad_weights),
                _TORCH_TO_NIMBLE[grad_weights.dtype] if grad_weights is not None else dt, 1 if accumulate else 0,
                SLAB_BYTES, ws.data_ptr(), ws.numel(), status_word(dev).data_ptr(), _stream_ptr(dev))


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """Contiguous and on a 16-byte boundary, as the TMA loads need it."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


class _TiedTokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h2d, weights, tokens, ignore_index, vocab_offset, vocab_size, group, grad_buffer):
        from nimbleml_b200 import vocab_parallel

        dev = h2d.device
        # 16-bit operands for the tensor cores; fp32 master weights still get an fp32 grad.
        w = _aligned(weights if weights.dtype == h2d.dtype else weights.to(h2d.dtype))
        h = _aligned(h2d)
        # A captured launch must not be joined by event queries and host copies.
        watch = not torch.cuda.is_current_stream_capturing()
        with _on(dev):
            if watch:
                poll_status(dev)
            part = shard_logprob_stats(h, w, tokens, vocab_offset)
            if vocab_parallel.world_size(group) > 1:
                part = vocab_parallel.gather_shard_stats(part, group).transpose(0, 1).contiguous()
            else:
                part = part.unsqueeze(0)
            lp, ent, lse = combine_logprob_stats(part, tokens, vocab_size, ignore_index)
            if watch:
                snapshot_status(dev)
        if CHECK_BOUNDS:
            check_status(dev)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(h, w, tokens, lse, ent)
        ctx.meta = (ignore_index, vocab_offset, vocab_size, group, weights.dtype)
        ctx.grad_buffer = grad_buffer
        return lp, ent

    @staticmethod
    @once_differentiable
    def backward(ctx, g_lp, g_ent):
        from nimbleml_b200 import vocab_parallel

        none = (None,) * 6
        if g_lp is None and g_ent is None:
            return (None, None, *none)
        h, w, tokens, lse, ent = ctx.saved_tensors
        ignore_index, vocab_offset, vocab_size, group, w_dtype = ctx.meta
        buf = ctx.grad_buffer
        dev = h.device
        world = vocab_parallel.world_size(group)
        gh = gw = None
        if ctx.needs_input_grad[0]:
            gh = torch.empty(h.shape, dtype=vocab_parallel.dh_reduce_dtype(h.dtype) if world > 1 else h.dtype,
                             device=dev)
        if buf is not None:
            gw = buf
        elif ctx.needs_input_grad[1]:
            gw = torch.empty(w.shape, dtype=w_dtype, device=dev)
        watch = not torch.cuda.is_current_stream_capturing()
        with _on(dev):
            if watch:
                poll_status(dev)
            shard_logprob_backward(_grad_rows(g_lp), _grad_rows(g_ent), h, w, tokens, lse, ent,
                                   vocab_offset=vocab_offset, vocab_size=vocab_size, ignore_index=ignore_index,
                                   grad_hidden=gh, grad_weights=gw, accumulate=buf is not None)
            if watch:
                snapshot_status(dev)
            if gh is not None and world > 1:
                gh = vocab_parallel.reduce_grad_hidden(gh, group).to(h.dtype)
        if CHECK_BOUNDS:
            check_status(dev)
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
    carry one 16-bit rounding more than their own.
    """
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
    h2d = hidden.reshape(-1, d)
    ids = as_label_indices(tokens, batch_size=h2d.shape[0], device=hidden.device)
    ign = _NO_IGNORE if ignore_index is None else int(ignore_index)
    lp, ent = _TiedTokenLogProbs.apply(h2d, weights, ids, ign, int(vocab_offset), vocab_size, group,
                                       grad_weights_buffer)
    return TokenLogProbs(lp.reshape(shape), ent.reshape(shape))


__all__ = ["TokenLogProbs", "token_logprobs", "tied_token_logprobs", "MAX_TOP_K"]
