"""Host logic of the vocab-sharded tied log probabilities on CPU ranks (gloo, world_size 2).

The kernels' calls are replaced by plain 64-bit statistics and gradients of each shard, so what is tested is what the
ranks exchange: the order of the gathered statistics, the sum of the partial grad_hidden and its type.
"""
import os

import torch
import torch.distributed as dist
import torch.multiprocessing as mp

N, D, V, IGN = 21, 16, 57, -100


def make():
    g = torch.Generator().manual_seed(4)
    h = torch.randn(N, D, generator=g).half()
    w = torch.randn(V, D, generator=g).half()
    tokens = torch.randint(0, V, (N,), generator=g)
    tokens[::5] = IGN
    return h, w, tokens, torch.randn(N, generator=g), torch.randn(N, generator=g)


def logit_grad(x, lse, ent, tokens, offset, a, b):
    """Gradient of the logits of classes offset, offset + 1, ... of which x holds the values."""
    logq = x - lse.unsqueeze(1)
    g = -logq.exp() * (a.unsqueeze(1) + b.unsqueeze(1) * (ent.unsqueeze(1) + logq))
    mine = (tokens >= offset) & (tokens < offset + x.shape[1])
    g[mine, tokens[mine] - offset] += a[mine]
    g[tokens == IGN] = 0
    return g


def shard_stats(h, w, tokens, offset):
    x = h.double() @ w.double().t()
    m = x.amax(1)
    d = (x - m.unsqueeze(1)) / torch.log(torch.tensor(2.0, dtype=torch.float64))
    mine = (tokens >= offset) & (tokens < offset + len(w))
    target = torch.where(mine, x.gather(1, (tokens - offset).clamp(0, len(w) - 1).unsqueeze(1)).squeeze(1), 0.0)
    return torch.stack([m, (2**d).sum(1), (d * 2**d).sum(1), target])


def combine(stats, tokens, vocab_size, ignore_index):
    assert stats.shape == (2, 4, N) and vocab_size == V and stats.is_contiguous()
    ln2 = torch.log(torch.tensor(2.0, dtype=torch.float64))
    m = stats[:, 0].amax(0)
    d = (stats[:, 0] - m) / ln2
    s = (stats[:, 1] * 2**d).sum(0)
    u = ((stats[:, 2] + stats[:, 1] * d) * 2**d).sum(0)
    lse = m + s.log()
    out = torch.stack([stats[:, 3].sum(0) - lse, s.log() - ln2 * u / s, lse])
    out[:2, tokens == ignore_index] = 0
    return out


def shard_backward(g_lp, g_ent, h, w, tokens, lse, ent, *, vocab_offset, vocab_size, ignore_index, grad_hidden,
                   grad_weights, accumulate):
    g = logit_grad(h.double() @ w.double().t(), lse, ent, tokens, vocab_offset, g_lp.double(), g_ent.double())
    grad_hidden.copy_(g @ w.double())
    if accumulate:
        grad_weights.add_(g.t() @ h.double())
    else:
        grad_weights.copy_(g.t() @ h.double())


def worker(rank, world, port, q):
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        import contextlib

        import nimbleml_b200.losses.logprobs as mod
        from nimbleml_b200.vocab_parallel import shard_range

        mod.shard_logprob_stats, mod.combine_logprob_stats = shard_stats, combine
        mod.shard_logprob_backward = shard_backward
        mod._on = lambda device: contextlib.nullcontext()
        torch.cuda.current_device = lambda: None
        torch.cuda.is_current_stream_capturing = lambda: True  # no status copies
        h, w, tokens, a, b = make()
        off, rows = shard_range(V, rank, world)
        buffer = torch.ones(rows, D) if rank else None  # each rank has its own way to take grad_weights
        hl, wl = h.requires_grad_(), w[off:off + rows].clone().requires_grad_()
        lp, ent = mod._ShardTokenLogProbs.apply(hl, wl, tokens, IGN, off, V, dist.group.WORLD, buffer)
        torch.autograd.backward((lp, ent), (a.double(), b.double()))
        gw = buffer - 1 if rank else wl.grad
        assert (wl.grad is None) == bool(rank) and hl.grad.dtype == torch.float16
        q.put((rank, lp.detach().numpy(), ent.detach().numpy(), hl.grad.double().numpy(), gw.double().numpy()))
    finally:
        dist.destroy_process_group()


def test_two_ranks_exchange():
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = 31500 + os.getpid() % 2000
    procs = [ctx.Process(target=worker, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    results = sorted((q.get(timeout=120) for _ in procs), key=lambda r: r[0])
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    h, w, tokens, a, b = make()
    x = h.double() @ w.double().t()
    lse = torch.logsumexp(x, 1)
    logq = x - lse.unsqueeze(1)
    used = tokens != IGN
    lp = torch.where(used, logq.gather(1, tokens.clamp(min=0).unsqueeze(1)).squeeze(1), 0.0)
    ent = -(logq.exp() * logq).sum(1)
    g = logit_grad(x, lse, ent, tokens, 0, a.double(), b.double())
    from nimbleml_b200.vocab_parallel import shard_range

    cut = shard_range(V, 0, 2)[1]
    gh = [g[:, :cut] @ w[:cut].double(), g[:, cut:] @ w[cut:].double()]
    # Partial grad_hidden in bf16, their sum in bf16, then fp16: half a step each.
    tol = 2.0**-8 * (gh[0].abs() + gh[1].abs()) * (1 + 2.0**-8) + (2.0**-8 + 2.0**-10) * (gh[0] + gh[1]).abs() + 2.0**-24
    gw = g.t() @ h.double()
    for rank, got_lp, got_ent, got_gh, got_gw in results:
        assert torch.allclose(torch.from_numpy(got_lp), lp, rtol=0, atol=1e-9)
        assert torch.allclose(torch.from_numpy(got_ent), torch.where(used, ent, 0.0), rtol=0, atol=1e-9)
        assert ((torch.from_numpy(got_gh) - gh[0] - gh[1]).abs() <= tol).all()
        want = gw[cut:] if rank else gw[:cut]
        # fp32 (added to ones) or fp16.
        t = 2.0**-23 * (1 + want.abs()) if rank else 2.0**-11 * want.abs() + 2.0**-25
        assert ((torch.from_numpy(got_gw) - want).abs() <= t).all()
