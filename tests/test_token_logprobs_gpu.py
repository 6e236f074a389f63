"""Token log probabilities over logits and from the tied matrix, against 64-bit definitions.

Tolerances are bounds, element by element, with u = 2^-24. Exponentials are taken of
d = x - f, f a logit within L = 16 ln 2 below the row's max or at it. Let D1 = sum p |x - m| + L
and D2 = sum p (|x - m| + L)^2. An exponential is off by 2^-22 of itself and by 2 u |d|
from its argument; a lane adds at most n = V / 256 + 48 terms in a row (the rest
is a tree), each addition off by u of the sum. So the sum is off by
e_s = n u + 2^-22 + 2 u D1 relative, ln s by e_s + u |ln s|; a log probability by that and
u (|x - m| + |logp|); the entropy ln s - sum(2^d d) / s by e_s + (n u + 2^-22 + e_s) D1 +
2 u D2 and roundings of its two terms (``row_bounds``).
"""
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF = [torch.float16, torch.bfloat16]
IGN = -100


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def exact_rows(x, tokens):
    """(logp, entropy, p, logq, d) in 64 bits; a row of -inf only: -inf, 0, 0, -inf, 0.

    log p is (x - m) - ln sum exp(x - m): next to an m of -3.4e38 even 64 bits lose the logarithm. A row with +inf
    or NaN has NaN everywhere."""
    x = x.double()
    m = x.amax(1, keepdim=True)
    d = x - torch.where(torch.isneginf(m), torch.zeros_like(m), m)
    total = d.exp().sum(1, keepdim=True)
    logq = torch.where(total > 0, d - total.log(), torch.full_like(d, -torch.inf))
    logq = torch.where((torch.isnan(x) | torch.isposinf(x)).any(1, keepdim=True), torch.full_like(d, torch.nan), logq)
    p = logq.exp()
    h = -(p * torch.where(p > 0, logq, torch.zeros_like(logq))).sum(1)
    return logq.gather(1, tokens.clamp(min=0).unsqueeze(1)).squeeze(1), h, p, logq, torch.where(p > 0, d, torch.zeros_like(d))


def row_bounds(p, d, h):
    """(of the sum's logarithm, of the entropy), each (rows,)."""
    u, v = 2.0**-24, p.shape[1]
    lag = 16 * np.log(2)
    d1, d2 = (p * d.abs()).sum(1) + lag, (p * (d.abs() + lag) ** 2).sum(1)
    n = v / 256 + 48
    e_s = n * u + 2.0**-22 + 2 * u * d1
    ls = h + d1  # ln s = H + ln 2 u / s
    return e_s + u * ls, e_s + u * ls + (n * u + 2.0**-22 + e_s) * d1 + 2 * u * d2 + 2 * u * (ls + d1 + h)


def make_logits(rows, v, dtype, seed, scale=2.5, pitch=None, offset=0):
    g = torch.Generator().manual_seed(seed)
    pitch = pitch or v
    flat = torch.zeros(rows * pitch + offset + 16, dtype=dtype, device="cuda")
    view = flat[offset:offset + rows * pitch].view(rows, pitch)[:, :v]
    view.copy_((torch.randn(rows, v, generator=g) * scale).to(dtype))
    tokens = torch.randint(0, v, (rows,), generator=g).cuda()
    return view, tokens, g


def check_rows(r, x, tokens, ignored=None):
    lp, h, p, logq, d = exact_rows(x, tokens)
    t_ls, t_h = row_bounds(p, d, h)
    used = tokens != IGN
    spoilt = used & torch.isnan(p).any(1)
    assert torch.isnan(r.logprobs[spoilt]).all() and torch.isnan(r.entropy[spoilt]).all()
    every, used = used, used & ~spoilt
    assert torch.isneginf(r.logprobs[used]).equal(torch.isneginf(lp[used]))
    fin = used & torch.isfinite(lp)
    # x - m and the result are rounded: 2^-24 of each, |x - m| <= |logp| + ln s.
    tol = t_ls + 2.0**-24 * (2 * lp.abs() + h + (p * d.abs()).sum(1))
    assert ((r.logprobs.double() - lp).abs() <= tol)[fin].all()
    assert ((r.entropy.double() - h).abs() <= t_h)[used].all()
    assert (r.logprobs[~every] == 0).all() and (r.entropy[~every] == 0).all()
    if r.top_ids is not None:
        k = r.top_ids.shape[1]
        ids = torch.sort(x.double(), dim=1, descending=True, stable=True).indices[:, :k]
        assert r.top_ids[used].equal(ids[used])  # (+inf is the best)
        assert r.top_ids[spoilt].equal(ids[spoilt]) or torch.isnan(x).any()
        want = logq.gather(1, ids)
        off = (r.top_logprobs.double() - want).abs()
        same = torch.isneginf(want) & torch.isneginf(r.top_logprobs)
        tol = t_ls.unsqueeze(1) + 2.0**-24 * (2 * want.abs() + (h + (p * d.abs()).sum(1)).unsqueeze(1))
        assert (same | (off <= tol))[used].all()
        assert (r.top_ids[~every] == -1).all() and torch.isneginf(r.top_logprobs[~every]).all()


def check_grad(got, x, tokens, a, b):
    """Rounded once, from a p off by the sum's error, 2^-22 and 4 u (|x - m| + ln s) relative; one below 2^-126 is
    zero (ex2 without subnormal results), off by at most that."""
    _, h, p, logq, d = exact_rows(x, tokens)
    zero = torch.zeros_like(p)
    lq = torch.where(p > 0, logq, zero)
    a, b = a.double().unsqueeze(1), b.double().unsqueeze(1)
    onehot = zero.scatter(1, tokens.clamp(min=0).unsqueeze(1), 1.0)
    dead = (tokens == IGN).unsqueeze(1) | torch.isneginf(x).all(1, keepdim=True)
    want = torch.where(dead, zero, a * onehot - p * (a + b * (h.unsqueeze(1) + lq)))
    t_ls, t_h = (t.unsqueeze(1) for t in row_bounds(p, d, h))
    h = h.unsqueeze(1)
    e_lp = t_ls + 2.0**-22 * (d.abs() + lq.abs())  # of log p
    coef = a.abs() + b.abs() * (h + lq.abs())
    slack = p * (coef * (e_lp + 2.0**-21) + b.abs() * (t_h + e_lp)) + torch.where(p > 0, 2.0**-126 * coef, zero)
    fin = torch.finfo(got.dtype)
    tol = half_step(got.dtype) * want.abs() + (1 + 2.0**-7) * slack + 2.0**-23 * a.abs() * onehot
    fine = ((got.double() - want).abs() <= tol * (1 + 2.0**-7) + fin.smallest_normal * fin.eps) | torch.isnan(want)
    assert fine.all()
    assert (got[dead.squeeze(1)] == 0).all()


SHAPES = [(1, 1), (3, 2), (2, 7), (5, 100), (33, 1001), (4, 2047), (3, 2304), (300, 4099), (6, 50257), (2, 128259),
          (700, 8200),
          # 1024 rows and more of at most 8 KB: a warp a row.
          (1024, 1), (1030, 7), (1100, 130), (1025, 1001), (1027, 2047), (1033, 2049), (1026, 4096), (1024, 4104)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_rows_and_gradient(dtype, shape):
    from nimbleml_b200.losses import token_logprobs

    rows, v = shape
    x, tokens, g = make_logits(rows, v, dtype, rows * 31 + v)
    if rows > 2:
        tokens[2::5] = IGN
    a, b = torch.randn(rows, generator=g).cuda(), torch.randn(rows, generator=g).cuda()
    for k in sorted({0, 1, min(5, v), min(64, v)}):
        leaf = x.detach().requires_grad_()
        r = token_logprobs(leaf, tokens, IGN, top_k=k)
        check_rows(r, x, tokens)
        (gx,) = torch.autograd.grad((r.logprobs, r.entropy), leaf, (a, b))
        check_grad(gx, x, tokens, a, b)
    # One gradient alone; the same call gives the same bits.
    leaf = x.detach().requires_grad_()
    r2 = token_logprobs(leaf, tokens, IGN)
    (g1,) = torch.autograd.grad(r2.entropy, leaf, b, retain_graph=True)
    check_grad(g1, x, tokens, torch.zeros_like(a), b)
    (g2,) = torch.autograd.grad(r2.logprobs, leaf, a)
    check_grad(g2, x, tokens, a, torch.zeros_like(b))
    assert r2.logprobs.equal(r.logprobs) and r2.entropy.equal(r.entropy)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["pitch", "offset", "odd_pitch", "transposed", "broadcast", "three_d"])
def test_strides(dtype, layout):
    from nimbleml_b200.losses import token_logprobs

    rows, v = 12, 1003
    es = torch.empty(0, dtype=dtype).element_size()
    if layout == "pitch":
        x, tokens, g = make_logits(rows, v, dtype, 1, pitch=1008)
    elif layout == "offset":
        x, tokens, g = make_logits(rows, v, dtype, 2, pitch=1008, offset=3)
    elif layout == "odd_pitch":
        x, tokens, g = make_logits(rows, v, dtype, 3, pitch=1037, offset=1)
    elif layout == "transposed":
        x, tokens, g = make_logits(v, rows, dtype, 4)
        x, tokens = x.t(), torch.arange(rows, device="cuda")
    elif layout == "broadcast":
        x, tokens, g = make_logits(1, v, dtype, 5)
        x, tokens = x.expand(rows, v), torch.arange(rows, device="cuda")
    else:
        x, tokens, g = make_logits(rows, v, dtype, 6, pitch=1000 + 16 // es)
        x3, t3 = x.view(3, 4, v), tokens.view(3, 4)
        r = token_logprobs(x3, t3, top_k=3)
        assert r.logprobs.shape == (3, 4) and r.top_ids.shape == (3, 4, 3)
    a, b = torch.randn(rows, generator=g).cuda(), torch.randn(rows, generator=g).cuda()
    leaf = x.detach().requires_grad_()
    r = token_logprobs(leaf, tokens, top_k=7)
    check_rows(r, x, tokens)
    (gx,) = torch.autograd.grad((r.logprobs, r.entropy), leaf, (a, b))
    check_grad(gx, x, tokens, a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,v", [(3, 300), (2, 9000), (400, 9000), (1040, 300), (1030, 2043), (1025, 4091)])
def test_masks_ties_and_orders(dtype, rows, v):
    """-inf masks, a row of -inf only, the type's lowest value, ties, and rows that rise or fall to their end."""
    from nimbleml_b200.losses import token_logprobs

    kinds = {}
    x, tokens, g = make_logits(rows, v, dtype, v + rows)
    low = torch.finfo(dtype).min
    masked = x.clone()
    masked[:, torch.rand(v, generator=g).cuda() < 0.5] = -torch.inf
    masked[0] = -torch.inf
    masked[1] = -torch.inf
    masked[1, v - 2] = 1.5
    kinds["masked"] = masked
    lowest = x.clone()
    lowest[:, ::2] = low
    lowest[0] = low
    kinds["lowest"] = lowest
    kinds["constant"] = torch.zeros_like(x)
    # Far apart from each other: one weight is 1, or some equal ones share it.
    huge = x * (1e4 if dtype == torch.float16 else 1e33)
    huge[0, 3:9] = huge[0].max()
    huge[1] = -huge[1].abs()
    kinds["huge"] = huge
    # A common offset, below, above and around where references stop being products with log2 e.
    for name, off in (("offset", 3e4 if dtype == torch.float16 else 3e6), ("below", -3e4 if dtype == torch.float16 else -2e7),
                      ("around", 2.0**15 if dtype == torch.float16 else 2.0**20)):
        kinds[name] = (x.double() * 6 + off).to(dtype)
    ties = (x * 1.0).round()
    ties[:, 5] = -0.0
    kinds["ties"] = ties
    kinds["rising"] = x.sort(dim=1).values
    kinds["falling"] = x.sort(dim=1, descending=True).values
    # Strictly rising bits, so that every logit beats all before it.
    step = torch.arange(v, device="cuda", dtype=torch.float64)
    kinds["ramp"] = (step / v * 8 - 4).to(dtype).expand(rows, v).contiguous()
    a, b = torch.randn(rows, generator=g).cuda(), torch.randn(rows, generator=g).cuda()
    for name, y in kinds.items():
        leaf = y.detach().requires_grad_()
        r = token_logprobs(leaf, tokens, top_k=min(64, v))
        check_rows(r, y, tokens)
        (gx,) = torch.autograd.grad((r.logprobs, r.entropy), leaf, (a, b))
        check_grad(gx, y, tokens, a, b)


@pytest.mark.parametrize("rows", [6, 1030])
def test_nan_inf_ignored_and_bad_tokens(rows):
    from nimbleml_b200.kernels.fused_tied_crossentropy import check_status
    from nimbleml_b200.losses import token_logprobs

    n = 5000 if rows == 6 else 2000
    x, tokens, _ = make_logits(rows, n, torch.float32, 9)
    x[0] = torch.nan  # ignored: not read
    tokens[0] = IGN
    x[1, 17] = torch.inf
    x[2, n - 1] = torch.nan
    x[3, :n - 1000] = -torch.inf
    x[3, n - 500] = torch.nan
    leaf = x.detach().requires_grad_()
    r = token_logprobs(leaf, tokens, IGN, top_k=5)
    assert r.logprobs[0] == 0 and r.entropy[0] == 0
    assert torch.isnan(r.logprobs[1:4]).all() and torch.isnan(r.entropy[1:4]).all()
    assert torch.isfinite(r.logprobs[4:]).all()
    assert r.top_ids[1, 0] == 17
    (gx,) = torch.autograd.grad(r.logprobs.sum(), leaf)
    assert (gx[0] == 0).all() and torch.isfinite(gx[4:]).all()
    check_status(x.device)
    tokens[5] = n
    leaf = x.detach().requires_grad_()
    r = token_logprobs(leaf, tokens, IGN)
    assert torch.isnan(r.logprobs[5]) and torch.isfinite(r.logprobs[4])
    (gx,) = torch.autograd.grad(r.logprobs[4:].sum(), leaf)
    assert (gx[5] == 0).all()
    with pytest.raises(ValueError):
        check_status(x.device)
    # No rows at all.
    r = token_logprobs(x[:0], tokens[:0], top_k=3)
    assert r.logprobs.shape == (0,) and r.top_ids.shape == (0, 3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_row_with_a_nan(dtype):
    """A NaN among classes that are all ruled out reaches the results and the gradient; a row of -inf only has none."""
    from nimbleml_b200.losses import token_logprobs

    x = torch.full((3, 700), -torch.inf, dtype=dtype, device="cuda")
    x[1, 333] = torch.nan
    x[2, 5] = 1.0
    tokens = torch.tensor([4, 7, 5], device="cuda")
    r = token_logprobs(x.requires_grad_(True), tokens)
    assert torch.isneginf(r.logprobs[0]) and torch.isnan(r.logprobs[1]) and torch.isnan(r.entropy[1])
    (g,) = torch.autograd.grad((r.logprobs + r.entropy).sum(), x)
    assert (g[0] == 0).all() and torch.isnan(g[1]).all() and (g[2] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [1, 20, 64])
def test_top_k_crowded(dtype, k):
    """Rows whose alternatives are hard to tell apart, over more segments than a block lists: equal ones, rising ones
    within a part in 300, masked ones, and NaN with few numbers among them (fewer than k in one row)."""
    from nimbleml_b200.losses import token_logprobs

    v = 70001
    g = torch.Generator().manual_seed(k)
    x = torch.full((7, v), 0.75)
    x[1] = 4.0 + torch.arange(v) / v / 80
    x[2] = -x[1]
    x[3] = -torch.inf
    x[4] = torch.where(torch.rand(v, generator=g) < 0.5, 0.75, -torch.inf)
    x[5] = torch.nan
    x[5, torch.randperm(v, generator=g)[:40]] = torch.randn(40, generator=g)
    x[6] = torch.where(torch.rand(v, generator=g) < 0.9, torch.nan, -1.0)
    x = x.to(dtype).cuda()
    r = token_logprobs(x, torch.zeros(7, dtype=torch.int64, device="cuda"), top_k=k)
    for i in range(7):
        row = x[i].double()
        at = (~torch.isnan(row)).nonzero().squeeze(1)
        order = at[torch.sort(row[at], descending=True, stable=True).indices[:k]]
        want = torch.full((k,), -1, device="cuda")
        want[:len(order)] = order
        assert r.top_ids[i].equal(want), i


def test_one_row_without_a_batch():
    from nimbleml_b200.losses import token_logprobs

    x, _, _ = make_logits(1, 500, torch.float16, 3)
    r = token_logprobs(x[0], torch.tensor(7), top_k=4)
    q = token_logprobs(x, torch.tensor([7]).cuda(), top_k=4)
    assert r.logprobs.shape == () and r.top_ids.shape == (4,)
    assert r.logprobs == q.logprobs[0] and r.top_ids.equal(q.top_ids[0])
    y = x[0].detach().requires_grad_()
    (g,) = torch.autograd.grad(token_logprobs(y, 7).logprobs, y, create_graph=False)
    assert g.shape == (500,)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(token_logprobs(y, 7).logprobs, y, create_graph=True)


def test_gradient_against_differences():
    """Central differences of the log probability and the entropy in x: off by h^2 / 6 |f'''| <= h^2 and by the values' own
    error (below 2e-6 for these rows) over h."""
    from nimbleml_b200.losses import token_logprobs

    x, tokens, g = make_logits(2, 19, torch.float32, 11, scale=1.0)
    a, b = torch.tensor([0.7, -1.1]).cuda(), torch.tensor([0.4, 0.9]).cuda()
    leaf = x.detach().requires_grad_()
    r = token_logprobs(leaf, tokens)
    (gx,) = torch.autograd.grad((r.logprobs, r.entropy), leaf, (a, b))
    h = 2.0**-6
    for j in range(19):
        f = []
        for s in (1, -1):
            y = x.clone()
            y[:, j] += s * h
            q = token_logprobs(y, tokens)
            f.append((a * q.logprobs + b * q.entropy).double())
        num = (f[0] - f[1]) / (2 * h)
        assert ((num - gx[:, j].double()).abs() <= 2 * h * h * 2 + 4e-6 / h).all()


def test_refusals_on_the_gpu():
    from nimbleml_b200.losses import tied_token_logprobs, token_logprobs

    x, tokens, _ = make_logits(3, 70, torch.float32, 1)
    for k in (-1, 65, 71):
        with pytest.raises(ValueError, match="top_k"):
            token_logprobs(x, tokens, top_k=k)
    with pytest.raises(ValueError, match="label count"):
        token_logprobs(x, tokens[:2])
    with pytest.raises(ValueError, match="dtype"):
        token_logprobs(x.double(), tokens)
    h, w = torch.zeros(3, 16, device="cuda").half(), torch.zeros(5, 16, device="cuda").half()
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        tied_token_logprobs(h.float(), w, tokens)
    with pytest.raises(ValueError, match="multiple of 8"):
        tied_token_logprobs(h[:, :12], w[:, :12], tokens)
    with pytest.raises(ValueError, match="d_model"):
        tied_token_logprobs(h, w[:, :8], tokens)
    with pytest.raises(ValueError, match="inside the vocabulary"):
        tied_token_logprobs(h, w, tokens, vocab_offset=3, vocab_size=7)
    with pytest.raises(ValueError, match="grad_weights_buffer"):
        tied_token_logprobs(h, w, tokens, grad_weights_buffer=torch.zeros(5, 16).half().cuda())


# ------------------------------------------------------------------- the tied form
def make_tied(n, d, v, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(n, d, generator=g).to(dtype).cuda()
    w = (torch.randn(v, d, generator=g) / d**0.5).to(dtype).cuda()
    tokens = torch.randint(0, v, (n,), generator=g).cuda()
    return h, w, tokens, g


def logit_error(h, w):
    """The logits are fp32 sums of d products: off by at most d 2^-23 of the sum of magnitudes, in any order."""
    return (h.double().abs() @ w.double().abs().t()).amax(1) * (h.shape[1] + 16) * 2.0**-23


def check_tied(r, h, w, tokens):
    used = tokens != IGN
    x = h.double() @ w.double().t()
    mag = logit_error(h, w)
    lp, ent, p, logq, d = exact_rows(x, tokens)
    t_ls, t_h = row_bounds(p, d, ent)
    # The epilogue's d is x log2 e - m log2 e: 2^-23 of the logits' size more.
    big = 2.0**-22 * x.abs().amax(1)
    assert ((r.logprobs.double() - lp).abs() <= t_ls + 2 * mag + 2 * big + 2.0**-23 * lp.abs())[used].all()
    spread = (p * (logq.abs() + ent.unsqueeze(1))).sum(1)  # |dH / dx| summed
    assert ((r.entropy.double() - ent).abs() <= t_h + 2 * (mag + big) * (1 + spread))[used].all()


def check_tied_grads(gh, gw, h, w, tokens, a, b, base=None):
    """G is rounded to 16 bits once (fp16: scaled by a power of two so that its largest bound lies in (2^14, 2^15], its
    smallest step is then at most 2^-24 2^-14 of that bound), then summed in fp32 and rounded to the result's type."""
    x = h.double() @ w.double().t()
    _, ent, p, logq, d = exact_rows(x, tokens)
    live = (tokens != IGN).unsqueeze(1)
    a, b = a.double().unsqueeze(1), b.double().unsqueeze(1)
    zero = torch.zeros_like(p)
    onehot = zero.scatter(1, tokens.clamp(min=0).unsqueeze(1), 1.0)
    t_ls, t_h = (t.unsqueeze(1) for t in row_bounds(p, d, ent))
    ent = ent.unsqueeze(1)
    big_g = torch.where(live, a * onehot - p * (a + b * (ent + logq)), zero)
    mag = logit_error(h, w).unsqueeze(1) + 2.0**-22 * x.abs().amax(1, keepdim=True)
    e_lp = t_ls + 4 * mag + 2.0**-22 * (d.abs() + logq.abs())
    spread = (p * (logq.abs() + ent)).sum(1, keepdim=True)
    slack = p * ((a.abs() + b.abs() * (ent + logq.abs())) * (e_lp + 2.0**-21) + b.abs() * (t_h + 2 * mag * (1 + spread) + e_lp))
    under = 0.0
    if h.dtype == torch.float16:
        under = 2.0**-24 * 2.0**-14 * torch.where(live, a.abs() + b.abs() * (ent + 0.37), zero[:, :1]).amax()
    err = torch.where(live, half_step(h.dtype) * big_g.abs() + (1 + 2.0**-6) * slack + under + 2.0**-22 * a.abs() * onehot, zero)
    for got, g, other, e in ((gh, big_g, w.double(), err), (gw, big_g.t(), h.double(), err.t())):
        if got is None:
            continue
        want = g @ other
        if got is gw and base is not None:
            want = want + base.double()
        fin = torch.finfo(got.dtype)
        tol = half_step(got.dtype) * want.abs() + e @ other.abs() + (g.shape[1] + 16) * 2.0**-23 * (g.abs() @ other.abs())
        off = (got.double() - want).abs()
        assert (off <= tol * (1 + 2.0**-6) + fin.smallest_normal * fin.eps).all(), float((off / (tol + 1e-300)).max())


TIED = [(1, 8, 1), (1, 8, 3), (2, 64, 5), (7, 64, 257), (129, 136, 1000), (300, 72, 5003), (513, 256, 256), (1, 1024, 20011), (16, 520, 4801),
        (17, 64, 33), (32, 128, 19001), (33, 72, 600), (128, 64, 3000), (260, 320, 6000)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("shape", TIED)
def test_tied(dtype, shape):
    from nimbleml_b200.losses import tied_token_logprobs

    n, d, v = shape
    h, w, tokens, g = make_tied(n, d, v, dtype, n * 7 + v)
    if n > 2:
        tokens[1::4] = IGN
    a, b = torch.randn(n, generator=g).cuda(), torch.randn(n, generator=g).cuda()
    hl, wl = h.requires_grad_(), w.requires_grad_()
    r = tied_token_logprobs(hl, wl, tokens, IGN)
    check_tied(r, h.detach(), w.detach(), tokens)
    assert (r.logprobs[tokens == IGN] == 0).all() and (r.entropy[tokens == IGN] == 0).all()
    gh, gw = torch.autograd.grad((r.logprobs, r.entropy), (hl, wl), (a, b), retain_graph=True)
    check_tied_grads(gh, gw, h.detach(), w.detach(), tokens, a, b)
    assert (gh[tokens == IGN] == 0).all()
    # The same again, bit for bit, and each gradient alone.
    gh2, gw2 = torch.autograd.grad((r.logprobs, r.entropy), (hl, wl), (a, b), retain_graph=True)
    assert gh2.equal(gh) and gw2.equal(gw)
    (gh3,) = torch.autograd.grad((r.logprobs, r.entropy), (hl,), (a, b), retain_graph=True)
    assert gh3.equal(gh)
    (gh4,) = torch.autograd.grad(r.entropy, (hl,), b, retain_graph=True)
    check_tied_grads(gh4, None, h.detach(), w.detach(), tokens, torch.zeros_like(a), b)
    (gw4,) = torch.autograd.grad(r.logprobs, (wl,), a)
    check_tied_grads(None, gw4, h.detach(), w.detach(), tokens, a, torch.zeros_like(b))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("shape", [(1024, 72, 700), (1153, 264, 2100), (2049, 64, 1300), (600, 2056, 900)])
@pytest.mark.parametrize("buffer", [False, True])
def test_tied_many_tokens(dtype, shape, buffer, monkeypatch):
    """Enough tokens for every kind of tile; grad_hidden in several runs, over one slab and over several."""
    import nimbleml_b200.losses.logprobs as mod

    n, d, v = shape
    h, w, tokens, g = make_tied(n, d, v, dtype, n + v)
    tokens[::7] = IGN
    a, b = torch.randn(n, generator=g).cuda(), torch.randn(n, generator=g).cuda()
    base = torch.randn(v, d, generator=g).cuda() if buffer else None
    for slab in (0, 512 * n * 2):  # at most 512 columns
        monkeypatch.setattr(mod, "SLAB_BYTES", slab)
        buf = base.clone() if buffer else None
        hl, wl = h.detach().requires_grad_(), w.detach().requires_grad_(not buffer)
        r = mod.tied_token_logprobs(hl, wl, tokens, IGN, grad_weights_buffer=buf)
        check_tied(r, h, w, tokens)
        grads = torch.autograd.grad((r.logprobs, r.entropy), (hl,) if buffer else (hl, wl), (a, b))
        check_tied_grads(grads[0], buf if buffer else grads[1], h, w, tokens, a, b, base)
        assert (grads[0][tokens == IGN] == 0).all()


@pytest.mark.parametrize("size", [1e-12, 1e-6, 1.0, 1e6])
def test_tied_fp16_upstream_sizes(size):
    """Upstream gradients of any size keep the 16-bit G in range; the fp32 weight grad shows it."""
    from nimbleml_b200.losses import tied_token_logprobs

    h, w, tokens, g = make_tied(64, 64, 3001, torch.float16, 3)
    a, b = (size * torch.randn(64, generator=g)).cuda(), (size * torch.randn(64, generator=g)).cuda()
    w32 = w.float().requires_grad_()
    r = tied_token_logprobs(h, w32, tokens)
    (gw,) = torch.autograd.grad((r.logprobs, r.entropy), (w32,), (a, b))
    assert gw.dtype == torch.float32
    check_tied_grads(None, gw, h, w, tokens, a, b)


@pytest.mark.parametrize("dtype", HALF)
def test_tied_slabs_buffer_and_layouts(dtype, monkeypatch):
    from nimbleml_b200.losses import tied_token_logprobs
    import nimbleml_b200.losses.logprobs as mod

    monkeypatch.setattr(mod, "SLAB_BYTES", 1)  # 256 columns a slab
    h, w, tokens, g = make_tied(70, 64, 1500, dtype, 21)
    a, b = torch.randn(70, generator=g).cuda(), torch.randn(70, generator=g).cuda()
    buf = torch.randn(1500, 64, generator=g).cuda()
    base = buf.clone()
    # Hidden rows in (7, 10) with a storage offset off the 16-byte grid.
    store = torch.zeros(70 * 64 + 1, dtype=dtype, device="cuda")
    hv = store[1:].view(7, 10, 64)
    hv.copy_(h.view(7, 10, 64))
    hl = hv.detach().requires_grad_()
    r = tied_token_logprobs(hl, w, tokens.view(7, 10), grad_weights_buffer=buf)
    assert r.logprobs.shape == (7, 10)
    (gh,) = torch.autograd.grad((r.logprobs, r.entropy), (hl,), (a.view(7, 10), b.view(7, 10)))
    check_tied_grads(gh.view(70, 64), buf, h, w, tokens, a, b, base=base)


def test_tied_shards_and_all_ignored():
    """Two vocabulary shards merge into the whole; partial hidden grads add up."""
    import nimbleml_b200.losses.logprobs as mod

    h, w, tokens, g = make_tied(50, 64, 1001, torch.bfloat16, 5)
    tokens[7] = IGN
    cut = 600
    s0 = mod.shard_logprob_stats(h, w[:cut].contiguous(), tokens, 0)
    s1 = mod.shard_logprob_stats(h, w[cut:].contiguous(), tokens, cut)
    lp, ent, lse = mod.combine_logprob_stats(torch.stack([s0, s1]), tokens, 1001, IGN).unbind(0)
    check_tied(mod.TokenLogProbs(lp, ent), h, w, tokens)
    a, b = torch.randn(50, generator=g).cuda(), torch.randn(50, generator=g).cuda()
    parts, rows = [], []
    for lo, hi in ((0, cut), (cut, 1001)):
        gh = torch.empty(50, 64, device="cuda")
        gw = torch.empty(hi - lo, 64, dtype=torch.bfloat16, device="cuda")
        mod.shard_logprob_backward(a, b, h, w[lo:hi].contiguous(), tokens, lse, ent, vocab_offset=lo, vocab_size=1001,
                                   ignore_index=IGN, grad_hidden=gh, grad_weights=gw)
        parts.append(gh)
        rows.append(gw)
    check_tied_grads(parts[0] + parts[1], torch.cat(rows), h, w, tokens, a, b)
    tokens[:] = IGN
    from nimbleml_b200.losses import tied_token_logprobs

    hl, wl = h.requires_grad_(), w.requires_grad_()
    r = tied_token_logprobs(hl, wl, tokens, IGN)
    gh, gw = torch.autograd.grad((r.logprobs, r.entropy), (hl, wl), (a, b))
    assert (r.logprobs == 0).all() and (gh == 0).all() and (gw == 0).all()
    r = tied_token_logprobs(hl[:0], wl, tokens[:0])
    (gw,) = torch.autograd.grad(r.logprobs.sum(), (wl,))
    assert r.logprobs.shape == (0,) and (gw == 0).all()


def test_tied_bad_token():
    from nimbleml_b200.kernels.fused_tied_crossentropy import check_status
    from nimbleml_b200.losses import tied_token_logprobs

    h, w, tokens, g = make_tied(40, 64, 300, torch.float16, 8)
    check_status(h.device)
    tokens[3] = 300
    tokens[4] = -7
    hl = h.requires_grad_()
    r = tied_token_logprobs(hl, w, tokens)
    assert torch.isnan(r.logprobs[3:5]).all() and torch.isfinite(r.logprobs[5:]).all()
    with pytest.raises(ValueError):  # at the latest a later call of the path raises by itself
        check_status(h.device)
    (gh,) = torch.autograd.grad((r.logprobs, r.entropy), (hl,), (torch.ones(40).cuda(), torch.ones(40).cuda()))
    assert (gh[3:5] == 0).all() and torch.isfinite(gh).all()
    check_status(h.device)


def test_tied_odd_calls():
    """One row without a batch, no rows, rows that repeat or lie apart, weights of other types and layouts."""
    from nimbleml_b200.losses import tied_token_logprobs

    h, w, tokens, g = make_tied(6, 64, 300, torch.bfloat16, 12)
    a, b = torch.randn(6, generator=g).cuda(), torch.randn(6, generator=g).cuda()
    whole = tied_token_logprobs(h, w, tokens)
    # One row.
    hl = h[2].detach().requires_grad_()
    one = tied_token_logprobs(hl, w, int(tokens[2]))
    assert one.logprobs.shape == () and one.logprobs == whole.logprobs[2] and one.entropy == whole.entropy[2]
    (gh,) = torch.autograd.grad(one.logprobs + one.entropy, hl)
    assert gh.shape == (64,)
    check_tied_grads(gh.view(1, 64), None, h[2:3], w, tokens[2:3], torch.ones(1).cuda(), torch.ones(1).cuda())
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(tied_token_logprobs(hl, w, 5).logprobs, hl, create_graph=True)
    # No rows.
    hl, wl = h[:0].detach().requires_grad_(), w.detach().requires_grad_()
    none = tied_token_logprobs(hl, wl, tokens[:0])
    assert none.logprobs.shape == (0,)
    gh, gw = torch.autograd.grad(none.logprobs.sum() + none.entropy.sum(), (hl, wl))
    assert gh.shape == (0, 64) and (gw == 0).all() and gw.shape == w.shape
    # One row for every token.
    hl = h[1].detach().requires_grad_()
    same = tied_token_logprobs(hl.expand(6, 64), w, tokens)
    rows = h[1:2].expand(6, 64).contiguous()
    assert same.logprobs.equal(tied_token_logprobs(rows, w, tokens).logprobs)
    # Rows apart, weights transposed in memory, fp32 masters: their gradient is fp32.
    wide = torch.zeros(6, 100, dtype=h.dtype, device="cuda")
    wide[:, 8:72] = h
    hl, wl = wide[:, 8:72].detach().requires_grad_(), w.t().contiguous().t().float().requires_grad_()
    assert not hl.is_contiguous() and not wl.is_contiguous()
    r = tied_token_logprobs(hl, wl, tokens)
    assert r.logprobs.equal(whole.logprobs) and r.entropy.equal(whole.entropy)
    gh, gw = torch.autograd.grad((r.logprobs, r.entropy), (hl, wl), (a, b))
    assert gw.dtype == torch.float32 and gh.dtype == h.dtype
    check_tied_grads(gh, gw, h, w, tokens, a, b)
    # Upstream gradients that repeat, and only one of the two results used.
    hl = h.detach().requires_grad_()
    r = tied_token_logprobs(hl.view(2, 3, 64), w, tokens.view(2, 3))
    (gh,) = torch.autograd.grad(r.entropy.sum(), hl)
    check_tied_grads(gh, None, h, w, tokens, torch.zeros(6).cuda(), torch.ones(6).cuda())


@pytest.mark.parametrize("grad", [False, True])
def test_tied_errors_reach_a_later_call(grad):
    """A bad token and a wait that ran out are raised by the next call, without a copy of the status word."""
    from nimbleml_b200._native_loader import STATUS_WAIT_TIMEOUT
    from nimbleml_b200.kernels import fused_tied_crossentropy as k
    from nimbleml_b200.losses import tied_token_logprobs

    for n in (5, 40):  # both forms of the forward
        h, w, tokens, g = make_tied(n, 64, 300, torch.bfloat16, n)
        dev = h.device
        k.check_status(dev)
        k.poll_status(dev)
        want = tied_token_logprobs(h, w, tokens).logprobs
        bad = tokens.clone()
        bad[2] = 300
        hl = h.detach().requires_grad_(grad)
        tied_token_logprobs(hl, w, bad)
        torch.cuda.synchronize()
        with pytest.raises(ValueError, match="out of range"):
            tied_token_logprobs(hl, w, tokens)
        assert tied_token_logprobs(hl, w, tokens).logprobs.equal(want)  # reported once
        k.status_word(dev).fill_(STATUS_WAIT_TIMEOUT)  # as a product before the merge leaves it
        tied_token_logprobs(hl, w, tokens)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="timed out"):
            tied_token_logprobs(hl, w, tokens)
        r = tied_token_logprobs(hl, w, tokens)
        assert r.logprobs.equal(want) and k.check_status(dev) == 0
        if grad:
            r = tied_token_logprobs(hl, w, bad)
            torch.cuda.synchronize()
            with pytest.raises(ValueError, match="out of range"):
                torch.autograd.grad(r.logprobs.nan_to_num().sum(), hl)
            assert k.check_status(dev) == 0
            # What a backward reports, the next forward finds.
            r = tied_token_logprobs(hl, w, tokens)
            torch.autograd.grad(r.logprobs.sum(), hl)
            k.status_word(dev).fill_(STATUS_WAIT_TIMEOUT)
            tied_token_logprobs(hl, w, tokens)
            torch.cuda.synchronize()
            with pytest.raises(RuntimeError, match="timed out"):
                k.poll_status(dev)
            assert k.check_status(dev) == 0


@pytest.mark.parametrize("grad", [False, True])
def test_tied_checked_calls(grad, monkeypatch):
    """With bounds checks on, the call itself raises."""
    import nimbleml_b200.losses.logprobs as mod

    monkeypatch.setattr(mod, "CHECK_BOUNDS", True)
    h, w, tokens, g = make_tied(40, 64, 300, torch.float16, 6)
    hl = h.requires_grad_(grad)
    r = mod.tied_token_logprobs(hl, w, tokens)
    if grad:
        (gh,) = torch.autograd.grad(r.entropy.sum(), hl, retain_graph=True)
        mod.status_word(h.device).fill_(1 << 1)
        with pytest.raises((RuntimeError, ValueError)):
            torch.autograd.grad(r.entropy.sum(), hl)
    tokens[1] = 300
    with pytest.raises(ValueError, match="out of range"):
        mod.tied_token_logprobs(hl, w, tokens)
    mod.check_status(h.device)


@pytest.mark.parametrize("tied", [False, True])
def test_captured_and_on_another_stream(tied):
    """Forward and backward in a CUDA graph, replayed on new values, equal the eager calls bit for bit."""
    from nimbleml_b200.losses import tied_token_logprobs, token_logprobs

    h, w, tokens, g = make_tied(33, 64, 700, torch.bfloat16, 2)
    up = (torch.randn(33, generator=g).cuda(), torch.randn(33, generator=g).cuda())

    def work(h, w):
        if tied:
            r = tied_token_logprobs(h, w, tokens)
        else:
            r = token_logprobs(h @ w.t(), tokens)
        return (r.logprobs.detach(), r.entropy.detach(), *torch.autograd.grad((r.logprobs, r.entropy), (h, w), up))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        hs, ws = h.clone().requires_grad_(), w.clone().requires_grad_()
        on_side = work(hs, ws)
    torch.cuda.current_stream().wait_stream(side)
    del hs, ws
    hc, wc = h.clone().requires_grad_(), w.clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work(hc, wc)
    for turn in range(2):
        if turn:
            with torch.no_grad():
                hc.copy_(-h)
                wc.mul_(0.5)
        graph.replay()
        want = work(hc.detach().clone().requires_grad_(), wc.detach().clone().requires_grad_())
        for x, y in zip(got, want):
            assert x.equal(y)
        if not turn:
            for x, y in zip(on_side, want):
                assert x.equal(y)


FIRST_CALL = """
import torch
from nimbleml_b200.losses import tied_token_logprobs, token_logprobs

g = torch.Generator().manual_seed(1)
h, w = torch.randn(4, 64, generator=g).cuda().half(), torch.randn(300, 64, generator=g).cuda().half()
x, tokens = torch.randn(4, 300, generator=g).cuda(), torch.tensor([1, 2, 3, 299], device="cuda")
side = torch.cuda.Stream()
for call in (lambda: token_logprobs(x, tokens), lambda: tied_token_logprobs(h, w, tokens)):
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=side):
            call()
    except RuntimeError as e:
        assert "once on this device" in str(e), e
    else:
        raise SystemExit("a first call was captured")
token_logprobs(x, tokens)  # readies the device for both
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=side):
    r = tied_token_logprobs(h, w, tokens)
graph.replay()
want = tied_token_logprobs(h, w, tokens)
assert r.logprobs.equal(want.logprobs) and r.entropy.equal(want.entropy)
print("ok")
"""


def test_first_call_in_a_capture_is_refused():
    run = subprocess.run([sys.executable, "-c", FIRST_CALL], capture_output=True, text=True, timeout=300,
                         cwd=Path(__file__).resolve().parents[1])
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout + run.stderr


def check_each_row(gh, gw, h, w, tokens, a, b):
    """As check_tied_grads, but every row of grad_hidden against its own size: whatever the other rows' upstream
    gradients are, a row's bound B_i = |a| + |b| (H + 1/e) is brought to 2^6 or more in fp16, whose smallest half step is 2^-25:
    2^-31 B_i an element of G. In dE a row that was raised by 2^k meets hidden 2^-k, off by half a smallest step, 2^-25."""
    x = h.double() @ w.double().t()
    _, ent, p, logq, d = exact_rows(x, tokens)
    live = (tokens != IGN).unsqueeze(1)
    a, b = a.double().unsqueeze(1), b.double().unsqueeze(1)
    zero = torch.zeros_like(p)
    onehot = zero.scatter(1, tokens.clamp(min=0).unsqueeze(1), 1.0)
    t_ls, t_h = (t.unsqueeze(1) for t in row_bounds(p, d, ent))
    ent = ent.unsqueeze(1)
    big_g = torch.where(live, a * onehot - p * (a + b * (ent + logq)), zero)
    mag = logit_error(h, w).unsqueeze(1) + 2.0**-22 * x.abs().amax(1, keepdim=True)
    e_lp = t_ls + 4 * mag + 2.0**-22 * (d.abs() + logq.abs())
    spread = (p * (logq.abs() + ent)).sum(1, keepdim=True)
    slack = p * ((a.abs() + b.abs() * (ent + logq.abs())) * (e_lp + 2.0**-21) + b.abs() * (t_h + 2 * mag * (1 + spread) + e_lp))
    bound = torch.where(live, a.abs() + b.abs() * (ent + 0.37), zero[:, :1])
    under = 2.0**-31 * bound * (1 + 2.0**-10) if h.dtype == torch.float16 else 0.0
    err = torch.where(live, half_step(h.dtype) * big_g.abs() + (1 + 2.0**-6) * slack + under + 2.0**-22 * a.abs() * onehot, zero)
    top = float(bound.max())
    raised = torch.where(bound > 0, (top / bound.clamp(min=2.0**-140)).clamp(min=1.0) * 2.0**-7, zero[:, :1])  # 2^k at most
    e_h = 2.0**-25 * torch.where(raised > 1, raised, zero[:, :1]) if h.dtype == torch.float16 else zero[:, :1]
    for got, want, tol in (
            (gh, big_g @ w.double(), err @ w.double().abs() + (p.shape[1] + 16) * 2.0**-23 * (big_g.abs() @ w.double().abs())),
            (gw, big_g.t() @ h.double(), err.t() @ h.double().abs() + (big_g.abs() + err).t() @ e_h.expand(h.shape) +
             (h.shape[0] + 16) * 2.0**-23 * (big_g.t().abs() @ h.double().abs()))):
        fin = torch.finfo(got.dtype)
        tol = tol + half_step(got.dtype) * want.abs()
        off = (got.double() - want).abs()
        assert (off <= tol * (1 + 2.0**-6) + fin.smallest_normal * fin.eps).all(), float((off / (tol + 1e-300)).max())


# (tokens, d, vocabulary): the split grad_hidden product, one run of it, several slabs, ragged edges.
UNEVEN = [(64, 64, 20011), (5, 72, 300), (40, 64, 1500), (260, 320, 6000)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("shape", UNEVEN)
@pytest.mark.parametrize("ratio", [1e2, 1e4, 1e6, 1e9, 1e30])
def test_tied_rows_beside_a_large_one(dtype, shape, ratio, monkeypatch):
    """One upstream gradient far above the others leaves the others' gradients their precision."""
    import nimbleml_b200.losses.logprobs as mod

    n, d, v = shape
    if n == 40:
        monkeypatch.setattr(mod, "SLAB_BYTES", 1)  # 256 columns a slab
    h, w, tokens, g = make_tied(n, d, v, dtype, n + d)
    a, b = torch.randn(n, generator=g).cuda(), 0.1 * torch.randn(n, generator=g).cuda()
    # Sizes from the largest down; the results are fp32 or scaled so that fp16 holds them.
    size = 1.0 / ratio if dtype == torch.float16 else 1.0
    a, b = a * size, b * size
    a[n // 2] = size * ratio
    if ratio == 1e6:  # every size between
        a = a * torch.logspace(0, 6, n, device="cuda")
        a[n // 2] = size * ratio
    tokens[1] = IGN
    h32 = h.float().to(dtype).requires_grad_()
    w32 = w.float().requires_grad_()
    r = mod.tied_token_logprobs(h32, w32, tokens, IGN)
    gh, gw = torch.autograd.grad((r.logprobs, r.entropy), (h32, w32), (a, b))
    gh32 = torch.empty(n, d, device="cuda")  # the same in fp32, as the shards' partial sums are kept
    gw32 = torch.empty(v, d, device="cuda")
    lse = torch.logsumexp(h.double() @ w.double().t(), 1).float()
    mod.shard_logprob_backward(a, b, h, w, tokens, lse, r.entropy.detach(), ignore_index=IGN, grad_hidden=gh32,
                               grad_weights=gw32)
    check_each_row(gh, gw, h, w, tokens, a, b)
    check_each_row(gh32, gw32, h, w, tokens, a, b)
    assert (gh[1] == 0).all() and (gh32[1] == 0).all()


@pytest.mark.parametrize("spoilt", [float("inf"), float("nan")])
def test_tied_rows_beside_a_spoilt_one(spoilt):
    """An infinite or NaN upstream gradient spoils its own row of grad_hidden; the others keep their precision."""
    from nimbleml_b200.losses import tied_token_logprobs

    h, w, tokens, g = make_tied(50, 64, 9000, torch.float16, 4)
    a, b = 1e-3 * torch.randn(50, generator=g).cuda(), 1e-4 * torch.randn(50, generator=g).cuda()
    keep = torch.arange(50, device="cuda") != 7
    for x in (a, b):
        bad = x.clone()
        bad[7] = spoilt
        up = (bad, b) if x is a else (a, bad)
        hl = h.detach().requires_grad_()
        r = tied_token_logprobs(hl, w, tokens)
        (gh,) = torch.autograd.grad((r.logprobs, r.entropy), (hl,), up)
        assert not torch.isfinite(gh[7]).all() and torch.isfinite(gh[keep]).all()
        # The others as without it, in bits (their largest row sets the factor).
        none = tokens.clone()
        none[7] = IGN
        hl = h.detach().requires_grad_()
        r = tied_token_logprobs(hl, w, none, IGN)
        (want,) = torch.autograd.grad((r.logprobs, r.entropy), (hl,), (a, b))
        assert gh[keep].equal(want[keep])


def test_checked_calls_over_logits(monkeypatch):
    """With bounds checks on, an eager call raises by itself; a captured one, which cannot wait, is recorded."""
    import nimbleml_b200.losses.logprobs as mod

    monkeypatch.setattr(mod, "CHECK_BOUNDS", True)
    x, tokens, _ = make_logits(6, 700, torch.float16, 5)
    want = mod.token_logprobs(x, tokens, top_k=3)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = mod.token_logprobs(x, tokens, top_k=3)
    graph.replay()
    assert all(a.equal(b) for a, b in zip(got, want))
    tokens[2] = 700
    with pytest.raises(ValueError, match="out of range"):
        mod.token_logprobs(x, tokens)
    mod.check_status(x.device)


# (tokens, d, vocabulary, columns a slab (0: the library's), slabs, runs of grad_hidden's product in each).
SLABS_AND_RUNS = [(300, 72, 5003, 2048, 3, 4), (300, 72, 4196, 2048, 3, 4), (70, 264, 3000, 1024, 3, 2), (513, 520, 4100, 1536, 3, 3),
                  (300, 72, 4097, 4096, 2, 8), (2700, 64, 50000, 0, 2, 6)]


def slab_workspace(n, d, cols, slabs, runs, dtype):
    """Bytes that the backward asks for with this many slabs and runs: G, the runs' sums, the row coefficients, the
    scale, and for fp16 the rows' factors and hidden copy, each from a multiple of 256."""
    up = lambda x: -(-x // 256) * 256  # noqa: E731
    total = up(2 * n * cols) + (up(4 * n * d * runs) if slabs > 1 or runs > 1 else 0) + up(16 * n) + up(4)
    return total + (up(4 * n) + up(2 * n * d) if dtype == torch.float16 else 0)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("shape", SLABS_AND_RUNS)
@pytest.mark.parametrize("buffer", [False, True])
def test_tied_several_slabs_in_several_runs(dtype, shape, buffer, monkeypatch):
    """The runs' partial grad_hidden goes from slab to slab; a last slab of 100 columns (two 64-column blocks) or one leaves
    runs without any."""
    import nimbleml_b200.losses.logprobs as mod
    from nimbleml_b200.embedding_grad import _TORCH_TO_NIMBLE

    n, d, v, cols, slabs, runs = shape
    slab_bytes = 2 * n * cols
    cols = cols or 25088  # half of 50000 columns in whole tiles
    assert -(-v // cols) == slabs
    assert mod.native.tied_logprobs_backward_workspace_size(n, d, v, _TORCH_TO_NIMBLE[dtype], slab_bytes) == slab_workspace(
        n, d, cols, slabs, runs, dtype)
    monkeypatch.setattr(mod, "SLAB_BYTES", slab_bytes)
    h, w, tokens, g = make_tied(n, d, v, dtype, n + v)
    tokens[::7] = IGN
    tokens[1] = v - 1  # in the last slab
    a, b = torch.randn(n, generator=g).cuda(), torch.randn(n, generator=g).cuda()
    base = torch.randn(v, d, generator=g).cuda() if buffer else None
    buf = base.clone() if buffer else None
    hl, wl = h.detach().requires_grad_(), w.detach().requires_grad_(not buffer)
    r = mod.tied_token_logprobs(hl, wl, tokens, IGN, grad_weights_buffer=buf)
    grads = torch.autograd.grad((r.logprobs, r.entropy), (hl,) if buffer else (hl, wl), (a, b))
    check_tied_grads(grads[0], buf if buffer else grads[1], h, w, tokens, a, b, base)
    assert (grads[0][tokens == IGN] == 0).all()


def test_a_step_of_the_tied_matrix_counts_as_a_write():
    """The backward recomputes the logits from the tied matrix: after a step it is refused, not taken from the new one."""
    from nimbleml_b200.gpt_head import TiedEmbedding

    h, w, tokens, g = make_tied(9, 64, 300, torch.float16, 5)
    emb = TiedEmbedding(w.float(), 300)
    hl = h.requires_grad_()
    r = emb.token_logprobs(hl, tokens)
    emb.grad.fill_(1.0)
    emb.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.logprobs.sum().backward()
    emb.token_logprobs(hl, tokens).logprobs.sum().backward()
    with torch.inference_mode():
        inside = TiedEmbedding(w.float(), 300)
        inside.grad.fill_(1.0)
        inside.step()
        assert (inside.master < w.float()).any()
