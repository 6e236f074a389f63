"""Layer norm against its definition in 64 bits.

Bounds, element by element (u = 2^-24): a row's mean is a sum of d terms, at most
64 of them in a row, off by e_m = 80 u mean|x|; the centred values by that and a
rounding; the variance by 80 u of itself and twice e_m sqrt(var). The results
follow, each rounded once to its type. A column sum over N rows adds at most N in a row.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0**-24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def exact(x, gamma, beta, eps, gy):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    c = x - mean
    var = c.square().mean(1, keepdim=True)
    r = 1 / (var + eps).sqrt()
    xh = c * r
    y = xh * gamma.double() + (0 if beta is None else beta.double())
    gy = gy.double()
    gg = gy * gamma.double()
    m1, m2 = gg.mean(1, keepdim=True), (gg * xh).mean(1, keepdim=True)
    gx = r * (gg - m1 - xh * m2)
    return y, gx, (gy * xh).sum(0), gy.sum(0), xh, r, m1, m2, mean, var


def check(x, gamma, beta, eps, gy, y, gx, ggam, gbet):
    n, d = x.shape
    y64, gx64, gg64, gb64, xh, r, m1, m2, mean, var = exact(x, gamma, beta, eps, gy)
    e_m = 80 * U * x.double().abs().mean(1, keepdim=True) + 2 * U * mean.abs()
    # Relative error of rstd, then of xh (absolute).
    e_v = (80 * U * var + 2 * e_m * var.sqrt() + e_m * e_m) / (var + eps) + 8 * U
    e_xh = xh.abs() * (e_v + 4 * U) + r * (e_m + 2 * U * (x.double() - mean).abs())
    e_xh = torch.minimum(e_xh, xh.abs() + r * e_m * 2 + 1)
    g64, gam = gy.double(), gamma.double()
    tiny = torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps
    tol = half_step(y.dtype) * y64.abs() + e_xh * gam.abs() + 8 * U * (xh * gam).abs() + 4 * U * y64.abs()
    assert ((y.double() - y64).abs() <= tol * 1.02 + tiny).all()
    if gx is None:
        return
    gg = g64 * gam
    e_m1 = 80 * U * gg.abs().mean(1, keepdim=True)
    e_m2 = 80 * U * (gg * xh).abs().mean(1, keepdim=True) + (gg.abs() * e_xh).mean(1, keepdim=True)
    tol = half_step(gx.dtype) * gx64.abs() + gx64.abs() * (e_v + 4 * U) + r * (
        e_m1 + xh.abs() * e_m2 + e_xh * (m2.abs() + e_m2) + 8 * U * (gg.abs() + m1.abs() + (xh * m2).abs()))
    assert ((gx.double() - gx64).abs() <= tol * 1.02 + tiny).all()
    tol = (n + 40) * U * (g64 * xh).abs().sum(0) + (g64.abs() * e_xh).sum(0) + half_step(ggam.dtype) * gg64.abs()
    assert ((ggam.double() - gg64).abs() <= tol * 1.02 + tiny).all()
    if gbet is not None:
        tol = (n + 40) * U * g64.abs().sum(0) + half_step(gbet.dtype) * gb64.abs()
        assert ((gbet.double() - gb64).abs() <= tol * 1.02 + tiny).all()


def run(x, gamma, beta, gy, eps=1e-5):
    from nimbleml_b200.norm import layer_norm

    xl = x.detach().requires_grad_()
    gl = gamma.detach().requires_grad_()
    bl = None if beta is None else beta.detach().requires_grad_()
    y = layer_norm(xl, gl, bl, eps)
    leaves = [xl, gl] + ([] if bl is None else [bl])
    grads = torch.autograd.grad(y, leaves, gy)
    with torch.no_grad():
        plain = layer_norm(x, gamma, beta, eps)
        assert ((plain == y) | (torch.isnan(plain) & torch.isnan(y))).all()
    return (y.detach(), *grads, *([None] if bl is None else []))


def make(n, d, dtype, pdtype, seed, mean=0.3):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, d, generator=g) * 1.5 + mean).to(dtype).cuda()
    gamma = (1 + 0.2 * torch.randn(d, generator=g)).to(pdtype).cuda()
    beta = (0.3 * torch.randn(d, generator=g)).to(pdtype).cuda()
    gy = torch.randn(n, d, generator=g).to(dtype).cuda()
    return x, gamma, beta, gy


DIMS = [1, 2, 8, 33, 256, 257, 264, 512, 513, 1000, 1024, 1032, 2048, 2049, 4096, 4104, 5000, 8191, 8192]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("n", [1, 5, 700])
def test_against_64_bits(dtype, d, n):
    pdtype = dtype if d % 3 == 0 else torch.float32
    x, gamma, beta, gy = make(n, d, dtype, pdtype, n * d)
    got = run(x, gamma, beta, gy)
    check(x, gamma, beta, 1e-5, gy, *got)
    again = run(x, gamma, beta, gy)
    for a, b in zip(got, again):
        assert a.equal(b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows_and_small_ones(dtype):
    x, gamma, beta, gy = make(9001, 264, dtype, torch.float32, 4)
    check(x, gamma, beta, 1e-5, gy, *run(x, gamma, beta, gy))
    # No bias; parameters of a third type; constant rows; a mean far above the spread.
    x, gamma, _, gy = make(13, 1000, dtype, torch.bfloat16, 5)
    check(x, gamma, None, 1e-5, gy, *run(x, gamma, None, gy))
    x[2] = 3.0
    x[5] = 0.0
    check(x, gamma, None, 1e-3, gy, *run(x, gamma, None, gy, eps=1e-3))
    x, gamma, beta, gy = make(9, 1024, dtype, torch.float32, 6, mean=100.0)
    check(x, gamma, beta, 1e-5, gy, *run(x, gamma, beta, gy))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["pitch", "odd", "transposed", "broadcast_grad", "three_d"])
def test_layouts(dtype, layout):
    x, gamma, beta, gy = make(24, 520, dtype, torch.float32, 8)
    if layout == "pitch":
        wide = torch.zeros(24, 600, dtype=dtype, device="cuda")
        wide[:, 16:536] = x
        x = wide[:, 16:536]
    elif layout == "odd":
        wide = torch.zeros(24 * 600, dtype=dtype, device="cuda")[3:3 + 24 * 521].view(24, 521)
        wide[:, :520] = x
        x = wide[:, :520]
    elif layout == "transposed":
        x = x.t().contiguous().t()
    elif layout == "broadcast_grad":
        gy = gy[:1].expand(24, 520)
    else:
        y3 = run(x.view(2, 12, 520), gamma, beta, gy.view(2, 12, 520))
        assert y3[0].shape == (2, 12, 520) and y3[1].shape == (2, 12, 520)
        check(x, gamma, beta, 1e-5, gy, y3[0].view(24, 520), y3[1].view(24, 520), y3[2], y3[3])
        return
    check(x, gamma, beta, 1e-5, gy, *run(x, gamma, beta, gy))


def test_rows_are_left_alone_and_empty():
    """NaN in one row stays there; rows behind the batch are not written."""
    from nimbleml_b200.norm import LayerNorm, layer_norm

    x, gamma, beta, gy = make(6, 300, torch.float16, torch.float32, 9)
    clean = run(x, gamma, beta, gy)
    y2 = x.clone()
    y2[4, 7] = torch.nan
    dirty = run(y2, gamma, beta, gy)
    keep = [0, 1, 2, 3, 5]
    assert dirty[0][keep].equal(clean[0][keep]) and dirty[1][keep].equal(clean[1][keep])
    assert torch.isnan(dirty[0][4]).all()
    got = run(x[:0], gamma, beta, gy[:0])
    assert got[0].shape == (0, 300) and (got[2] == 0).all() and (got[3] == 0).all()
    layer = LayerNorm(300, device="cuda")
    assert torch.allclose(layer(x).float(), torch.nn.functional.layer_norm(x.float(), (300,)), atol=4e-3)
    with pytest.raises(ValueError, match="gamma"):
        layer_norm(x, gamma[:10])
    with pytest.raises(ValueError, match="8192"):
        layer_norm(torch.zeros(2, 8200, device="cuda"), torch.ones(8200, device="cuda"))
    with pytest.raises(ValueError, match="is on"):
        layer_norm(x, gamma.cpu())


def test_gradient_against_differences():
    """Central differences in fp32: off by 1e-3 h^2-terms and 1e-6 / h from the values' rounding."""
    from nimbleml_b200.norm import layer_norm

    x, gamma, beta, gy = make(2, 11, torch.float32, torch.float32, 10)
    _, gx, gg, gb = run(x, gamma, beta, gy)
    h = 2.0**-7

    def f(x, gamma, beta):
        return (layer_norm(x, gamma, beta).double() * gy.double())

    for j in range(11):
        d = torch.zeros_like(x)
        d[:, j] = h
        num = (f(x + d, gamma, beta) - f(x - d, gamma, beta)).sum(1) / (2 * h)
        assert ((num - gx[:, j].double()).abs() <= 20 * h * h + 2e-5 / h * 0.5).all()
        e = torch.zeros_like(gamma)
        e[j] = h
        num = (f(x, gamma + e, beta) - f(x, gamma - e, beta)).sum() / (2 * h)
        assert abs(float(num - gg[j])) <= 2e-5 / h
        num = (f(x, gamma, beta + e) - f(x, gamma, beta - e)).sum() / (2 * h)
        assert abs(float(num - gb[j])) <= 2e-5 / h


def test_captured_and_on_another_stream():
    x, gamma, beta, gy = make(40, 1024, torch.bfloat16, torch.float32, 12)
    want = run(x, gamma, beta, gy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = run(x, gamma, beta, gy)
    torch.cuda.current_stream().wait_stream(side)

    def once():
        from nimbleml_b200.norm import layer_norm

        leaves = [t.detach().requires_grad_() for t in (x, gamma, beta)]
        y = layer_norm(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, gy))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once()
    graph.replay()
    for a, b, c in zip(got, want, on_side):
        assert a.equal(b) and c.equal(b)
    with torch.no_grad():
        x.mul_(-2)
    graph.replay()
    for a, b in zip(got, run(x, gamma, beta, gy)):
        assert a.equal(b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d,off", [(1, 520, 0), (7, 520, 0), (13, 33, 0), (7, 520, 1), (15, 4104, 0), (33, 8191, 0), (3, 2048, 0)])
def test_nothing_behind_the_outputs_is_written(dtype, n, d, off):
    """Rows go in pairs and eights: odd counts and widths, with vectors and (off the 16-byte grid) without."""
    from nimbleml_b200._native_loader import native
    from nimbleml_b200.embedding_grad import _TORCH_TO_NIMBLE, _stream_ptr

    x, gamma, beta, gy = make(n, d, dtype, torch.float32, n + d)
    want = run(x, gamma, beta, gy)

    def room(size, dt):  # `size` elements behind `off`, with a sentinel on both sides
        buf = torch.full((off + size + 64 * 1024,), 7.0, device="cuda").to(dt)
        return buf, buf[off:off + size]

    bufs = {k: room(size, dt) for k, size, dt in (("y", n * d, dtype), ("mean", n, torch.float32), ("rstd", n, torch.float32),
                                                  ("gx", n * d, dtype), ("gg", d, torch.float32), ("gb", d, torch.float32))}
    at = {k: part.data_ptr() for k, (_, part) in bufs.items()}
    need = native.layernorm_backward_workspace_size(n, d)
    ws = torch.full((need + 4096,), 7, dtype=torch.uint8, device="cuda")
    t, s = _TORCH_TO_NIMBLE[dtype], _stream_ptr(x.device)
    f32 = _TORCH_TO_NIMBLE[torch.float32]
    native.call("nimble_layernorm_forward", x.data_ptr(), d, gamma.data_ptr(), beta.data_ptr(), n, d, 1e-5, t, f32, at["y"],
                at["mean"], at["rstd"], s)
    native.call("nimble_layernorm_backward", gy.data_ptr(), x.data_ptr(), d, gamma.data_ptr(), at["mean"], at["rstd"], n, d, t, f32,
                at["gx"], at["gg"], at["gb"], ws.data_ptr(), need, s)
    y, gx, gg, gb = (bufs[k][1] for k in ("y", "gx", "gg", "gb"))
    if off == 0:
        assert y.equal(want[0].view(-1)) and gx.equal(want[1].view(-1)) and gg.equal(want[2]) and gb.equal(want[3])
    else:  # element by element: sums in another order
        check(x, gamma, beta, 1e-5, gy, y.view(n, d), gx.view(n, d), gg, gb)
    for buf, part in bufs.values():
        assert (buf[:off] == 7).all() and (buf[off + part.numel():] == 7).all()
    assert (ws[need:] == 7).all()
