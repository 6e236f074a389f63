"""AdamW over many tensors: 32-bit moments bit for bit as the single-tensor step, 8-bit moments bit for bit as
their definition, and the weights against 64 bits."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

SIZES = [0, 1, 3, 7, 8, 127, 128, 129, 255, 1000, 8191, 8192, 8193, 20011]
HYPER = dict(learning_rate=2e-2, beta1=0.9, beta2=0.99, epsilon=1e-8, weight_decay=0.1)
MAX, TINY = 448.0, 2.0**-9


def views(sizes, dtype, gap, fill=0.0):
    """Tensors cut from one buffer, `gap` elements apart, and the buffer."""
    at, out = gap, []
    buf = torch.full((sum(sizes) + gap * (len(sizes) + 1),), fill, device="cuda").to(dtype)
    for n in sizes:
        out.append(buf[at:at + n])
        at += n + gap
    return out, buf


def make(sizes, gdtype, cdtype, gap, seed):
    g = torch.Generator().manual_seed(seed)
    ps, pbuf = views(sizes, torch.float32, gap, 7.0)
    gs, _ = views(sizes, gdtype, gap)
    cs, cbuf = views(sizes, cdtype, gap, 7.0) if cdtype else ([None] * len(sizes), None)
    for p, gr in zip(ps, gs):
        p.copy_(torch.randn(p.shape, generator=g))
        gr.copy_(torch.randn(gr.shape, generator=g) * 10 ** float(torch.empty(()).uniform_(-4, 0, generator=g)))
    return ps, gs, cs, pbuf, cbuf, g


def gaps_untouched(buf, sizes, gap):
    keep = torch.ones(buf.numel(), dtype=torch.bool)
    at = gap
    for n in sizes:
        keep[at:at + n] = False
        at += n + gap
    return (buf.cpu()[keep] == 7).all()


@pytest.mark.parametrize("gdtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cdtype", [None, torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gap", [16, 1])
def test_32_bits_as_the_single_step(gdtype, cdtype, gap):
    from nimbleml_b200.embedding_grad import _TORCH_TO_NIMBLE, _stream_ptr, adamw_step_many, native

    sizes = [16 * ((n + 15) // 16) if gap == 16 else n for n in SIZES]
    ps, gs, cs, pbuf, cbuf, _ = make(sizes, gdtype, cdtype, gap, 5)
    ms, vs = [torch.zeros_like(p) for p in ps], [torch.zeros_like(p) for p in ps]
    ref = [(p.clone(), torch.zeros_like(p), torch.zeros_like(p), None if c is None else torch.zeros_like(c))
           for p, c in zip(ps, cs)]
    start = [p.double() for p in ps]
    m64, v64 = [torch.zeros_like(p) for p in start], [torch.zeros_like(p) for p in start]
    for step in (1, 2, 3):
        adamw_step_many(ps, gs, ms, vs, step=step, copies=cs, **HYPER)
        for (p, m, v, c), g in zip(ref, gs):
            h = HYPER
            native.call("nimble_adamw_step", p.data_ptr(), g.contiguous().data_ptr(), _TORCH_TO_NIMBLE[g.dtype], m.data_ptr(),
                        v.data_ptr(), p.numel(), h["learning_rate"], h["beta1"], h["beta2"], 1 - h["beta1"]**step,
                        1 - h["beta2"]**step, h["epsilon"], h["weight_decay"], c.data_ptr() if c is not None else None,
                        _TORCH_TO_NIMBLE[c.dtype] if c is not None else 0, _stream_ptr(p.device))
        for i, g in enumerate(gs):
            g64 = g.double()
            m64[i] = 0.9 * m64[i] + 0.1 * g64
            v64[i] = 0.99 * v64[i] + 0.01 * g64 * g64
            start[i] = start[i] * (1 - 2e-3) - 2e-2 * (m64[i] / (1 - 0.9**step)) / ((v64[i] / (1 - 0.99**step)).sqrt() + 1e-8)
    for p, m, v, c, (rp, rm, rv, rc), w64 in zip(ps, ms, vs, cs, ref, start):
        if gap == 16:  # whole eights on 16-byte boundaries: the single step's vector kernel
            assert p.equal(rp) and m.equal(rm) and v.equal(rv)
            assert c is None or c.equal(rc)
        else:  # its scalar kernel rounds a moment's two products in another order
            assert c is None or c.equal(p.to(c.dtype))
        # Three steps of about 12 roundings each: 40 2^-24 of the weight and of the steps taken (< 0.1).
        assert ((p.double() - w64).abs() <= 40 * 2.0**-24 * (w64.abs() + 0.2)).all()
    assert gaps_untouched(pbuf, sizes, gap)
    assert cbuf is None or gaps_untouched(cbuf, sizes, gap)


# The definition of the 8-bit step in fp32 operations, each rounded on its own.
def encode(x, root):
    n = x.numel()
    b = torch.zeros(-(-n // 128) * 128)
    b[:n] = x
    b = b.view(-1, 128)
    top = b.abs().amax(1, keepdim=True)
    live = top >= 2.0**-100
    up = torch.where(live, torch.div(torch.full_like(top, MAX), top), torch.zeros_like(top))
    y = b * up
    if root:
        y = torch.where((b > 0) & (y < TINY), torch.full_like(y, TINY), y)
    scale = torch.where(live, top * (1.0 / MAX), torch.zeros_like(top))
    return y.clamp(-MAX, MAX).to(torch.float8_e4m3fn).flatten()[:n], scale.flatten()


def decode(codes, scales):
    n = codes.numel()
    return codes.float() * scales.repeat_interleave(128)[:n]


def step8(w, g, mq, vq, step, h):
    f = torch.float32
    sc = {k: torch.tensor(v, dtype=torch.float64).to(f) for k, v in dict(
        b1=h["beta1"], omb1=1 - h["beta1"], b2=h["beta2"], omb2=1 - h["beta2"],
        decay=1 - h["learning_rate"] * h["weight_decay"], c1=h["learning_rate"] / (1 - h["beta1"]**step),
        c2=1 / math.sqrt(1 - h["beta2"]**step), eps=h["epsilon"]).items()}
    m, r = decode(*mq), decode(*vq)
    m = m * sc["b1"] + g * sc["omb1"]
    # NumPy's root is the rounded one; torch's on the CPU may be a last bit off.
    r = torch.from_numpy(np.sqrt(((r * r) * sc["b2"] + (g * g) * sc["omb2"]).numpy()))
    w = w * sc["decay"] - (m * sc["c1"]) / (r * sc["c2"] + sc["eps"])
    return w, encode(m, False), encode(r, True)


def same_codes(a, b):
    return a.view(torch.uint8).equal(b.view(torch.uint8))


@pytest.mark.parametrize("gdtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cdtype", [None, torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gap", [16, 1])
def test_8_bits_as_defined(gdtype, cdtype, gap):
    from nimbleml_b200.embedding_grad import QuantizedMoment, adamw_step_many, dequantize_moment

    sizes = [16 * ((n + 15) // 16) if gap == 16 else n for n in SIZES]
    ps, gs, cs, pbuf, cbuf, g = make(sizes, gdtype, cdtype, gap, 6)
    cut, codebuf = views(sizes, torch.float32, gap)
    code = [torch.zeros(codebuf.numel(), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)]
    place, at = [], gap
    for n in sizes:
        place.append(slice(at, at + n))
        at += n + gap
    blocks = [-(-n // 128) for n in sizes]
    ms = [QuantizedMoment(code[0][s], torch.zeros(b, device="cuda")) for s, b in zip(place, blocks)]
    vs = [QuantizedMoment(code[1][s], torch.zeros(b, device="cuda")) for s, b in zip(place, blocks)]
    ref = [(p.cpu(), (m.codes.cpu(), m.scales.cpu()), (v.codes.cpu(), v.scales.cpu())) for p, m, v in zip(ps, ms, vs)]
    for step in (1, 2, 3, 4):
        for gr in gs:  # small entries, and some that are zero
            gr.mul_(torch.rand(gr.shape, generator=g).cuda().round() * 0.7)
        adamw_step_many(ps, gs, ms, vs, step=step, copies=cs, **HYPER)
        ref = [step8(w, gr.float().cpu(), m, v, step, HYPER) for (w, m, v), gr in zip(ref, gs)]
        for p, m, v, c, (w, rm, rv) in zip(ps, ms, vs, cs, ref):
            assert same_codes(m.codes.cpu(), rm[0]) and m.scales.cpu().equal(rm[1])
            assert same_codes(v.codes.cpu(), rv[0]) and v.scales.cpu().equal(rv[1])
            # A step's quotient is off by 2 ulp, its terms by a rounding each, the weight by one a step: 4 steps of at
            # most 3 lr (|m| / root is below 1 / sqrt(1 - beta2) = 10 sqrt(bc2) / bc1 at worst; these stay below 3).
            assert ((p.cpu() - w).abs() <= step * (8 * 2.0**-24 * 3 * HYPER["learning_rate"] + 2.0**-23 * (w.abs() + 0.1))).all()
            assert c is None or c.equal(p.to(c.dtype))
            assert dequantize_moment(*m).cpu().equal(decode(*rm))
            assert dequantize_moment(*v, root=True).cpu().equal(decode(*rv) * decode(*rv))
    assert gaps_untouched(pbuf, sizes, gap)
    assert cbuf is None or gaps_untouched(cbuf, sizes, gap)
    inside = torch.zeros(code[0].numel(), dtype=torch.bool)
    for s in place:
        inside[s] = True
    for c in code:
        assert (c.view(torch.uint8).cpu()[~inside] == 0).all()


@pytest.mark.parametrize("n", [1, 127, 128, 129, 5000])
def test_quantised_values(n):
    """A code is off by at most half a step of e4m3, 2^-4 of the value, or 2^-10 of the block's scale below 2^-6 of
    it; a positive root never becomes zero; blocks of zeros stay zeros."""
    from nimbleml_b200.embedding_grad import dequantize_moment, quantize_moment

    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, generator=g) * torch.exp(4 * torch.randn(n, generator=g))
    x[: n // 3] = 0.0
    q = quantize_moment(x.cuda())
    assert same_codes(q.codes.cpu(), encode(x, False)[0])
    back = dequantize_moment(*q).cpu()
    scale = q.scales.cpu().repeat_interleave(128)[:n]
    assert ((back - x).abs() <= torch.maximum(x.abs() * 2.0**-4, scale * 2.0**-10) * (1 + 2.0**-20)).all()
    v = x.abs()
    q = quantize_moment(v.cuda(), root=True)
    r = dequantize_moment(*q).cpu()
    assert (r[v > 0] > 0).all() and (r[v == 0] == 0).all()
    z = quantize_moment(torch.zeros(n, device="cuda"))
    assert (dequantize_moment(*z) == 0).all() and (z.scales == 0).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_many_tensors_none_and_twice(bits):
    """Over 400 tensors go in two launches; None leaves a tensor; one listed twice is updated twice in order."""
    from nimbleml_b200.embedding_grad import AdamW

    ps = [torch.full((5 + i % 3,), 1.0 + i, device="cuda") for i in range(405)]
    opt = AdamW(ps, learning_rate=0.5, state_bits=bits)
    for i, p in enumerate(ps):
        p.grad = None if i == 403 else torch.full_like(p, 0.25)
    before = ps[403].clone()
    opt.step()
    assert ps[403].equal(before)
    lone = AdamW([torch.full((5,), 1.0, device="cuda")], learning_rate=0.5, state_bits=bits)
    lone.params[0].grad = torch.full((5,), 0.25, device="cuda")
    lone.step()
    assert ps[0].equal(lone.params[0])
    assert all(torch.isfinite(p).all() for p in ps) and not ps[404].eq(405.0).any()
    p = torch.ones(300, device="cuda")
    p.grad = torch.ones(300, device="cuda")
    twice = AdamW([p, p], state_bits=bits, learning_rate=0.1, weight_decay=0.0)
    twice.step()
    # m / (sqrt v + eps) is 1 in each of the two updates, to roundings of 2^-24 and, with fp32 moments, to that of
    # 1 - 0.999 taken in fp32 as the single step takes it: 0.00099998713 for 0.001, whose root is 6.5e-6 less than one,
    # so 2 x 0.1 x 6.5e-6 = 1.3e-6 and a few 2^-24.
    assert ((p - 0.8).abs() <= 1.3e-6 + 8 * 2.0**-24).all()
    m, v = twice.moments()
    assert ((m[0] - 0.1).abs() <= 0.1 * 2.0**-4).all() and ((v[0] - 0.001).abs() <= 0.001 * 2.0**-2).all()


def test_8_bit_root_follows_its_gradients():
    """With a constant gradient the root of the second moment decays and grows as the exact one (block scales)."""
    from nimbleml_b200.embedding_grad import AdamW

    p = torch.zeros(256, device="cuda")
    opt = AdamW([p], learning_rate=1e-3, beta2=0.99, state_bits=8)
    want = 0.0
    for size, steps in ((1.0, 50), (1e-3, 200)):
        for _ in range(steps):
            p.grad = torch.full((256,), size, device="cuda")
            opt.step()
            want = 0.99 * want + 0.01 * size * size
        v = opt.moments()[1][0]
        # Equal elements share the block's maximum: 448 exactly, so only fp32 roundings add up (steps x 8).
        assert ((v.double() / want - 1).abs() <= 250 * 8 * 2.0**-24).all()


def test_non_finite_gradients_stay_in_their_block():
    from nimbleml_b200.embedding_grad import AdamW

    for bits in (32, 8):
        p, q = torch.ones(512, device="cuda"), torch.ones(512, device="cuda")
        opt = AdamW([p, q], state_bits=bits)
        p.grad, q.grad = torch.full((512,), 0.5, device="cuda"), torch.full((512,), 0.5, device="cuda")
        p.grad[200] = torch.nan
        opt.step()
        p.grad[200] = 0.5
        opt.step()
        bad = torch.isnan(p)
        assert bad[200] and not bad[:128].any() and not bad[256:].any() and not torch.isnan(q).any()
        if bits == 32:
            assert int(bad.sum()) == 1


def test_optimizer_step_keeps_the_bits_of_single_steps():
    """AdamW.step equals a loop of nimble_adamw_step over its tensors bit for bit, odd sizes and offsets included."""
    from nimbleml_b200.embedding_grad import _TORCH_TO_NIMBLE, AdamW, _stream_ptr, native

    for cdtype in (None, torch.float16, torch.bfloat16):
        for gap in (16, 1):
            ps, gs, cs, _, _, _ = make(SIZES[1:], torch.bfloat16, cdtype, gap, 3)
            ps2, _, cs2, _, _, _ = make(SIZES[1:], torch.bfloat16, cdtype, gap, 3)
            ref = [(p, torch.zeros_like(p), torch.zeros_like(p), c) for p, c in zip(ps2, cs2)]
            opt = AdamW(ps, learning_rate=1e-2, copies=cs)
            for step in (1, 2):
                for p, g in zip(ps, gs):
                    p.grad = g.float() if step == 1 else g.float() * 0.3
                opt.step()
                for (p, m, v, c), q in zip(ref, ps):
                    native.call("nimble_adamw_step", p.data_ptr(), q.grad.data_ptr(), _TORCH_TO_NIMBLE[q.grad.dtype],
                                m.data_ptr(), v.data_ptr(), p.numel(), 1e-2, 0.9, 0.999, 1 - 0.9**step,
                                1 - 0.999**step, 1e-8, 0.01, c.data_ptr() if c is not None else None,
                                _TORCH_TO_NIMBLE[c.dtype] if c is not None else 0, _stream_ptr(p.device))
            for (p, m, v, c), q, mm, vv, cc in zip(ref, ps, opt.m, opt.v, cs):
                assert p.equal(q) and m.equal(mm) and v.equal(vv) and (c is None or c.equal(cc))


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_and_on_another_stream(bits):
    from nimbleml_b200.embedding_grad import adamw_step_many, quantize_moment

    sizes = [300, 9000]
    ps, gs, cs, _, _, _ = make(sizes, torch.float16, torch.bfloat16, 1, 9)

    def state():
        p = [x.clone() for x in ps]
        z = [torch.zeros_like(x) for x in ps]
        if bits == 8:
            return p, [quantize_moment(x) for x in z], [quantize_moment(x) for x in z]
        return p, z, [x.clone() for x in z]

    a, b = state(), state()
    for _ in range(2):
        adamw_step_many(a[0], gs, a[1], a[2], step=7, **HYPER)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        adamw_step_many(b[0], gs, b[1], b[2], step=7, **HYPER)
    graph.replay()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(a[0], b[0]):
        assert x.equal(y)


def test_gradients_with_strides():
    from nimbleml_b200.embedding_grad import adamw_step_many

    w = torch.ones(64, 48, device="cuda")
    g = torch.randn(48, 64, device="cuda").t()
    one = [x.clone() for x in (w, torch.zeros_like(w), torch.zeros_like(w))]
    two = [x.clone() for x in one]
    adamw_step_many([one[0]], [g], [one[1]], [one[2]], step=1)
    adamw_step_many([two[0]], [g.contiguous()], [two[1]], [two[2]], step=1)
    assert one[0].equal(two[0])
    with pytest.raises(ValueError, match="contiguous float32"):
        adamw_step_many([w.t()], [g], [one[1]], [one[2]], step=1)
    with pytest.raises(ValueError, match="elements"):
        adamw_step_many([w], [g[:3]], [one[1]], [one[2]], step=1)
    with pytest.raises(ValueError, match="moments"):
        adamw_step_many([w], [g], [one[1]], [one[2][:3]], step=1)


@pytest.mark.parametrize("size", [5, 301, 16])
@pytest.mark.parametrize("fault", ["short", "long", "strided", "type", "moment", "late"])
def test_a_refused_step_changes_nothing(size, fault):
    """Copies and moments that do not fit, whatever the weights' sizes: ValueError before anything is launched."""
    from nimbleml_b200.embedding_grad import AdamW

    ps = [torch.full((7,), 2.0, device="cuda"), torch.full((size,), 1.0, device="cuda"), torch.full((24,), 3.0, device="cuda")]
    for p in ps:
        p.grad = torch.full_like(p, 0.5)
    bad = {"short": torch.zeros(size - 1, device="cuda"), "long": torch.zeros(size + 1, device="cuda"),
           "strided": torch.zeros(2 * size, device="cuda")[::2], "type": torch.zeros(size, dtype=torch.float64, device="cuda")}
    opt = AdamW(ps, copies=[None, bad.get(fault), None])
    if fault == "moment":
        opt.v[1] = torch.zeros(size + 8, device="cuda")
    elif fault == "late":  # the last of three, behind one that steps alone
        opt.copies[2] = torch.zeros(23, device="cuda")
    with pytest.raises(ValueError, match="moments must have" if fault == "moment" else "a copy must be"):
        opt.step()
    torch.cuda.synchronize()
    assert opt.t == 0 and all((p == x).all() for p, x in zip(ps, (2.0, 1.0, 3.0)))
    assert all((m == 0).all() for m in opt.m) and all((v == 0).all() for v in opt.v)
    if fault != "moment":
        assert all(c is None or (c == 0).all() for c in opt.copies)
        opt.copies = [None] * 3
        opt.step()
        assert opt.t == 1 and all((p < x).all() for p, x in zip(ps, (2.0, 1.0, 3.0)))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_refused_list_changes_nothing(bits):
    """A tensor that is listed twice makes two launches: the second one's checks come before the first one too."""
    from nimbleml_b200.embedding_grad import adamw_step_many, quantize_moment

    p = torch.ones(130, device="cuda")
    z = torch.zeros(130, device="cuda")
    m = [quantize_moment(z) if bits == 8 else z.clone() for _ in range(6)]
    g = torch.full((130,), 0.5, device="cuda")
    with pytest.raises(ValueError, match="elements"):
        adamw_step_many([p, p, p], [g, g, g[:100]], m[:3], m[3:], step=1)
    torch.cuda.synchronize()
    assert (p == 1).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_state(bits):
    """Weights, moments (codes and scales) and copies of a replayed step, bit for bit as eager ones."""
    from nimbleml_b200.embedding_grad import adamw_step_many, quantize_moment

    sizes = [1, 300, 16, 9000, 129]
    ps, gs, cs, _, _, _ = make(sizes, torch.bfloat16, torch.float16, 1, 19)

    def state():
        p = [x.clone() for x in ps]
        z = [torch.zeros_like(x) for x in ps]
        if bits == 8:
            return p, [quantize_moment(x) for x in z], [quantize_moment(x) for x in z], [x.clone() for x in cs]
        return p, z, [x.clone() for x in z], [x.clone() for x in cs]

    a, b = state(), state()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        adamw_step_many(b[0], gs, b[1], b[2], step=3, copies=b[3], **HYPER)
    side = torch.cuda.Stream()
    for turn in range(3):
        adamw_step_many(a[0], gs, a[1], a[2], step=3, copies=a[3], **HYPER)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side if turn == 1 else torch.cuda.current_stream()):
            graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        for one, two in zip(a, b):
            for x, y in zip(one, two):
                for u, v in zip(x, y) if isinstance(x, tuple) else ((x, y),):
                    assert u.view(torch.uint8).equal(v.view(torch.uint8))
        for g in gs:
            g.mul_(0.5)


@pytest.mark.parametrize("beta2", [0.9, 0.999, 0.9999])
def test_32_bit_moments_against_64_bits(beta2):
    """The step's betas are fp32 numbers and its 1 - beta is theirs, exactly: with these, v is off by three roundings a
    step (all its terms are positive), m by three of the sum of magnitudes. Against the betas as given, off by e <= 2^-25,
    a term (1 - beta2) beta2^k g^2 moves by e / (1 - beta2) + k e / beta2 of itself."""
    from nimbleml_b200.embedding_grad import adamw_step_many

    g = torch.Generator().manual_seed(7)
    n, steps, u = 1027, 25, 2.0**-24
    p, m, v = torch.randn(n, generator=g).cuda(), torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    b1f, b2f = float(np.float32(0.9)), float(np.float32(beta2))
    m64, v64, big, given = (torch.zeros(n, dtype=torch.float64, device="cuda") for _ in range(4))
    for t in range(1, steps + 1):
        gr = torch.randn(n, generator=g).cuda()
        adamw_step_many([p], [gr], [m], [v], step=t, beta1=0.9, beta2=beta2)
        g64 = gr.double()
        m64 = b1f * m64 + (1 - b1f) * g64
        big = b1f * big + (1 - b1f) * g64.abs()
        v64 = b2f * v64 + (1 - b2f) * g64 * g64
        given = beta2 * given + (1 - beta2) * g64 * g64
        assert ((m.double() - m64).abs() <= 1.01 * 3 * t * u * big).all()
        assert ((v.double() - v64).abs() <= 1.01 * 3 * t * u * v64).all()
        e = 2.0**-25
        assert ((v.double() - given).abs() <= (1.01 * 3 * t * u + e / (1 - beta2) + t * e / beta2) * 1.01 * given).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_counts_as_a_write(bits):
    """A backward pass over what a step has overwritten since the forward is refused, not taken from the new values."""
    from nimbleml_b200.embedding_grad import AdamW
    from nimbleml_b200.losses import tied_token_logprobs
    from nimbleml_b200.norm import layer_norm

    gamma = torch.ones(64, device="cuda", requires_grad=True)
    master = torch.randn(300, 64, device="cuda")
    weight = master.half().requires_grad_()
    x = torch.randn(5, 64, device="cuda").half().requires_grad_()
    opt = AdamW([gamma, master], copies=[None, weight.detach()], state_bits=bits, learning_rate=0.1)
    gamma.grad, master.grad = torch.ones_like(gamma), torch.ones_like(master)
    y = layer_norm(x.float(), gamma)
    r = tied_token_logprobs(x, weight, torch.arange(5, device="cuda"))
    before = [t._version for t in (gamma, master, weight)]
    opt.step()
    assert all(t._version > v for t, v in zip((gamma, master, weight), before))
    assert all(m._version > 0 for q in (*opt.m, *opt.v) for m in (q if bits == 8 else (q,)))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.logprobs.sum().backward()
    # Afresh all is well; inference tensors, which count nothing, are stepped too.
    (layer_norm(x.float(), gamma).sum() + tied_token_logprobs(x, weight, torch.arange(5, device="cuda")).logprobs.sum()).backward()
    with torch.inference_mode():
        p = torch.ones(40, device="cuda")
        p.grad = torch.ones(40, device="cuda")
        inside = AdamW([p], state_bits=bits)
        inside.step()
        assert (p < 1).all()
