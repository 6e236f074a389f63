"""Argument checks of the token log probabilities, layer norm and many-tensor AdamW (no GPU needed)."""
import pytest
import torch

from nimbleml_b200._native_loader import DTYPE_BF16, DTYPE_F16, DTYPE_F32, native
from nimbleml_b200.embedding_grad import AdamW, QuantizedMoment, adamw_step_many, dequantize_moment, quantize_moment
from nimbleml_b200.losses import tied_token_logprobs, token_logprobs
from nimbleml_b200.norm import LayerNorm, layer_norm


def test_there_is_no_cpu_path():
    with pytest.raises(RuntimeError, match="CUDA"):
        token_logprobs(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="CUDA"):
        tied_token_logprobs(torch.zeros(2, 8).half(), torch.zeros(4, 8).half(), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="CUDA"):
        layer_norm(torch.zeros(2, 3), torch.ones(3))
    with pytest.raises(ValueError, match="CUDA"):
        adamw_step_many([torch.zeros(3)], [torch.zeros(3)], [torch.zeros(3)], [torch.zeros(3)], step=1)
    with pytest.raises(ValueError):
        quantize_moment(torch.zeros(3))
    with pytest.raises(ValueError):
        dequantize_moment(torch.zeros(3, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(1))


def test_adamw_lists_and_state():
    with pytest.raises(ValueError, match="one entry per tensor"):
        adamw_step_many([torch.zeros(3)], [], [torch.zeros(3)], [torch.zeros(3)], step=1)
    with pytest.raises(ValueError, match="from 1, got 0"):  # a formatted number: one C++ runtime in the process
        adamw_step_many([], [], [], [], step=0)
    adamw_step_many([], [], [], [], step=1)
    adamw_step_many([torch.zeros(3)], [None], [torch.zeros(3)], [torch.zeros(3)], step=1)
    with pytest.raises(ValueError, match="state_bits"):
        AdamW([torch.zeros(3)], state_bits=16)
    for size in (3, 16):  # a step of its own, and one of the list
        opt = AdamW([torch.zeros(size)])
        opt.params[0].grad = torch.zeros(size)
        with pytest.raises(ValueError, match="CUDA"):
            opt.step()
    opt = AdamW([torch.zeros(300)], state_bits=8)
    assert isinstance(opt.m[0], QuantizedMoment) and opt.m[0].scales.numel() == 3
    with pytest.raises(ValueError, match="float32"):
        AdamW([torch.zeros(3, dtype=torch.float16)])
    with pytest.raises(ValueError, match="Expected last dim"):
        LayerNorm(4)(torch.zeros(2, 5))


def _fails(code, name, *args):
    with pytest.raises(RuntimeError, match=rf"\({code}\)"):
        native.call(name, *args)


def test_native_token_logprobs_arguments():
    p = 1 << 20  # never dereferenced: the checks come first

    def fwd(x=p, ld=10, tok=p, n=4, v=10, dt=DTYPE_F32, k=0, out=p, top=None):
        return (x, ld, tok, n, v, dt, -1, k, out, out, out, out, top, top, None, None)

    _fails(-1, "nimble_token_logprobs_forward", *fwd(dt=7))
    _fails(-1, "nimble_token_logprobs_forward", *fwd(ld=9))
    _fails(-1, "nimble_token_logprobs_forward", *fwd(v=0))
    _fails(-1, "nimble_token_logprobs_forward", *fwd(n=-1))
    _fails(-1, "nimble_token_logprobs_forward", *fwd(v=2**31, ld=2**31))
    _fails(-1, "nimble_token_logprobs_forward", *fwd(k=11))
    _fails(-1, "nimble_token_logprobs_forward", *fwd(v=100, ld=100, k=65, top=p))
    _fails(-1, "nimble_token_logprobs_forward", *fwd(k=2))  # no place for the alternatives
    _fails(-1, "nimble_token_logprobs_forward", *fwd(x=None))
    _fails(-1, "nimble_token_logprobs_forward", *fwd(x=p + 2))
    _fails(-1, "nimble_token_logprobs_forward", *fwd(out=None))
    native.call("nimble_token_logprobs_forward", *fwd(n=0))

    def bwd(ld=10, gld=10, g=p, v=10, n=4):
        return (p, p, p, ld, p, p, p, p, n, v, DTYPE_F16, -1, g, gld, None)

    _fails(-1, "nimble_token_logprobs_backward", *bwd(gld=9))
    _fails(-1, "nimble_token_logprobs_backward", *bwd(g=None))
    _fails(-1, "nimble_token_logprobs_backward", *bwd(g=p + 1))
    _fails(-1, "nimble_token_logprobs_backward", *bwd(n=2**31))
    native.call("nimble_token_logprobs_backward", *bwd(n=0))


def test_native_tied_logprobs_arguments():
    p = 1 << 20
    with pytest.raises(RuntimeError, match="f16 / bf16"):
        native.tied_logprobs_forward_workspace_size(4, 8, 10, DTYPE_F32)
    with pytest.raises(RuntimeError, match="positive"):
        native.tied_logprobs_backward_workspace_size(4, 8, 0, DTYPE_F16)
    assert native.tied_logprobs_forward_workspace_size(0, 8, 10, DTYPE_F16) == 0
    native.tied_logprobs_backward_workspace_size(0, 8, 10, DTYPE_F16)
    need = native.tied_logprobs_forward_workspace_size(4096, 4096, 128256, DTYPE_BF16)
    assert need < 4096 * 128256 * 2 / 16  # no N x V buffer
    assert native.tied_logprobs_backward_workspace_size(4096, 4096, 128256, DTYPE_BF16) < 4096 * 128256 * 2

    def fwd(d=8, dt=DTYPE_F16, ws=1 << 20, off=0, out=p, n=4, res=(None, None, None), flag=None):
        return (p, p, p, n, d, 100, off, dt, -1, out, *res, p, ws, None, flag, None)

    _fails(-1, "nimble_tied_logprobs_forward", *fwd(dt=DTYPE_F32))
    _fails(-1, "nimble_tied_logprobs_forward", *fwd(d=9))
    _fails(-1, "nimble_tied_logprobs_forward", *fwd(off=-1))
    _fails(-1, "nimble_tied_logprobs_forward", *fwd(out=None))
    _fails(-1, "nimble_tied_logprobs_forward", *fwd(out=None, res=(p, p, None)))
    _fails(-1, "nimble_tied_logprobs_forward", *fwd(off=5, res=(p, p, p)))  # not the whole vocabulary
    _fails(-1, "nimble_tied_logprobs_forward", *fwd(flag=p))  # nothing to tell without a status word
    _fails(-2, "nimble_tied_logprobs_forward", *fwd(ws=8))
    native.call("nimble_tied_logprobs_forward", *fwd(n=0))

    def bwd(d=8, off=0, vocab=100, gh=p, gdt=DTYPE_F16, ws=1 << 30, lse=p):
        return (p, p, p, p, p, lse, p, 4, d, 100, off, vocab, -1, DTYPE_F16, gh, gdt, p, gdt, 0, 0, p, ws, None, None)

    _fails(-1, "nimble_tied_logprobs_backward", *bwd(off=1))
    _fails(-1, "nimble_tied_logprobs_backward", *bwd(gh=p + 2))
    _fails(-1, "nimble_tied_logprobs_backward", *bwd(gdt=9))
    _fails(-1, "nimble_tied_logprobs_backward", *bwd(lse=None))
    _fails(-2, "nimble_tied_logprobs_backward", *bwd(ws=64))
    _fails(-1, "nimble_tied_logprobs_combine", p, 0, p, 4, 100, -1, p, p, p, None, None)
    _fails(-1, "nimble_tied_logprobs_combine", None, 1, p, 4, 100, -1, p, p, p, None, None)
    native.call("nimble_tied_logprobs_combine", None, 1, None, 0, 100, -1, None, None, None, None, None)


def test_native_layernorm_arguments():
    p = 1 << 20

    def fwd(d=8, pitch=8, dt=DTYPE_F16, pdt=DTYPE_F32, mean=p, rstd=p, n=4, x=p):
        return (x, pitch, p, None, n, d, 1e-5, dt, pdt, p, mean, rstd, None)

    _fails(-1, "nimble_layernorm_forward", *fwd(d=8193, pitch=8193))
    _fails(-1, "nimble_layernorm_forward", *fwd(d=0))
    _fails(-1, "nimble_layernorm_forward", *fwd(pitch=7))
    _fails(-1, "nimble_layernorm_forward", *fwd(pdt=DTYPE_BF16))
    _fails(-1, "nimble_layernorm_forward", *fwd(dt=5))
    _fails(-1, "nimble_layernorm_forward", *fwd(mean=None))
    _fails(-1, "nimble_layernorm_forward", *fwd(x=None))
    native.call("nimble_layernorm_forward", *fwd(n=0))
    with pytest.raises(RuntimeError):
        native.layernorm_backward_workspace_size(4, 8193)
    need = native.layernorm_backward_workspace_size(5000, 1000)
    args = (p, p, 1000, p, p, p, 5000, 1000, DTYPE_F16, DTYPE_F32, p, p, p, p)
    _fails(-2, "nimble_layernorm_backward", *args, need - 1, None)
    _fails(-1, "nimble_layernorm_backward", p, p, 1000, p, p, p, 5000, 1000, DTYPE_F16, DTYPE_F32, p, None, p, p, need,
           None)


def test_native_adamw_many_arguments():
    from array import array

    p = 1 << 20

    def row(w=p, g=p, m=p, v=p, ms=p, vs=p, c=0, n=4, gdt=DTYPE_F32, cdt=0):
        return array("q", (w, g, m, v, ms, vs, c, n, gdt | cdt << 32))

    kept = []

    def call(r, bits=32, count=1):
        kept.append(r)  # the call reads the array's memory
        return (r.buffer_info()[0], count, bits, 1e-3, 0.9, 0.999, 0.1, 0.001, 1e-8, 0.0, None)

    for bad in (row(w=0), row(g=0), row(m=0), row(v=0), row(n=-1), row(gdt=8), row(c=p, cdt=4), row(w=p + 2),
                row(g=p + 1, gdt=DTYPE_F16), row(m=p + 1), row(c=p + 1, cdt=DTYPE_F16), row(n=2**62)):
        _fails(-1, "nimble_adamw_step_many", *call(bad))
    _fails(-1, "nimble_adamw_step_many", *call(row(ms=0), bits=8))
    _fails(-1, "nimble_adamw_step_many", *call(row(), bits=16))
    _fails(-1, "nimble_adamw_step_many", *call(row(), count=-1))
    _fails(-1, "nimble_adamw_step_many", None, 1, 32, 1e-3, 0.9, 0.999, 0.1, 0.001, 1e-8, 0.0, None)
    native.call("nimble_adamw_step_many", *call(row(n=0)))
    native.call("nimble_adamw_step_many", None, 0, 32, 1e-3, 0.9, 0.999, 0.1, 0.001, 1e-8, 0.0, None)
    _fails(-1, "nimble_adamw_dequantize", None, p, 4, 0, p, None)
    _fails(-1, "nimble_adamw_quantize", p, -1, 0, p, p, None)
    native.call("nimble_adamw_dequantize", None, None, 0, 0, None, None)


def test_adamw_copies_match_the_weights():
    with pytest.raises(ValueError, match="one entry per tensor: 1 for 2"):
        AdamW([torch.zeros(3), torch.zeros(8)], copies=[None])
    # A refused step (these weights are on the CPU) does not count.
    opt = AdamW([torch.zeros(3), torch.zeros(16)], copies=[None, None])
    for p in opt.params:
        p.grad = torch.ones_like(p)
    with pytest.raises(ValueError, match="CUDA"):
        opt.step()
    assert opt.t == 0


def test_tracing_and_forward_mode_are_refused():
    """The kernels write through raw pointers: a trace would hold none of them, and a tangent would be lost."""
    refuse_tracing_and_forward_mode("cpu")


def refuse_tracing_and_forward_mode(device):
    import torch.autograd.forward_ad as fw
    from torch.fx.experimental.proxy_tensor import make_fx

    def t(*shape, dtype=torch.float32):
        return torch.ones(shape, dtype=dtype, device=device)

    ids = torch.zeros(2, dtype=torch.int64, device=device)
    w = t(5, 16, dtype=torch.float16)
    codes = torch.zeros(16, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)

    def step(p):
        adamw_step_many([p], [t(2, 16)], [t(2, 16)], [t(2, 16)], step=1)
        return p

    def step_grad(g):
        adamw_step_many([t(2, 16)], [g], [t(2, 16)], [t(2, 16)], step=1)
        return g

    calls = {
        "layer_norm": (lambda x: layer_norm(x, t(16)), t(2, 16)),
        "layer_norm ": (lambda g: layer_norm(t(2, 16), g), t(16)),
        "layer_norm  ": (lambda b: layer_norm(t(2, 16), t(16), b), t(16)),
        "layer_norm   ": (LayerNorm(16, device=device), t(2, 16)),
        "token_logprobs": (lambda x: token_logprobs(x, ids).logprobs, t(2, 16)),
        "tied_token_logprobs": (lambda h: tied_token_logprobs(h, w, ids).logprobs, t(2, 16, dtype=torch.float16)),
        "tied_token_logprobs ": (lambda e: tied_token_logprobs(t(2, 16, dtype=torch.float16), e, ids).entropy, w),
        "tied_token_logprobs  ": (lambda h: tied_token_logprobs(h, w, ids, vocab_size=9).logprobs,
                                  t(2, 16, dtype=torch.float16)),
        "adamw_step_many": (step, t(2, 16)),
        "adamw_step_many ": (step_grad, t(2, 16)),
        "quantize_moment": (lambda x: quantize_moment(x).scales, t(16)),
        "dequantize_moment": (lambda s: dequantize_moment(codes, s), t(1)),
    }
    for name, (call, x) in calls.items():
        name = name.strip()
        with pytest.raises(RuntimeError, match=f"{name} cannot be traced"):
            torch.jit.trace(call, (x,), check_trace=False)
        with pytest.raises(RuntimeError, match=f"{name} cannot be traced"):
            make_fx(call)(x)
        with fw.dual_level():
            dual = fw.make_dual(x, torch.ones_like(x))
            with pytest.raises(NotImplementedError, match=f"{name} has no forward-mode derivative"):
                call(dual)
            if not name.startswith("adamw"):  # the same where a node would be built
                with pytest.raises(NotImplementedError, match=f"{name} has no forward-mode derivative"):
                    call(fw.make_dual(x.clone().requires_grad_(), torch.ones_like(x)))


def test_native_tied_logprobs_backward_alignment():
    """The row kernels use 16-byte accesses: what does not allow them is refused before any launch."""
    p = 1 << 20
    for h, ws in ((p + 2, p), (p + 8, p), (p, p + 8)):
        _fails(-1, "nimble_tied_logprobs_backward", p, p, h, p, p, p, p, 4, 8, 100, 0, 100, -1, DTYPE_F16, p, DTYPE_F16, p,
               DTYPE_F16, 0, 0, ws, 1 << 30, None, None)


def test_host_module_of_another_torch(monkeypatch):
    """After a torch upgrade the module that the old one was built with is neither loaded nor up to date."""
    from nimbleml_b200 import build_native
    from nimbleml_b200._host import load_host

    here = build_native.host_module_path()
    assert here.exists() and not build_native._stale(here, [build_native.HOST_SOURCE, build_native.LIB_PATH])
    monkeypatch.setattr(torch, "__version__", "99.0.0+cu999")
    other = build_native.host_module_path()
    assert other != here and build_native._stale(other, [build_native.HOST_SOURCE])
    with pytest.raises(ImportError, match="build_native"):
        load_host()
