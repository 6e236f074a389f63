"""The operators in one run: final layer norm -> log probabilities and entropies of the sampled tokens from the tied
matrix -> a clipped policy loss -> backward -> an AdamW step with 8-bit moments; then scoring with the new weights."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def loss_of(lp, ent, old, adv, live):
    ratio = (lp - old).exp()
    gain = torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv) + 0.01 * ent
    return -(gain * live).sum() / live.sum()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_policy_step(dtype):
    from nimbleml_b200.embedding_grad import AdamW
    from nimbleml_b200.gpt_head import TiedEmbedding
    from nimbleml_b200.lm_head import last_token_logits
    from nimbleml_b200.losses import token_logprobs
    from nimbleml_b200.norm import LayerNorm

    g = torch.Generator().manual_seed(1)
    b, s, d, v = 3, 40, 128, 2001
    x = torch.randn(b, s, d, generator=g).to(dtype).cuda()
    emb = TiedEmbedding((0.1 * torch.randn(v, d, generator=g)).cuda(), v, compute_dtype=dtype)
    norm = LayerNorm(d, device="cuda")
    tokens = torch.randint(0, v, (b, s), generator=g).cuda()
    tokens[1, 25:] = -100
    adv = torch.randn(b, s, generator=g).cuda()
    live = (tokens != -100).float()
    scale = 1024.0 if dtype == torch.float16 else 1.0

    xl = x.clone().requires_grad_()
    y = norm(xl)
    r = emb.token_logprobs(y, tokens, -100)
    old = r.logprobs.detach() + 0.1 * torch.randn(b, s, generator=g).cuda()
    loss = loss_of(r.logprobs, r.entropy, old, adv, live)
    (loss * scale).backward()

    # The same in 64 bits, from the same 16-bit E.
    x64 = x.double().requires_grad_()
    gam, bet = torch.ones(d, dtype=torch.float64, device="cuda", requires_grad=True), torch.zeros(
        d, dtype=torch.float64, device="cuda", requires_grad=True)
    e64 = emb.weight.double().requires_grad_()
    y64 = torch.nn.functional.layer_norm(x64, (d,), gam, bet, 1e-5)
    q = torch.log_softmax(y64 @ e64.t(), -1)
    lp = q.gather(-1, tokens.clamp(min=0).unsqueeze(-1)).squeeze(-1)
    ent = -(q.exp() * q).sum(-1)
    want = loss_of(lp * live, ent * live, old.double(), adv.double(), live.double())
    want.backward()
    # y is rounded to 16 bits on the way (half a step), G once more and the results once: three half steps, with
    # the products' growth of a row's relative error below 8.
    tol = 3 * 8 * torch.finfo(dtype).eps / 2
    assert abs(float(loss) - float(want)) <= tol * max(1.0, abs(float(want)))
    for got, ref in ((xl.grad, x64.grad), (norm.gamma.grad, gam.grad), (norm.beta.grad, bet.grad), (emb.grad, e64.grad)):
        ref = ref * scale
        assert float((got.double() - ref).norm()) <= tol * float(ref.norm())
    assert (xl.grad[1, 25:] == 0).all()

    # One optimizer for the head and the norm, moments in 8 bits, E's 16-bit copy refreshed in the same launch.
    emb.master.grad = emb.grad / scale
    norm.gamma.grad /= scale
    norm.beta.grad /= scale
    params = [emb.master, norm.gamma.data, norm.beta.data]
    params[1].grad, params[2].grad = norm.gamma.grad, norm.beta.grad
    opt = AdamW(params, learning_rate=1e-2, weight_decay=0.0, copies=[emb.weight, None, None], state_bits=8)
    before = emb.master.clone()
    opt.step()
    moved = emb.master - before
    # A first step moves every weight with a gradient by lr against its sign (eps is far below the gradients' roots).
    far = emb.grad.abs() > 1e-5 * scale
    assert ((moved + 1e-2 * emb.grad.sign()).abs()[far] <= 2e-5).all()
    assert emb.weight.equal(emb.master.to(dtype))

    # Scoring: the next token's alternatives from the last position's logits.
    with torch.no_grad():
        logits = last_token_logits(norm(x), emb.weight)
        top = token_logprobs(logits, tokens[:, 0], top_k=5)
    want_ids = torch.sort(logits.double(), dim=1, descending=True, stable=True).indices[:, :5]
    assert top.top_ids.equal(want_ids)


def test_tracing_and_forward_mode_are_refused_on_the_gpu():
    from test_operator_refusals import refuse_tracing_and_forward_mode

    refuse_tracing_and_forward_mode("cuda")
    # A level without tangents, and tangents that are switched off, refuse nothing.
    import torch.autograd.forward_ad as fw

    from nimbleml_b200.norm import layer_norm

    x, g = torch.randn(3, 64, device="cuda"), torch.ones(64, device="cuda")
    want = layer_norm(x, g)
    with fw.dual_level():
        assert layer_norm(x, g).equal(want)
        dual = fw.make_dual(x, torch.ones_like(x))
        with fw._set_fwd_grad_enabled(False):
            assert layer_norm(dual, g).equal(want)
        assert layer_norm(fw.unpack_dual(dual).primal, g).equal(want)
