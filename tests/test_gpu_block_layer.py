"""SimpleMoE without quantisation, with a shared expert and with the block's
norms: against autograd over the formulas in 64 bits, and against the
operators called one by one."""
import math

import pytest
import torch

import smoe

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def rand(shape, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g) * std


def layer(dev, H, I, E, K, **kw):
    m = smoe.SimpleMoE(H, I, E, K, device=dev, **kw)
    with torch.no_grad():
        for i, p in enumerate(m.parameters()):
            if p.dim() == 1:
                p.copy_(1 + rand(p.shape, 40 + i, 0.2))
            else:
                p.copy_(rand(p.shape, 40 + i, 1 / math.sqrt(p.shape[-1] if p.dim() != 2 or p is not m.w_gate else H)))
    return m


def swiglu(z):
    g, u = z.chunk(2, -1)
    return g * torch.sigmoid(g) * u


def formula(p, x, idx, scale, norm, shared, top_k):
    """The block in 64 bits for given picks; differentiable by all of p and x."""
    rms = lambda v, w: v / torch.sqrt(v.square().mean(1, keepdim=True) + 1e-6) * w
    h = rms(x, p["norm_in"]) if norm else x
    prob = torch.softmax(h @ p["w_gate"], -1).gather(1, idx)
    w = prob / prob.sum(1, keepdim=True)
    y = 0
    for k in range(top_k):
        z = torch.einsum("tnh,th->tn", p["w1"][idx[:, k]], h)
        y = y + w[:, k:k + 1] * torch.einsum("thi,ti->th", p["w2"][idx[:, k]], swiglu(z))
    if shared:
        y = y + swiglu(h @ p["ws1"].t()) @ p["ws2"].t()
    return scale * x + p["block_gate"] * rms(y, p["norm_out"]) if norm else y


@pytest.mark.parametrize("T,H,I", [(1, 64, 48), (37, 72, 40), (150, 128, 64)])
@pytest.mark.parametrize("norm,shared", [(False, 0), (False, 56), (True, 0), (True, 56)])
def test_block_against_autograd(dev, T, H, I, norm, shared):
    """Forward and every gradient.  Between x and the output lie about ten
    tensors of bf16 (u = 2^-8), forward and backward together, whose rounding
    errors add as squares: root mean square, sqrt(10) u at most."""
    E, K, scale = 6, 2, 0.7
    m = layer(dev, H, I, E, K, recipe="bf16", shared_intermediate=shared, block_norm=norm, residual_scale=scale)
    x = rand((T, H), 1).to(BF16).to(dev).requires_grad_(True)
    dout = rand((T, H), 2).to(BF16)
    out = m(x)
    out.backward(dout.to(dev))
    # the picks: from the bits of h that the layer itself routes by
    with torch.no_grad():
        h = smoe.block_norm_in(x, m.norm_in, m.norm_eps)[0] if norm else x
        idx = smoe.router_topk(m._gate_logits(h).contiguous(), K)[0].cpu().long()
    p = {k: v.detach().cpu().double().requires_grad_(True) for k, v in m.named_parameters()}
    x64 = x.detach().cpu().double().requires_grad_(True)
    ref = formula(p, x64, idx, scale, norm, shared, K)
    ref.backward(dout.double())
    rel = lambda a, b: float((a.detach().cpu().double() - b.detach()).norm() / b.detach().norm())
    bound = math.sqrt(10) * 2.0 ** -8
    assert rel(out, ref) <= bound
    assert rel(x.grad, x64.grad) <= bound
    for name, q in m.named_parameters():
        # what reaches the router is a difference of nearly equal terms (the
        # renormalised weights' gradients less their mean): its error is
        # measured against the terms, which are up to a few times larger
        assert rel(q.grad, p[name].grad) <= bound * (8 if name == "w_gate" else 1), name


@pytest.mark.parametrize("recipe", ["bf16", "blockwise", "e8m0"])
def test_block_is_its_operators(dev, recipe):
    """Bit for bit: the norms and the shared expert around the routed layer,
    with and without autograd."""
    T, H, I, E, K, S = 96, 256, 128, 8, 2, 192
    m = layer(dev, H, I, E, K, recipe=recipe, shared_intermediate=S, block_norm=True, residual_scale=0.5)
    plain = smoe.SimpleMoE(H, I, E, K, device=dev, recipe=recipe)
    plain.load_state_dict({k: v for k, v in m.state_dict().items() if k in plain.state_dict()})
    x = rand((T, H), 3).to(BF16).to(dev)
    with torch.no_grad():
        got = m(x)
        h, _ = smoe.block_norm_in(x, m.norm_in)
        y = plain(h)
        y = smoe.linear_act(smoe.linear_act(h, m.ws1, act="swiglu"), m.ws2, residual=y)
        want, _ = smoe.block_norm_out(y, x, m.norm_out, gate=m.block_gate, residual_scale=0.5)
    assert got.equal(want)
    if recipe == "bf16":
        logits = plain._gate_logits(h).detach()
        idx, w, _, inv, _, off = smoe.route_topk_sort(logits, K)
        xp = smoe.permute_tokens_rows(h, inv, K)
        yy = smoe.linear_act(smoe.linear_act(xp, plain.w1, act="swiglu", offsets=off), plain.w2, offsets=off)
        assert plain(h).equal(smoe.unpermute_tokens(yy, inv, K, w))
        assert m(x.requires_grad_(True)).equal(got)


def test_expanded_gradient_and_second_backward(dev):
    """A sum's gradient is an expanded tensor; retain_graph gives the same
    gradients again."""
    m = layer(dev, 64, 32, 4, 2, recipe="bf16", shared_intermediate=32, block_norm=True)
    x = rand((20, 64), 5).to(BF16).to(dev).requires_grad_(True)
    loss = m(x).sum()
    loss.backward(retain_graph=True)
    first = [x.grad.clone()] + [p.grad.clone() for p in m.parameters()]
    x.grad = None
    m.zero_grad()
    loss.backward()
    for a, b in zip(first, [x.grad] + [p.grad for p in m.parameters()]):
        assert a.equal(b)


def test_main_grad_and_backward_from(dev):
    """Weight gradients added into main_grad buffers are what the plain call
    returns, added; backward_from on intermediates gives autograd's."""
    T, H, I, E, K = 60, 64, 40, 6, 2
    m = layer(dev, H, I, E, K, recipe="bf16", shared_intermediate=24)
    x = rand((T, H), 6).to(BF16).to(dev)
    g = rand((T, H), 7).to(BF16).to(dev)
    m(x).backward(g)
    names = ("w1", "w2", "ws1", "ws2")
    for n in names:
        p = getattr(m, n)
        p.main_grad = torch.ones(p.shape, dtype=torch.float32, device=dev)
    ref = {n: getattr(m, n).grad.clone() for n in names}
    m.zero_grad()
    m(x).backward(g)
    for n in names:
        p = getattr(m, n)
        assert p.grad is None
        # the bf16 gradient is the fp32 one rounded once (2^-8), the sum with
        # one is rounded to fp32
        assert ((p.main_grad - 1 - ref[n].float()).abs() <= 2.0 ** -8 * ref[n].float().abs() + 2.0 ** -22).all(), n
    r = smoe.SimpleMoE(H, I, E, K, device=dev, recipe="bf16")
    r.load_state_dict({k: v for k, v in m.state_dict().items() if k in r.state_dict()})
    out, inter = r(x, return_intermediates=True)
    grads = r.backward_from(inter, g, wgrad_dtype=BF16)
    xg = x.clone().requires_grad_(True)
    o2 = r(xg)
    o2.backward(g)
    assert out.equal(o2) and grads["dw1"].equal(r.w1.grad) and grads["dw2"].equal(r.w2.grad)
    assert grads["dw_gate"].shape == r.w_gate.shape and grads["dx"].shape == x.shape


def test_empty_batch_refusals_and_state(dev):
    m = layer(dev, 64, 32, 4, 2, recipe="bf16", shared_intermediate=32, block_norm=True)
    x = torch.empty((0, 64), dtype=BF16, device=dev)
    with torch.no_grad():
        assert m(x).shape == (0, 64)
    m(x.requires_grad_(True)).sum().backward()
    assert all(p.grad is None or not p.grad.any() for p in m.parameters())
    with pytest.raises(ValueError):
        m(x.detach(), return_intermediates=True)
    with pytest.raises(ValueError):
        smoe.SimpleMoE(64, 32, 4, 2, recipe="fp16")
    assert set(smoe.SimpleMoE(64, 32, 4, 2, device=dev).state_dict()) == {"w_gate", "w1", "w2"}


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_module_of_another_type(dev, dtype):
    """Parameters held in another type are converted at each call: the same
    output, and gradients that arrive in the parameters' type."""
    m = layer(dev, 64, 32, 4, 2, recipe="bf16", shared_intermediate=32, block_norm=True)
    x = rand((30, 64), 9).to(BF16).to(dev)
    with torch.no_grad():
        want = m(x)
        gate = m.w_gate.detach().clone()
        m.to(dtype)
        m.w_gate = torch.nn.Parameter(gate)
        # fp32 holds every bf16 value, fp16 those of 2^-17 and above: what the
        # few smaller ones of these seeded weights lose is below the output's bits
        assert m(x).equal(want)
    m(x).sum().backward()
    assert all(p.grad is not None and p.grad.dtype == p.dtype for p in m.parameters())


def test_inference_in_a_graph(dev):
    """A captured forward of the whole block, replayed on new tokens with eager
    calls in between, gives the eager bits each time."""
    T, H = 40, 128
    m = layer(dev, H, 64, 8, 2, recipe="bf16", shared_intermediate=96, block_norm=True)
    x = rand((T, H), 8).to(BF16).to(dev)
    with torch.no_grad():
        m(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = m(x)
        for i in range(4):
            x.copy_(rand((T, H), 20 + i).to(BF16))
            graph.replay()
            torch.cuda.synchronize()
            kept = held.clone()
            assert kept.equal(m(x))
