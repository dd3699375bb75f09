"""GPU: the operators around a layer's experts as they are used together: the output projection into the stream, the norm, the
gate, the experts and the way back, for serving over fp8 leaves and for training."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
F8 = torch.float8_e4m3fn
LIMIT, EPS = 7.0, 1e-5
D, I, E, K = 512, 256, 16, 4


def _rand(shape, seed, scale=1.0, dtype=BF16):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (scale * torch.randn(shape, device="cuda", generator=g)).to(dtype)


def _leaf(pkg, shape, seed):
    w = _rand(shape, seed, 0.05, torch.float32)
    R, C = shape[-2:]
    b = w.view(*shape[:-2], R // 128, 128, C // 128, 128)
    s = b.abs().amax((-3, -1)) / 448.0
    return pkg.Fp8Leaf((b / s[..., :, None, :, None]).view(shape).to(F8), s.contiguous())


@pytest.mark.parametrize("T", [1, 5, 16, 40, 300])
def test_serving_layer(pkg, gpu, T):
    """Each call against the framework's separate ones, from the same inputs."""
    o_proj, norm_w = pkg.Bf16Leaf(_rand((D, D), 1, 0.05)), _rand((D,), 2, 0.1) + 1
    experts = [_leaf(pkg, s, 3 + n) for n, s in enumerate(((E, I, D), (E, I, D), (E, D, I)))]
    shared = [_leaf(pkg, s, 6 + n) for n, s in enumerate(((I, D), (I, D), (D, I)))]
    router, bias = _rand((D, E), 9, 0.1, torch.float32), _rand((E,), 10, 0.05, torch.float32)
    attn, h = _rand((T, D), 11), _rand((T, D), 12)

    def layer(attn, h):
        mid = pkg.bf16_linear(attn, o_proj)
        pair, h, y = pkg.fp8_rms_norm(mid, norm_w, EPS, residual=h, want_y=True)
        idx, w = pkg.moe_gate(y.float() @ router, K, bias=bias, n_group=4, topk_group=2, scaling=2.5)
        out, _ = pkg.fp8_moe(*experts, y, idx, w, LIMIT)
        return h, y, pair, idx, w, pkg.fp8_mlp(pair, *shared, LIMIT), out

    h2, y, (q, qs), idx, w, sh, out = layer(attn, h)
    mid = pkg.bf16_linear(attn, o_proj)
    if T <= 32:                                       # bf16_project's product, in another order of its f32 sums
        p, pf = pkg.bf16_project(attn, o_proj, want_f32=True)
        mag = attn.double().abs() @ o_proj.wT.double().abs().t()
        assert bool(((mid.double() - pf.double()).abs() <= 2.0 ** -8 * pf.double().abs() + 2.0 ** -23 * 64 * mag).all())
    assert torch.equal(h2, (mid.float() + h.float()).to(BF16))
    y2, s2 = pkg.rms_norm(mid, norm_w, EPS, residual=h)
    assert torch.equal(y2, y) and torch.equal(s2, h2)
    v = h2.float()
    r = (1.0 / torch.sqrt(v.double().square().mean(-1, keepdim=True) + EPS)).float()
    q2, qs2 = pkg.fp8_quantize((v * r) * norm_w.float())
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(qs, qs2)
    assert torch.equal(sh, pkg.fp8_mlp((q2, qs2), *shared, LIMIT))
    c = torch.sigmoid((y.float() @ router).double()) + bias.double()
    top = c.view(T, 4, 4).sort(-1, descending=True)[0][..., :2].sum(-1).argsort(-1, descending=True)[:, :2]
    assert all(set((idx[t] // 4).tolist()) <= set(top[t].tolist()) for t in range(T))
    assert bool(((w.sum(-1) - 2.5).abs() <= 2.5 * 2.0 ** -21).all())

    # captured: one graph a step, replayed on new inputs
    a, b = attn.clone(), h.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(a, b)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = layer(a, b)
    for k in range(3):
        a.copy_(_rand((T, D), 20 + k)), b.copy_(_rand((T, D), 30 + k))
        want = layer(a.clone(), b.clone())
        g.replay()
        torch.cuda.synchronize()
        for x, y in zip(outs, want):
            for p, n in zip(x if isinstance(x, tuple) else (x,), y if isinstance(y, tuple) else (y,)):
                assert torch.equal(p.view(torch.uint8), n.view(torch.uint8))


@pytest.mark.parametrize("T", [3, 50, 260])
def test_training_layer(pkg, gpu, T):
    """Gradients through all of them at once against autograd in 64 bits on the same choices.  On the way of any of them lie at
    most 10 roundings to bf16, each at most 2^-8 of its tensor (2-norm), and no step stretches a relative error more than
    about twofold (the norm's and the gate's projections; the sums of k terms shrink it)."""
    w1, w2, wo = _rand((I, D), 1, 0.05), _rand((D, I), 2, 0.05), _rand((D, D), 3, 0.04)
    b1, nw, router = _rand((I,), 4, 0.1), _rand((D,), 5, 0.1) + 1, _rand((E, D), 6, 0.05)
    attn, h, gout = _rand((T, D), 7), _rand((T, D), 8), _rand((T, D), 9)
    factor = 0.5 + torch.arange(E, device="cuda") / 16.0            # one pair of matrices, times what tells the experts apart

    def layer(attn, h, wo, nw, router, w1, b1, w2):
        y, s = pkg.rms_norm(pkg.bf16_linear(attn, pkg.Bf16Leaf(wo), residual=h), nw, EPS, residual=h)
        idx, w = pkg.moe_gate(pkg.bf16_linear(y, pkg.Bf16Leaf(router), dtype=torch.float32), K, scores="softmax")
        plan = pkg.ragged_plan(idx, w.detach(), E, 16)
        xs = pkg.moe_dispatch(y, plan)
        ys = pkg.bf16_linear(pkg.bf16_linear(xs, pkg.Bf16Leaf(w1), bias=b1, act="silu"), pkg.Bf16Leaf(w2))
        ys = ys * factor[plan["blk_expert"].long()].repeat_interleave(16)[:, None].to(BF16)
        return pkg.moe_combine(ys, plan, w) + s, idx

    ins = [attn, h, wo, nw, router, w1, b1, w2]
    leaves = [t.detach().requires_grad_() for t in ins]
    out, idx = layer(*leaves)
    got = torch.autograd.grad(out, leaves, gout)

    d = [t.detach().double().requires_grad_() for t in ins]
    a_, h_, wo_, nw_, r_, w1_, b1_, w2_ = d
    s = a_ @ wo_.t() + h_ + h_
    y = s / torch.sqrt(s.square().mean(-1, keepdim=True) + EPS) * nw_
    p = torch.softmax(y @ r_.t(), -1).gather(1, idx.long())
    w = p / p.sum(-1, keepdim=True)
    f = torch.nn.functional.silu(y @ w1_.t() + b1_) @ w2_.t()
    want_out = (w * factor[idx.long()].double()).sum(-1, keepdim=True) * f + s
    want = torch.autograd.grad(want_out, d, gout.double())
    rel = lambda x, y: float((x.double() - y).norm() / y.norm().clamp_min(1e-30))  # noqa: E731
    assert rel(out, want_out) <= 10 * 2.0 ** -8
    for n, (x, y) in enumerate(zip(got, want)):
        assert rel(x, y) <= 20 * 2.0 ** -8, (n, rel(x, y))
