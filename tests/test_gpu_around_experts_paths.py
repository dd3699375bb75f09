"""GPU: a training layer's gradients one path at a time (the gate's, the experts', the stream's), so that the bound of a path is
of its own size and a part that is missing from a small path shows."""
import pytest
import torch

from tests.test_gpu_around_experts import BF16, D, E, EPS, I, K, _rand

pytestmark = pytest.mark.gpu
NAMES = ["attn", "h", "wo", "nw", "router", "w1", "b1", "w2"]
REACHED = {"gate": {"attn", "h", "wo", "nw", "router"}, "experts": {"attn", "h", "wo", "nw", "w1", "b1", "w2"}, "stream": {"attn", "h", "wo"}}


def _layer(pkg, factor, path, attn, h, wo, nw, router, w1, b1, w2):
    y, s = pkg.rms_norm(pkg.bf16_linear(attn, pkg.Bf16Leaf(wo), residual=h), nw, EPS, residual=h)
    idx, w = pkg.moe_gate(pkg.bf16_linear(y, pkg.Bf16Leaf(router), dtype=torch.float32), K, scores="softmax")
    if path == "stream":
        return s, idx
    plan = pkg.ragged_plan(idx, w.detach(), E, 16)
    xs = pkg.moe_dispatch(y, plan)
    ys = pkg.bf16_linear(pkg.bf16_linear(xs, pkg.Bf16Leaf(w1), bias=b1, act="silu"), pkg.Bf16Leaf(w2))
    ys = ys * factor[plan["blk_expert"].long()].repeat_interleave(16)[:, None].to(BF16)
    return (pkg.moe_combine(ys.detach(), plan, w) if path == "gate" else pkg.moe_combine(ys, plan, w.detach())), idx


def _layer64(factor, path, idx, attn, h, wo, nw, router, w1, b1, w2):
    s = attn @ wo.t() + h + h
    if path == "stream":
        return s
    y = s / torch.sqrt(s.square().mean(-1, keepdim=True) + EPS) * nw
    p = torch.softmax(y @ router.t(), -1).gather(1, idx)
    w = p / p.sum(-1, keepdim=True)
    f = torch.nn.functional.silu(y @ w1.t() + b1) @ w2.t()
    if path == "gate":
        f = f.detach()
    else:
        w = w.detach()
    return (w * factor[idx].double()).sum(-1, keepdim=True) * f


@pytest.mark.parametrize("path", ["gate", "experts", "stream"])
@pytest.mark.parametrize("T", [50, 260])
def test_one_path(pkg, gpu, path, T):
    """Against autograd in 64 bits on the same choices.  The gate's path: at most 5 roundings to bf16 lie before the weights'
    gradient (s, y, h, y of the experts, its factor), which renormalising stretches by mean over spread of the four chosen factors,
    about 4; 4 more (dz, dx, ds, the result) follow: 24 times 2^-8 (2-norm).  The other paths: 10, stretched twofold at most."""
    w1, w2, wo = _rand((I, D), 1, 0.05), _rand((D, I), 2, 0.05), _rand((D, D), 3, 0.04)
    b1, nw, router = _rand((I,), 4, 0.1), _rand((D,), 5, 0.1) + 1, _rand((E, D), 6, 0.05)
    attn, h, gout = _rand((T, D), 7), _rand((T, D), 8), _rand((T, D), 9)
    factor = 0.5 + torch.arange(E, device="cuda") / 16.0
    ins = [attn, h, wo, nw, router, w1, b1, w2]
    leaves = [t.detach().requires_grad_() for t in ins]
    out, idx = _layer(pkg, factor, path, *leaves)
    got = torch.autograd.grad(out, leaves, gout, allow_unused=True)
    d = [t.detach().double().requires_grad_() for t in ins]
    want = torch.autograd.grad(_layer64(factor, path, idx.long(), *d), d, gout.double(), allow_unused=True)
    bound = (24 if path == "gate" else 20) * 2.0 ** -8
    for name, x, y in zip(NAMES, got, want):
        assert (x is not None) == (y is not None) == (name in REACHED[path]), name
        if y is not None:
            rel = float((x.double() - y).norm() / y.norm())
            assert float(y.norm()) > 0 and rel <= bound, (name, rel)
