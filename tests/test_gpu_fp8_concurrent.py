"""GPU: fp8 and sort calls beside each other: two streams, two host threads, a captured backward pass with frozen weights, rows
that are not numbers."""
import threading

import numpy as np
import pytest
import torch

from oracle import fp8 as of8
from tests import fp8_cases as fc

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def _leaf(pkg, bits, s):
    return pkg.Fp8Leaf(torch.from_numpy(bits).cuda().view(F8), torch.from_numpy(s).cuda())


def _layer(pkg, rng, E=6, D=400, I=272):
    leaves = [_leaf(pkg, *of8.random_weights(rng, R, K, 0.05, E)) for R, K in ((I, D), (I, D), (D, I))]
    return leaves, [pkg.Fp8Leaf(l.q[1], l.s[1]) for l in leaves]


def _inputs(rng, T, E=6, k=2, D=400):
    idx = torch.from_numpy(np.stack([rng.permutation(E)[:k] for _ in range(T)]).astype(np.int32)).cuda()
    return fc.acts(rng, T, D).cuda(), idx, torch.from_numpy(rng.uniform(0, 1, (T, k)).astype(np.float32)).cuda()


def _run(pkg, leaves, one, x, idx, w):
    plan = pkg.ragged_plan(idx, w, 6, 16)
    y = pkg.fp8_grouped(pkg.moe_dispatch(x, plan), plan, leaves[0])
    return [pkg.fp8_moe(*leaves, x, idx, w, fc.LIMIT)[0], pkg.fp8_project(x, one[0]), pkg.fp8_mlp(x, *one, fc.LIMIT),
            pkg.moe_combine(y, plan, w)]


def test_two_streams_at_once(pkg, gpu):
    rng = np.random.default_rng(1)
    leaves, one = _layer(pkg, rng)
    work = [_inputs(rng, T) for T in (1, 300, 20, 64, 130, 7)]
    want = [_run(pkg, leaves, one, *ins) for ins in work]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(4):
        for n in range(len(work)):
            for j, s in enumerate(streams):
                with torch.cuda.stream(s):
                    at = (n + 3 * j) % len(work)
                    got[j].append((at, _run(pkg, leaves, one, *work[at])))
    torch.cuda.synchronize()
    for at, outs in got[0] + got[1]:
        assert all(torch.equal(a, b) for a, b in zip(outs, want[at]))


def test_two_threads_at_once(pkg, gpu):
    rng = np.random.default_rng(2)
    leaves, one = _layer(pkg, rng)
    work = [_inputs(rng, T) for T in (2, 200, 40, 16)]
    want = [_run(pkg, leaves, one, *ins) for ins in work]
    torch.cuda.synchronize()
    wrong, gate = [], threading.Barrier(2)

    def body(first):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                gate.wait(30)
                for n in range(12):
                    at = (n + first) % len(work)
                    outs = _run(pkg, leaves, one, *work[at])
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(outs, want[at])):
                        wrong.append((first, n))
        except Exception as e:                             # noqa: BLE001 (a thread's error would be lost)
            wrong.append(e)

    threads = [threading.Thread(target=body, args=(j,)) for j in (0, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not wrong, wrong


def test_backward_on_the_forward_stream(pkg, gpu):
    """The pair on a stream of its own, the backward pass called from another: autograd returns to the forward's."""
    rng = np.random.default_rng(3)
    x, idx, w = _inputs(rng, 150)
    plan = pkg.ragged_plan(idx, w, 6, 16)

    def step(x, w):
        x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
        out = pkg.moe_combine(pkg.moe_dispatch(x, plan) * 3.0, plan, w)
        return x, w, out

    a = step(x, w)
    want = torch.autograd.grad(a[2].float().sum(), a[:2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = step(x, w)
        loss = b[2].float().sum()
    torch.cuda.current_stream().wait_stream(side)
    got = torch.autograd.grad(loss, b[:2])
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_frozen_weights_captured(pkg, gpu):
    """Forward and backward with frozen routing weights in one graph, replayed with new inputs between eager steps."""
    rng = np.random.default_rng(4)
    x, idx, w = _inputs(rng, 90)
    plan = pkg.ragged_plan(idx, w, 6, 16)
    sx, sw, sg = x.clone(), w.clone(), torch.randn_like(x)

    def step(x0, w0, g0):
        x1 = x0.detach().requires_grad_()
        out = pkg.moe_combine(pkg.moe_dispatch(x1, plan) * 2.0, plan, w0)
        return (out.detach(),) + torch.autograd.grad(out, [x1], g0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(sx, sw, sg)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step(sx, sw, sg)
    for _ in range(4):
        nx, nw, ng = torch.randn_like(x), torch.rand_like(w), torch.randn_like(x)
        sx.copy_(nx), sw.copy_(nw), sg.copy_(ng)
        want = step(nx, nw, ng)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("B", [2, 20, 40, 200])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_mlp_row_that_is_no_number(pkg, gpu, B, value):
    """Infinities and NaN become NaN when quantised: that row is NaN throughout, the others keep their bits."""
    rng = np.random.default_rng(B)
    _, one = _layer(pkg, rng)
    x = fc.acts(rng, B, 400).cuda()
    for form in (torch.bfloat16, torch.float32):
        a = x.to(form)
        clean = pkg.fp8_mlp(a, *one, fc.LIMIT, want_f32=True)[1]
        for col in (0, 399):
            bad = a.clone()
            bad[1, col] = value
            for rows in (bad, pkg.fp8_quantize(bad)):
                y = pkg.fp8_mlp(rows, *one, fc.LIMIT, want_f32=True)[1]
                keep = torch.arange(B, device="cuda") != 1
                assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[1]).all()


@pytest.mark.parametrize("B", [1, 20, 40, 200])
def test_mlp_without_a_clamp(pkg, gpu, B):
    """limit inf: no clamp; a gate far below zero gives h 0, not NaN."""
    rng = np.random.default_rng(B)
    D, I = 128, 32
    raw = [of8.random_weights(rng, R, K, 0.05) for R, K in ((I, D), (I, D), (D, I))]
    x = torch.from_numpy(rng.standard_normal((B, D)).astype(np.float32) * 100).to(torch.bfloat16)
    want, bound = of8.mlp(fc.values(x), *[of8.weights_dense(*r) for r in raw], np.inf, f32_gate_up=B <= 128)
    got = pkg.fp8_mlp(x.cuda(), *[_leaf(pkg, *r) for r in raw], float("inf"), want_f32=True)[1].double().cpu().numpy()
    assert np.all(np.abs(got - want) <= bound)
