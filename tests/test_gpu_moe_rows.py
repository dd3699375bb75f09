"""GPU: tokens into expert order and back, and the gradients, against the formulas in 64 bits (f32 sums of k terms: k + 1
roundings of 2^-24 of the magnitudes; dot products over D: D roundings of at most 2^-24 each of the partial sums; bf16
results 2^-8 of the value more) and the gradients against differences."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
CASES = [(1, 4, 1, 1, 8), (1, 64, 8, 16, 6144), (3, 8, 2, 32, 136), (37, 64, 8, 16, 1360), (200, 5, 3, 40, 2056),
         (65, 96, 4, 1, 768), (5, 3, 3, 64, 16), (1000, 16, 2, 128, 64), (2, 4, 40, 16, 24)]


def _setup(pkg, rng, T, E, k, tm, D, dtype):
    idx = np.stack([rng.permutation(max(E, k))[:k] for _ in range(T)]).astype(np.int32) % E
    if T > 1:
        idx[0] = idx[0, 0]                                 # the same expert in every column
        idx[1, -1] = -1                                    # slots without a row
        idx[T - 1, 0] = E
    w = rng.standard_normal((T, k)).astype(np.float32)
    it, wt = torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda()
    plan = pkg.ragged_plan(it, wt, E, tm)
    x = torch.from_numpy(rng.standard_normal((T, D)).astype(np.float32)).to(dtype).cuda()
    y = torch.from_numpy(rng.standard_normal((plan["tok_row"].numel(), D)).astype(np.float32)).to(dtype).cuda()
    return plan, x, y, wt


def _np(t):
    return t.detach().to(torch.float64).cpu().numpy()


def _want(plan, x, y, w, gxs=None, gout=None):
    slot = plan["row_slot"].cpu().numpy()
    T, k = slot.shape
    xs, out, mag = np.zeros(y.shape), np.zeros(x.shape), np.zeros(x.shape)
    dx, dxm, dy, dw, dwm = np.zeros(x.shape), np.zeros(x.shape), np.zeros(y.shape), np.zeros(w.shape), np.zeros(w.shape)
    for t in range(T):
        for j in range(k):
            r = slot[t, j]
            if r < 0:
                continue
            xs[r] = x[t]
            out[t] += w[t, j] * y[r]
            mag[t] += np.abs(w[t, j] * y[r])
            if gout is not None:
                dx[t] += gxs[r]
                dxm[t] += np.abs(gxs[r])
                dy[r] = w[t, j] * gout[t]
                dw[t, j] = gout[t] @ y[r]
                dwm[t, j] = np.abs(gout[t]) @ np.abs(y[r])
    return xs, (out, mag), (dx, dxm), dy, (dw, dwm)


def _near(got, want, mag, n, dtype):
    f32 = (n + 1) * 2.0 ** -24 * mag
    half = 2.0 ** -8 * (np.abs(want) + f32) if dtype == torch.bfloat16 else 0.0
    assert np.all(np.abs(_np(got) - want) <= f32 + half)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,E,k,tm,D", CASES)
def test_values_and_gradients(pkg, gpu, T, E, k, tm, D, dtype):
    rng = np.random.default_rng(T * 7 + D)
    plan, x, y, w = _setup(pkg, rng, T, E, k, tm, D, dtype)
    for t in (x, y, w):
        t.requires_grad_(True)
    gxs = torch.from_numpy(rng.standard_normal(y.shape).astype(np.float32)).to(dtype).cuda()
    gout = torch.from_numpy(rng.standard_normal(x.shape).astype(np.float32)).to(dtype).cuda()
    xs, out = pkg.moe_dispatch(x, plan), pkg.moe_combine(y, plan, w)
    dx, dy, dw = torch.autograd.grad([xs, out], [x, y, w], [gxs, gout])
    wxs, wout, wdx, wdy, wdw = _want(plan, _np(x), _np(y), _np(w), _np(gxs), _np(gout))
    assert np.array_equal(_np(xs), wxs) and xs.dtype == dtype and out.dtype == dtype
    _near(out, *wout, k, dtype)
    _near(dx, *wdx, k, dtype)
    _near(dy, wdy, np.abs(wdy), 1, dtype)
    _near(dw, *wdw, D, torch.float32)
    live = np.zeros(y.shape[0], bool)
    slot = plan["row_slot"].cpu().numpy()
    live[slot[slot >= 0]] = True
    assert (_np(dy)[~live] == 0).all() and (_np(dw)[slot < 0] == 0).all()


def test_gradients_against_differences(pkg, gpu):
    """Both maps are linear in each input, so a difference quotient is exact up to f32 rounding: for a step of 1, the sum's
    magnitude times 2^-24 per term, over the whole output."""
    rng = np.random.default_rng(5)
    T, E, k, tm, D = 12, 4, 2, 16, 40
    plan, x, y, w = _setup(pkg, rng, T, E, k, tm, D, torch.float32)
    gxs, gout = torch.randn_like(y), torch.randn_like(x)
    f = lambda x, y, w: (pkg.moe_dispatch(x, plan).double() * gxs).sum() + (pkg.moe_combine(y, plan, w).double() * gout).sum()
    tol = 2.0 ** -24 * 8 * float((gout.abs().sum() + gxs.abs().sum()) * (w.abs().max() + 1) * (y.abs().max() + x.abs().max() + 1))
    ins = [t.requires_grad_(True) for t in (x, y, w)]
    grads = torch.autograd.grad(f(*ins), ins)
    with torch.no_grad():
        base = f(*ins)
        for n, (t, g) in enumerate(zip(ins, grads)):
            for at in rng.integers(0, t.numel(), 12):
                moved = t.detach().clone()
                moved.view(-1)[at] += 1.0
                d = f(*[moved if m == n else o for m, o in enumerate(ins)]) - base
                assert abs(float(d) - float(g.view(-1)[at])) <= tol


def test_broadcast_and_strided_gradients(pkg, gpu):
    """Inputs that are views or broadcast, and gradients that arrive expanded (a sum's), give what contiguous ones do."""
    rng = np.random.default_rng(6)
    plan, x, y, w = _setup(pkg, rng, 9, 4, 2, 16, 64, torch.float32)
    base = torch.randn((64,), device="cuda", requires_grad=True)
    wb = torch.randn((2,), device="cuda", requires_grad=True)
    xs = pkg.moe_dispatch(base.expand(9, 64), plan)
    out = pkg.moe_combine(xs, plan, wb.expand(9, 2))
    gb, gw = torch.autograd.grad(out.sum(), [base, wb])
    live = (plan["row_slot"] >= 0).double()
    wbd = wb.detach().double()
    # 18 terms a column of gb; 64 x 9 terms an element of gw: as many roundings of 2^-24 of the magnitudes
    assert float((gb.double() - (live * wbd).sum()).abs().max()) <= 2.0 ** -24 * 20 * float(9 * wbd.abs().sum())
    want = live.sum(0) * base.detach().double().sum()
    assert float((gw.double() - want).abs().max()) <= 2.0 ** -24 * 80 * float(9 * base.detach().abs().sum())
    wide = torch.randn((9, 128), device="cuda")
    assert torch.equal(pkg.moe_dispatch(wide[:, ::2], plan), pkg.moe_dispatch(wide[:, ::2].contiguous(), plan))
    odd = torch.randn(9 * 64 + 1, device="cuda")[1:].view(9, 64)
    assert torch.equal(pkg.moe_dispatch(odd, plan), pkg.moe_dispatch(odd.clone(), plan))


def test_only_what_is_asked(pkg, gpu):
    rng = np.random.default_rng(7)
    plan, x, y, w = _setup(pkg, rng, 6, 4, 2, 16, 64, torch.float32)
    out = pkg.moe_combine(y, plan, w.requires_grad_(True))
    gw, = torch.autograd.grad(out.sum(), [w])
    assert gw.shape == w.shape
    out = pkg.moe_combine(y.requires_grad_(True), plan, w.detach())
    gy, = torch.autograd.grad(out.sum(), [y])
    assert gy.shape == y.shape
    assert not pkg.moe_dispatch(x, plan).requires_grad
    out = pkg.moe_combine(y, plan, w)
    gy, = torch.autograd.grad(out.sum(), [y], create_graph=True)
    with pytest.raises(RuntimeError):                       # first order only
        gy.sum().backward()


def test_rows_outside_the_buffers_count_as_none(pkg, gpu):
    T, k, D = 3, 2, 32
    plan = {"tok_row": torch.tensor([0, 7, -1, 2, -9, 1], dtype=torch.int32, device="cuda"),
            "row_slot": torch.tensor([[0, 99], [5, -4], [3, 6]], dtype=torch.int32, device="cuda")}
    x = torch.randn((T, D), device="cuda")
    xs = pkg.moe_dispatch(x, plan)
    assert torch.equal(xs[[0, 3, 5]], x[[0, 2, 1]]) and (xs[[1, 2, 4]] == 0).all()
    y = torch.randn((6, D), device="cuda")
    w = torch.ones((T, k), device="cuda")
    assert torch.equal(pkg.moe_combine(y, plan, w), y[[0, 5, 3]])


@pytest.mark.parametrize("T,E,k,tm,D", [(5, 4, 2, 1, 8), (40, 8, 3, 16, 136), (300, 6, 17, 40, 520)])
def test_slots_taken_out_of_a_plan(pkg, gpu, T, E, k, tm, D):
    """Slots dropped by the caller (row_slot -1): their rows are zeros in xs and dy, their weights' gradients zero, the
    others as before."""
    rng = np.random.default_rng(T)
    plan, x, y, w = _setup(pkg, rng, T, E, k, tm, D, torch.float32)
    gone = torch.from_numpy(rng.random((T, k)) < 0.4).cuda()
    gone[0], gone[1] = True, False                        # a token that keeps none, one that keeps all
    slot = plan["row_slot"]
    plan["row_slot"] = torch.where(gone, -1, slot)
    y.requires_grad_(), w.requires_grad_()
    out = pkg.moe_combine(y, plan, w)
    gout = torch.randn_like(out)
    dy, dw = torch.autograd.grad(out, [y, w], gout)
    want = _want(plan, _np(x), _np(y), _np(w), np.zeros(y.shape), _np(gout))
    assert np.array_equal(_np(pkg.moe_dispatch(x, plan)), want[0])
    _near(out, *want[1], k, torch.float32)
    assert (out[0] == 0).all() and (dw[gone] == 0).all()
    _near(dy, want[3], np.abs(want[3]), 1, torch.float32)
    _near(dw, *want[4], D, torch.float32)


def test_training_step_captured(pkg, gpu):
    """Forward and backward of the pair in one captured graph, replayed three times with new inputs."""
    rng = np.random.default_rng(9)
    plan, x, y, w = _setup(pkg, rng, 40, 8, 2, 16, 136, torch.bfloat16)
    sx, sw, gout = x.clone(), w.clone(), torch.randn_like(x)

    def step(x0, w0, g0):
        x1, w1 = x0.detach().requires_grad_(True), w0.detach().requires_grad_(True)
        out = pkg.moe_combine(pkg.moe_dispatch(x1, plan) * 2.0, plan, w1)
        return (out.detach(),) + torch.autograd.grad(out, [x1, w1], g0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(sx, sw, gout)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step(sx, sw, gout)
    for _ in range(3):
        nx, nw, ng = torch.randn_like(x), torch.randn_like(w), torch.randn_like(gout)
        sx.copy_(nx), sw.copy_(nw), gout.copy_(ng)
        want = step(nx, nw, ng)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
