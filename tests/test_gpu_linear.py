"""GPU: bf16_linear against products in 64 bits: every tile, split and the streaming form, epilogues, odd sizes and strides, its
gradients against the formula's and against differences, captured and on several streams."""
import math
import threading

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
ACTS = [None, "silu", "gelu", "gelu_tanh", "relu"]


def _rand(shape, seed, scale=1.0, dtype=BF16):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (scale * torch.randn(shape, device="cuda", generator=g)).to(dtype)


def _act(z, name):
    """The activation and its derivative in 64 bits."""
    if name == "relu":
        return z.clamp_min(0), (z > 0).double()
    if name == "silu":
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p))
    if name == "gelu":
        p = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        a = math.sqrt(2 / math.pi)
        t = torch.tanh(a * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * 0.044715 * z * z)
    return z, torch.ones_like(z)


def _forward(x, wT, bias, act, res):
    """y in 64 bits, z, and how far f32 may be from z (err) and y (yerr)."""
    z = x.double() @ wT.double().t()
    mag = x.double().abs() @ wT.double().abs().t()
    if bias is not None:
        z, mag = z + bias.double(), mag + bias.double().abs()
    # f32 sums of n_in exact products: of an instruction's 32, then one addition per instruction, split or wavefront
    err = 2.0 ** -24 * (x.shape[1] / 32 + 48) * mag
    a, d = _act(z, act)
    # |act'| <= 1.13; the activation itself: 8 roundings, e^x within |x| 2^-24 (and 2^-24), Phi within 7.5e-8 (gelu)
    yerr = err if act in (None, "relu") else 1.13 * err + 2.0 ** -24 * (16 + 2 * z.abs()) * a.abs() + (8e-8 * z.abs() if act == "gelu" else 0)
    # gelu_tanh: the inner polynomial's roundings, 4 of 1.6 |z| (1 + 0.045 z^2), through sigmoid' <= 1/4 times |z|; past 8 it is 0 or z
    if act == "gelu_tanh":
        zc = z.abs().clamp_max(8.0)
        yerr = yerr + 2.0 ** -24 * 4 * zc * 0.25 * 1.6 * zc * (1 + 0.045 * zc * zc)
    if res is not None:
        a = a + res.double()
        yerr = yerr + 2.0 ** -24 * a.abs()
    return a, z, err, yerr, d


def _near(got, want, err, what=""):
    half = 2.0 ** -8 if got.dtype is BF16 else 2.0 ** -24
    bad = (got.double() - want).abs() - (err * (1 + half) + half * want.abs() + 1e-38)
    assert got.shape == want.shape and bool((bad <= 0).all()), (what, float(bad.max()), float(want.abs().max()))


def _check(pkg, B, K, R, bias=False, act=None, res=False, dtype=BF16, seed=0, **kw):
    x, wT = _rand((B, K), seed + 1), _rand((R, K), seed + 2, 1.5 / math.sqrt(K))
    b = _rand((R,), seed + 3) if bias else None
    r = _rand((B, R), seed + 4, 3.0, dtype) if res else None
    y = pkg.bf16_linear(x, pkg.Bf16Leaf(wT), bias=b, act=act, residual=r, dtype=dtype, **kw)
    assert y.dtype is dtype
    want, _, _, yerr, _ = _forward(x, wT, b, act, r)
    _near(y, want, yerr, (B, K, R, bias, act, res, dtype))
    return x, wT, b, r, y


SIZES = [(1, 8, 1), (1, 64, 16), (2, 72, 33), (3, 1000, 20), (16, 4096, 130), (5, 8, 4), (4, 6144, 6144), (17, 64, 64), (33, 520, 77),
         (64, 128, 256), (65, 1032, 129), (100, 2048, 300), (129, 264, 515), (300, 640, 1030), (37, 6144, 2051), (517, 200, 2048),
         (700, 1360, 592), (2100, 264, 2052), (4096, 64, 8)]


@pytest.mark.parametrize("B,K,R", SIZES)
def test_forward(pkg, gpu, B, K, R):
    _check(pkg, B, K, R)
    _check(pkg, B, K, R, res=True, dtype=F32)
    _check(pkg, B, K, R, bias=True, act="silu", res=True)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("B,R", [(1, 48), (7, 50), (40, 131), (300, 260)])
def test_epilogues(pkg, gpu, act, B, R):
    for bias in (False, True):
        for res in (False, True):
            for dtype in (BF16, F32):
                _check(pkg, B, 136, R, bias, act, res, dtype)


TILES = [(128, 64), (128, 128), (256, 128), (256, 256), (192, 256)]


@pytest.mark.parametrize("tw,tt", TILES)
@pytest.mark.parametrize("S", [1, 2, 3, 8])
@pytest.mark.parametrize("B,K,R", [(17, 520, 40), (70, 1992, 400), (300, 712, 515), (530, 136, 772)])
def test_every_tile_and_split(pkg, gpu, tw, tt, S, B, K, R):
    """Each tile of the forward product and (but for the first-form one) of the gradients', with every count of splits."""
    with pkg.tuning(LIN_TW=tw, LIN_TT=tt, LIN_S=S, LIN_STREAM=0):
        _check(pkg, B, K, R, bias=True, act="gelu", res=True)
        x, wT, _, _, _ = _check(pkg, B, K, R)
        if tw != 192:
            _grads(pkg, x, wT, None, None, None, BF16)


def _grads(pkg, x, wT, b, act, r, dtype, seed=50):
    leaves = {n: t.detach().requires_grad_() for n, t in (("x", x), ("w", wT), ("b", b), ("r", r)) if t is not None}
    y = pkg.bf16_linear(leaves["x"], pkg.Bf16Leaf(leaves["w"]), bias=leaves.get("b"), act=act, residual=leaves.get("r"), dtype=dtype)
    gy = _rand(tuple(y.shape), seed, 1.0, dtype)
    got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), gy)))
    _, z, err, _, d = _forward(x, wT, b, act, r)
    dz = gy.double() * d
    # z's error through act'' (|act''| <= 1.2), act' itself: within 2^-24 (24 + 6 |z|) (and gelu's 7.5e-8); where relu's z is
    # within its error of 0 the derivative may be either
    derr = 1.2 * err + 2.0 ** -24 * (24 + 6 * z.abs().clamp_max(30.0)) + 1e-7 if act not in (None, "relu") else torch.zeros_like(z)
    if act == "gelu_tanh":
        # the inner polynomial u (4 roundings of |u| <= 1.6 z (1 + .045 z^2)): through sigmoid', and sigmoid'' times z u'
        zc = z.abs().clamp_max(8.0)
        u = 1.6 * zc * (1 + 0.045 * zc * zc)
        derr = derr + 2.0 ** -24 * 4 * u * (0.25 + 0.1 * zc * 1.6 * (1 + 0.135 * zc * zc))
    if act == "relu":
        derr = (z.abs() <= err).double()
    # dz is rounded to bf16 for the products, if it is not dy itself; sums in f32
    half = 0.0 if act is None and dtype is BF16 else 2.0 ** -8
    e = gy.double().abs() * derr + half * dz.abs()
    m = dz.abs() + e
    B, K, R = x.shape[0], x.shape[1], wT.shape[0]
    _near(got["x"], dz @ wT.double(), e @ wT.double().abs() + 2.0 ** -24 * (R / 32 + 48) * (m @ wT.double().abs()), "dx")
    _near(got["w"], dz.t() @ x.double(), e.t() @ x.double().abs() + 2.0 ** -24 * (B / 32 + 48) * (m.t() @ x.double().abs()), "dw")
    if b is not None:
        # of dz before its rounding: a lane's rows (B / 8 at most), 8 lanes, up to 64 workgroups
        _near(got["b"], dz.sum(0), (gy.double().abs() * derr + 2.0 ** -24 * (B / 8 + 80) * m).sum(0), "db")
    if r is not None:
        assert torch.equal(got["r"], gy)
    assert all(got[n].dtype is t.dtype and got[n].shape == t.shape for n, t in leaves.items())


@pytest.mark.parametrize("B,K,R", [(1, 8, 1), (1, 64, 16), (3, 72, 33), (16, 520, 130), (17, 64, 64), (40, 1032, 129), (129, 264, 515),
                                   (300, 640, 1030), (600, 512, 768), (2100, 264, 300)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gradients(pkg, gpu, B, K, R, dtype):
    x, wT, b, r = _rand((B, K), 1), _rand((R, K), 2, 1.5 / math.sqrt(K)), _rand((R,), 3), _rand((B, R), 4, 3.0, dtype)
    for act in ACTS:
        _grads(pkg, x, wT, b, act, r, dtype)
    _grads(pkg, x, wT, None, None, None, dtype)
    _grads(pkg, x, wT, None, "silu", r, dtype)


def test_gradient_against_differences(pkg, gpu):
    """At a few values of bf16 inputs: differences of the 64-bit function, with the roundings of dz and of the results."""
    x, wT, b = _rand((3, 16), 1), _rand((9, 16), 2, 0.3), _rand((9,), 3)
    gy = _rand((3, 9), 4, 1.0, F32)
    h = 2.0 ** -12
    for act in ACTS[:4]:
        t = [a.detach().requires_grad_() for a in (x, wT, b)]
        got = torch.autograd.grad(pkg.bf16_linear(t[0], pkg.Bf16Leaf(t[1]), bias=t[2], act=act, dtype=F32), t, gy)
        args = [a.double() for a in (x, wT, b)]
        scale = float(gy.abs().sum()) / 3
        for k in range(3):
            for at in (0, args[k].numel() - 1):
                f = []
                for d in (h, -h):
                    a = [v.clone() for v in args]
                    a[k].view(-1)[at] += d
                    f.append(float((_act(a[0] @ a[1].t() + a[2], act)[0] * gy.double()).sum()))
                want = (f[0] - f[1]) / (2 * h)
                # 2^-8 of the terms (dz) and of the result; the differences' h^2 and 64 bits are far below
                assert abs(float(got[k].view(-1)[at]) - want) <= 2.0 ** -8 * (abs(want) + scale * 3)


def test_far_values(pkg, gpu):
    """Activations and derivatives where their factors leave f32, NaN and infinities in their own rows."""
    K = 64
    x = torch.zeros((8, K), device="cuda", dtype=BF16)
    vals = [0.0, 35.0, -35.0, 1e4, -1e4, 3e38, -3e38, 150.0]
    x[:, 0] = torch.tensor(vals, device="cuda").to(BF16)
    wT = torch.zeros((5, K), device="cuda", dtype=BF16)
    wT[:, 0] = 1.0
    for act in ACTS[1:]:
        for n in (8, 40):
            xx = x.repeat(n // 8, 1)
            lx = xx.detach().requires_grad_()
            y = pkg.bf16_linear(lx, pkg.Bf16Leaf(wT), act=act, dtype=F32)
            z = xx[:, :1].double()
            want = torch.where(z > 0, z, 0.0).expand(-1, 5)
            assert bool(((y.double() - want).abs() <= 2.0 ** -22 * want.abs() + 1e-12).all()), act
            g, = torch.autograd.grad(y, lx, torch.ones_like(y))
            d = torch.where(z > 0, 5.0, torch.where(z < 0, 0.0, 2.5 if act != "relu" else 0.0))
            assert torch.isfinite(g).all() and bool(((g[:, :1].double() - d).abs() <= 2.0 ** -7).all()), act
    for B in (3, 50):
        x, wT, b, r, y = _check(pkg, B, 136, 40, bias=True, act="gelu", res=True)
        x[1, 5] = float("nan")
        x[2, 7] = float("inf")
        y2 = pkg.bf16_linear(x, pkg.Bf16Leaf(wT), bias=b, act="gelu", residual=r)
        keep = torch.arange(B, device="cuda").ne(1) & torch.arange(B, device="cuda").ne(2)
        assert torch.equal(y2[keep], y[keep]) and torch.isnan(y2[1]).all()
        assert torch.isnan(pkg.bf16_linear(x, pkg.Bf16Leaf(wT), act="relu")[1]).all()


def test_rounds_to_nearest_even(pkg, gpu):
    """y in bf16 is y in f32 rounded by torch, subnormal values, large ones and infinities among them."""
    w = torch.zeros((64, 64), device="cuda", dtype=BF16)
    w[:, 0], w[:, 1], w[:, 2] = _rand((64,), 1), _rand((64,), 2, 2.0 ** -7), _rand((64,), 3, 2.0 ** -9)
    for n in (4, 300):
        for scale in (1.0, 2.0 ** -126, 2.0 ** -130, 2.0 ** 126):
            x = (torch.ones((n, 64), device="cuda") * _rand((n, 1), 4, 1.0, F32) * scale).to(BF16)
            yb, yf = pkg.bf16_linear(x, pkg.Bf16Leaf(w)), pkg.bf16_linear(x, pkg.Bf16Leaf(w), dtype=F32)
            assert torch.equal(yb.view(torch.int16), yf.to(BF16).view(torch.int16))


def test_rows_as_they_lie(pkg, gpu):
    """Strided, transposed, broadcast and unaligned inputs; W instead of a leaf; outputs and workspaces of the caller."""
    wT, b = _rand((72, 128), 1, 0.1), _rand((72,), 2)
    leaf = pkg.Bf16Leaf(wT)
    wide = _rand((50, 512), 3)
    for view in (wide[:, 128:256], wide[:, 8:136], wide[::2, 128:256], wide[:, ::4], wide[:, 3:131], _rand((128, 50), 4).t(),
                 _rand((1, 128), 5).expand(50, 128), wide[:3, 128:256]):
        dense = view.contiguous()
        want = pkg.bf16_linear(dense, leaf, bias=b)
        assert torch.equal(pkg.bf16_linear(view, leaf, bias=b), want)
        lx, ly = view.detach().requires_grad_(), dense.detach().requires_grad_()
        lw, lv = wT.detach().requires_grad_(), wT.detach().requires_grad_()
        ga = torch.autograd.grad(pkg.bf16_linear(lx, pkg.Bf16Leaf(lw), act="silu").sum(), [lx, lw])
        gb = torch.autograd.grad(pkg.bf16_linear(ly, pkg.Bf16Leaf(lv), act="silu").sum(), [ly, lv])
        assert all(torch.equal(p, q) for p, q in zip(ga, gb))
    x = wide[:, :128].contiguous()
    want = pkg.bf16_linear(x, leaf)
    assert torch.equal(pkg.bf16_linear(x, wT.t().contiguous()), want)
    assert torch.equal(pkg.bf16_linear(x, pkg.bf16_leaf(wT.t())), want)
    odd = torch.empty(72 * 128 + 1, device="cuda", dtype=BF16)[1:].view(72, 128).copy_(wT)
    assert torch.equal(pkg.bf16_linear(x, pkg.Bf16Leaf(odd)), want)
    for n, R in ((50, 72), (3, 72), (300, 71)):                     # y and the residual at odd addresses
        wv, xv = _rand((R, 128), 6, 0.1), _rand((n, 128), 7)
        buf = torch.zeros(n * R + 3, device="cuda", dtype=BF16)
        y = buf[1:1 + n * R].view(n, R)
        r = _rand((n * R + 1,), 8)[1:].view(n, R)
        got = pkg.bf16_linear(xv, pkg.Bf16Leaf(wv), residual=r, y=y)
        assert got is y and torch.equal(y, pkg.bf16_linear(xv, pkg.Bf16Leaf(wv), residual=r.clone()))
        assert float(buf[0]) == 0 and (buf[1 + n * R:] == 0).all()
    from_w = wT.t().contiguous().requires_grad_()                   # W's own gradient, through the transposition
    g, = torch.autograd.grad(pkg.bf16_linear(x, from_w).sum(), from_w)
    lw = wT.detach().requires_grad_()
    g2, = torch.autograd.grad(pkg.bf16_linear(x, pkg.Bf16Leaf(lw)).sum(), lw)
    assert torch.equal(g, g2.t())
    L = pkg._lib.lib()
    for n in (1, 16, 17, 200, 2000):
        need = L.mi_bf16_linear_workspace(n, 128, 72)
        xv = _rand((n, 128), 9)
        ws = torch.full((max(need, 16),), 0xff, dtype=torch.uint8, device="cuda")
        assert torch.equal(pkg.bf16_linear(xv, leaf, workspace=ws), pkg.bf16_linear(xv, leaf))
    with pytest.raises(pkg._lib.MiError):
        pkg.bf16_linear(x, leaf, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))


def test_workspace_serves_smaller_calls(pkg, gpu):
    L = pkg._lib.lib()
    for K, R in ((128, 72), (6144, 6144), (8192, 8192), (64, 65536)):
        sizes = [L.mi_bf16_linear_workspace(B, K, R) for B in (1, 4, 5, 16, 17, 64, 65, 1000, 1 << 20)]
        assert sizes == sorted(sizes) and L.mi_bf16_linear_workspace(0, K, R) == 0
        sizes = [L.mi_bf16_linear_grad_workspace(B, K, R) for B in (1, 4, 5, 16, 17, 64, 65, 1000, 1 << 20)]
        assert sizes == sorted(sizes) and sizes[0] > 0


def test_no_rows_and_only_what_is_asked(pkg, gpu):
    wT, b = _rand((24, 64), 1).requires_grad_(), _rand((24,), 2).requires_grad_()
    x = torch.empty((0, 64), device="cuda", dtype=BF16, requires_grad=True)
    y = pkg.bf16_linear(x, pkg.Bf16Leaf(wT), bias=b, act="gelu")
    g = torch.autograd.grad(y, [x, wT, b], torch.empty_like(y))
    assert y.shape == (0, 24) and g[0].shape == (0, 64) and (g[1] == 0).all() and (g[2] == 0).all()
    x, r = _rand((30, 64), 3), _rand((30, 24), 4)
    t = [a.detach().requires_grad_() for a in (x, wT, b, r)]
    want = torch.autograd.grad(pkg.bf16_linear(t[0], pkg.Bf16Leaf(t[1]), bias=t[2], act="silu", residual=t[3]).sum(), t)
    for k in range(4):
        t = [a.detach() for a in (x, wT, b, r)]
        t[k] = t[k].requires_grad_()
        g, = torch.autograd.grad(pkg.bf16_linear(t[0], pkg.Bf16Leaf(t[1]), bias=t[2], act="silu", residual=t[3]).sum(), [t[k]])
        assert torch.equal(g, want[k])
    lx = x.detach().requires_grad_()
    with torch.no_grad():
        assert not pkg.bf16_linear(lx, pkg.Bf16Leaf(wT)).requires_grad
    g, = torch.autograd.grad(pkg.bf16_linear(lx, pkg.Bf16Leaf(wT.detach()), act="silu").sum(), lx, create_graph=True)
    with pytest.raises(RuntimeError):                               # first order only
        g.sum().backward()


def test_refusals(pkg, gpu):
    x, leaf = _rand((4, 64), 1), pkg.Bf16Leaf(_rand((24, 64), 2))
    f = pkg.bf16_linear
    for bad, err in ((lambda: f(x.float(), leaf), TypeError), (lambda: f(x[0], leaf), TypeError),
                     (lambda: f(x, leaf.wT.float()), TypeError), (lambda: f(x, leaf, act="tanh"), ValueError),
                     (lambda: f(x[:, :32].contiguous(), leaf), ValueError), (lambda: f(x, leaf, dtype=torch.float16), TypeError),
                     (lambda: f(x, leaf, bias=torch.zeros(24, device="cuda")), ValueError),
                     (lambda: f(x, leaf, bias=_rand((23,), 3)), ValueError),
                     (lambda: f(x, leaf, residual=_rand((4, 23), 3)), ValueError),
                     (lambda: f(x, leaf, residual=_rand((4, 24), 3, 1.0, F32)), ValueError),
                     (lambda: f(x, leaf, y=_rand((3, 24), 3)), ValueError),
                     (lambda: f(x, pkg.Bf16Leaf(leaf.wT.cpu())), ValueError),
                     (lambda: f(x[:, :12].contiguous(), pkg.Bf16Leaf(leaf.wT[:, :12].contiguous())), pkg._lib.MiError),
                     (lambda: f(x.requires_grad_(), leaf, y=_rand((4, 24), 3)), RuntimeError)):
        with pytest.raises(err):
            bad()
        x = x.detach()
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(forward_ad.make_dual(x, torch.ones_like(x)), leaf)


def _step(pkg, x, wT, b, r, gy):
    t = [a.detach().requires_grad_() for a in (x, wT, b, r)]
    y = pkg.bf16_linear(t[0], pkg.Bf16Leaf(t[1]), bias=t[2], act="gelu", residual=t[3])
    return (y.detach(),) + torch.autograd.grad(y, t, gy)


def _work(B, K, R, seed):
    return [_rand((B, K), seed), _rand((R, K), seed + 1, 0.1), _rand((R,), seed + 2), _rand((B, R), seed + 3), _rand((B, R), seed + 4)]


def test_training_steps_captured(pkg, gpu):
    """Two graphs captured one after the other, replayed in turn: neither reads what the other left."""
    held = _work(90, 520, 200, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(pkg, *held)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = _step(pkg, *held)
        graphs.append((g, outs))
    for k in range(1, 4):
        new = _work(90, 520, 200, 10 * k)
        for a, b in zip(held, new):
            a.copy_(b)
        want = _step(pkg, *new)
        for g, outs in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, outs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_streams_and_threads(pkg, gpu):
    work = [_work(B, 520, R, B) for B, R in ((1, 200), (40, 77), (300, 513), (17, 64))]
    want = [_step(pkg, *a) for a in work]
    torch.cuda.synchronize()
    wrong, gate = [], threading.Barrier(2)

    def body(first):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                gate.wait(30)
                for n in range(8):
                    at = (n + first) % len(work)
                    got = _step(pkg, *work[at])
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[at])):
                        wrong.append((first, n))
        except Exception as e:                                     # noqa: BLE001 (a thread's error would be lost)
            wrong.append(e)

    threads = [threading.Thread(target=body, args=(j,)) for j in (0, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not wrong, wrong


@pytest.mark.parametrize("B,K,R", [(40000, 64, 65536), (1 << 20, 2048, 16)])
def test_sizes_past_32_bits(pkg, gpu, B, K, R):
    """More than 2^31 outputs, or inputs: the last rows are those of a small call."""
    x = torch.zeros((B, K), dtype=BF16, device="cuda")
    x[-200:], x[B // 2] = _rand((200, K), 1), _rand((K,), 2)
    wT = _rand((R, K), 3, 0.1)
    y = pkg.bf16_linear(x, pkg.Bf16Leaf(wT))
    for rows in (x[-200:], x[B // 2:B // 2 + 1]):
        want, _, _, yerr, _ = _forward(rows, wT, None, None, None)
        _near(y[-200:] if rows.shape[0] > 1 else y[B // 2:B // 2 + 1], want, yerr)
    assert (y[:100] == 0).all()
