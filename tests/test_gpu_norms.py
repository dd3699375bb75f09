"""GPU: rms_norm and fp8_rms_norm against plain implementations in 64 bits, their gradients against the formula's and against
differences, strided and odd rows, captured and on several streams."""
import threading

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}      # half a step, relative
EPS = 1e-5


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(shape, device="cuda", generator=g) * scale
    if len(shape) and shape[-1] > 3:
        x[..., 3] *= 20.0                                           # a large channel
    return x.to(dtype)


def _chain(x, w, eps, residual=None):
    """The documented steps: the stream, r rounded to f32, and both products rounded to f32."""
    s = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    v = s.float()
    r = (1.0 / torch.sqrt(v.double().square().mean(-1, keepdim=True) + eps)).float()
    return s, r, (v * r) * w.float()


def _near(got, want, terms, bound):
    """|got - want| <= bound * terms, elementwise (a NaN fails)."""
    assert got.shape == want.shape
    assert bool(((got.double() - want.double()).abs() <= bound * terms.double() + 1e-300).all()), \
        float(((got.double() - want.double()).abs() / (terms.double() + 1e-300)).max() / bound)


SHAPES = [(1, 8), (3, 16), (5, 128), (2, 136), (17, 512), (9, 520), (4, 1024), (7, 1032), (3, 2048), (2, 4096), (5, 4104), (3, 6144),
          (2, 8192), (2, 8200), (2, 16392), (2, 32768), (700, 264), (1100, 6144)]


@pytest.mark.parametrize("T,D", SHAPES)
@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32), (torch.bfloat16, torch.float32)])
def test_forward(pkg, gpu, T, D, dtype, wdtype):
    """Every step is one rounding of the exact value of its inputs, so the bits are the documented chain's."""
    x, res, w = _rand((T, D), dtype, 1), _rand((T, D), dtype, 2, 3.0), _rand((D,), wdtype, 3)
    y = pkg.rms_norm(x, w, EPS)
    assert torch.equal(y, _chain(x, w, EPS)[2].to(dtype)) and y.dtype is dtype
    s, _, want = _chain(x, w, EPS, res)
    y, stream = pkg.rms_norm(x, w, EPS, residual=res)
    assert torch.equal(stream, s) and torch.equal(y, want.to(dtype))
    if D % 16 == 0:
        (q, qs), stream, yy = pkg.fp8_rms_norm(x, w, EPS, residual=res, want_y=True)
        wq, ws = pkg.fp8_quantize(want)
        assert torch.equal(stream, s) and torch.equal(yy, y)
        assert torch.equal(q.view(torch.uint8), wq.view(torch.uint8)) and torch.equal(qs, ws)
        (q, qs), stream, yy = pkg.fp8_rms_norm(x, w, EPS)
        wq, ws = pkg.fp8_quantize(_chain(x, w, EPS)[2])
        assert stream is None and yy is None
        assert torch.equal(q.view(torch.uint8), wq.view(torch.uint8)) and torch.equal(qs, ws)


def _grad_want(x, w, res, gy, gs):
    """The gradients in 64 bits, and the magnitudes that are added in each."""
    s = x.double() if res is None else (x.double() + res.double()).to(x.dtype).double()
    r = 1.0 / torch.sqrt(s.square().mean(-1, keepdim=True) + EPS)
    n, g = s * r, gy.double() * w.double()
    dot, mag = (g * n).mean(-1, keepdim=True), (g * n).abs().mean(-1, keepdim=True)
    ds = r * (g - n * dot) + (0.0 if gs is None else gs.double())
    terms = r * (g.abs() + n.abs() * mag) + (0.0 if gs is None else gs.double().abs())
    return ds, terms, (gy.double() * n).sum(0), (gy.double() * n).abs().sum(0)


@pytest.mark.parametrize("T,D", SHAPES)
@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32), (torch.float32, torch.bfloat16)])
def test_gradients(pkg, gpu, T, D, dtype, wdtype):
    x, res, w = _rand((T, D), dtype, 1), _rand((T, D), dtype, 2, 3.0), _rand((D,), wdtype, 3)
    gy, gs = _rand((T, D), dtype, 4), _rand((T, D), dtype, 5)
    for r, g in ((None, None), (res, gs), (res, None)):
        leaves = [t.detach().requires_grad_() for t in ((x, w) if r is None else (x, w, r))]
        out = pkg.rms_norm(leaves[0], leaves[1], EPS, residual=None if r is None else leaves[2])
        outs, gouts = ([out], [gy]) if r is None else (list(out), [gy, g]) if g is not None else ([out[0]], [gy])
        got = torch.autograd.grad(outs, leaves, gouts)
        ds, terms, dw, dwterms = _grad_want(x, w, r, gy, g)
        # f32: r, n, g, the mean of D terms (a lane's 32, then 10 levels of a tree), three more operations
        f32 = 2.0 ** -24 * 52
        _near(got[0], ds, terms, f32 + HALF[dtype])
        # dw: T terms in a workgroup's turn (at most 4 of a lane and 512 partial sums), each from n of three roundings
        _near(got[1], dw, dwterms, 2.0 ** -24 * (min(T, 90) + 90) + HALF[wdtype])
        assert got[0].dtype is dtype and got[1].dtype is wdtype
        if r is not None:
            assert torch.equal(got[2], got[0])


def test_gradient_against_differences(pkg, gpu):
    x, res, w = _rand((3, 24), torch.float32, 1), _rand((3, 24), torch.float32, 2), _rand((24,), torch.float32, 3)
    gy, gs = _rand((3, 24), torch.float32, 4), _rand((3, 24), torch.float32, 5)
    leaves = [t.detach().requires_grad_() for t in (x, w, res)]
    got = torch.autograd.grad(list(pkg.rms_norm(leaves[0], leaves[1], EPS, residual=leaves[2])), leaves, [gy, gs])

    def f(x, w, res):
        s = x.double() + res.double()
        y = s / torch.sqrt(s.square().mean(-1, keepdim=True) + EPS) * w.double()
        return float((y * gy).sum() + (s * gs).sum())

    h = 2.0 ** -10
    for k, t in enumerate((x, w, res)):
        for at in (0, 3, 11, t.numel() - 1):
            args = [a.double() for a in (x, w, res)]
            up, lo = [a.clone() for a in args], [a.clone() for a in args]
            up[k].view(-1)[at] += h
            lo[k].view(-1)[at] -= h
            d = (f(*up) - f(*lo)) / (2 * h)
            # the third derivative's h^2 / 6 (values of a few units), and f32
            assert abs(float(got[k].view(-1)[at]) - d) <= 1e-4 * (1.0 + abs(d))


def test_shapes_strides_and_outputs(pkg, gpu):
    w = _rand((256,), torch.bfloat16, 1)
    x = _rand((4, 5, 256), torch.bfloat16, 2)
    want = pkg.rms_norm(x.reshape(20, 256), w).view(4, 5, 256)
    assert torch.equal(pkg.rms_norm(x, w), want) and torch.equal(pkg.rms_norm(x[2, 3], w), want[2, 3])
    wide = _rand((20, 1024), torch.bfloat16, 3)
    for view in (wide[:, 256:512], wide[:, 4:260], wide[::2, 8:264], wide[:, ::4], wide[3:4, 1:257], wide[:1, 512:768],
                 _rand((256, 20), torch.bfloat16, 4).t(), _rand((1, 256), torch.bfloat16, 5).expand(20, 256)):
        dense = view.contiguous()
        assert torch.equal(pkg.rms_norm(view, w), pkg.rms_norm(dense, w))
        a, b = pkg.rms_norm(view, w, residual=view), pkg.rms_norm(dense, w, residual=dense)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        q, p = pkg.fp8_rms_norm(view, w), pkg.fp8_rms_norm(dense, w)
        assert torch.equal(q[0][0].view(torch.uint8), p[0][0].view(torch.uint8)) and torch.equal(q[0][1], p[0][1])
        # gradients arrive broadcast, inputs are views
        a, b = view.detach().requires_grad_(), dense.detach().requires_grad_()
        ga, = torch.autograd.grad(pkg.rms_norm(a, w).sum(), a)
        gb, = torch.autograd.grad(pkg.rms_norm(b, w).sum(), b)
        assert torch.equal(ga, gb)
    odd = _rand((256 * 3 + 1,), torch.float32, 6)[1:].view(3, 256)          # an address that is no multiple of 16
    assert torch.equal(pkg.rms_norm(odd, w[::1]), pkg.rms_norm(odd.clone(), w))
    y, s = torch.empty_like(x), torch.empty_like(x)
    got = pkg.rms_norm(x, w, residual=x, y=y, stream=s)
    assert got[0] is y and got[1] is s and torch.equal(s, x * 2)
    base = _rand((256,), torch.bfloat16, 7).requires_grad_()                # a broadcast input's gradient is summed
    g, = torch.autograd.grad(pkg.rms_norm(base.expand(6, 256), w).float().sum(), base)
    one = base.detach().requires_grad_()
    g1, = torch.autograd.grad(pkg.rms_norm(one, w).float().sum(), one)
    _near(g, 6 * g1.double(), 6 * g1.double().abs(), 6 * 2.0 ** -8)


def test_no_rows(pkg, gpu):
    w = torch.ones(64, device="cuda", requires_grad=True)
    x = torch.empty((0, 64), device="cuda", requires_grad=True)
    y, s = pkg.rms_norm(x, w, residual=torch.empty((0, 64), device="cuda"))
    assert y.shape == s.shape == (0, 64)
    gx, gw = torch.autograd.grad([y, s], [x, w], [torch.empty_like(y), torch.empty_like(s)])
    assert gx.shape == (0, 64) and (gw == 0).all()
    (q, qs), _, _ = pkg.fp8_rms_norm(x.detach(), w.detach())
    assert q.shape == (0, 64) and qs.shape == (0, 1)


def test_values_at_the_ends(pkg, gpu):
    """Zeros, tiny and huge values (whose squares leave f32), infinities and NaN: each in its own row."""
    x = _rand((8, 256), torch.float32, 1)
    x[1] = 0.0
    x[2] *= 1e-30
    x[3] *= 1e37
    x[4, 7] = float("inf")
    x[5, 9] = float("nan")
    w = _rand((256,), torch.float32, 2)
    for eps in (EPS, 0.0):
        want = _chain(x, w, eps)[2]
        y = pkg.rms_norm(x, w, eps)
        assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(y.nan_to_num(), want.nan_to_num())
        assert torch.isfinite(y[3]).all() and torch.isfinite(y[[0, 6, 7]]).all()
    (q, qs), _, _ = pkg.fp8_rms_norm(x, w, EPS)
    wq, ws = pkg.fp8_quantize(_chain(x, w, EPS)[2])
    assert torch.equal(q.float().nan_to_num(999.0), wq.float().nan_to_num(999.0)) and torch.equal(qs, ws)
    lv = x.detach().requires_grad_()
    g, = torch.autograd.grad(pkg.rms_norm(lv, w).sum(), lv)
    ds = _grad_want(x, w, None, torch.ones_like(x), None)[0]
    clean = [0, 3, 6, 7]
    assert torch.isfinite(g[clean]).all() and torch.isnan(g[5]).all()
    _near(g[clean], ds[clean], _grad_want(x, w, None, torch.ones_like(x), None)[1][clean], 2.0 ** -24 * 60)


def test_only_what_is_asked(pkg, gpu):
    x, w, res = _rand((6, 64), torch.float32, 1), _rand((64,), torch.float32, 2), _rand((6, 64), torch.float32, 3)
    full = [t.detach().requires_grad_() for t in (x, w, res)]
    want = torch.autograd.grad(pkg.rms_norm(full[0], full[1], EPS, residual=full[2])[0].sum(), full)
    for k in range(3):
        t = [a.detach() for a in (x, w, res)]
        t[k] = t[k].requires_grad_()
        y, s = pkg.rms_norm(t[0], t[1], EPS, residual=t[2])
        g, = torch.autograd.grad(y.sum(), [t[k]])
        assert torch.equal(g, want[k])
    a = x.detach().requires_grad_()                                # the stream alone
    g, = torch.autograd.grad(pkg.rms_norm(a, w, EPS, residual=res)[1].sum(), a)
    assert (g == 1).all()
    with torch.no_grad():
        assert not pkg.rms_norm(a, w).requires_grad
    y = pkg.rms_norm(a, w)
    g, = torch.autograd.grad(y.sum(), a, create_graph=True)
    with pytest.raises(RuntimeError):                               # first order only
        g.sum().backward()


def test_refusals(pkg, gpu):
    x, w = torch.randn((4, 64), device="cuda"), torch.ones(64, device="cuda")
    for bad, err in ((lambda: pkg.rms_norm(x.half(), w), TypeError), (lambda: pkg.rms_norm(x, w.half()), TypeError),
                     (lambda: pkg.rms_norm(x, w[:8]), ValueError), (lambda: pkg.rms_norm(x, w, -1.0), ValueError),
                     (lambda: pkg.rms_norm(x, w, float("nan")), ValueError),
                     (lambda: pkg.rms_norm(x, w, residual=x[:2]), ValueError),
                     (lambda: pkg.rms_norm(x, w, residual=x.bfloat16()), ValueError),
                     (lambda: pkg.rms_norm(x, w, y=x[:2]), ValueError), (lambda: pkg.rms_norm(x, w, stream=x), ValueError),
                     (lambda: pkg.rms_norm(x, w.cpu()), ValueError),
                     (lambda: pkg.rms_norm(x[:, :12].contiguous(), w[:12]), pkg._lib.MiError),
                     (lambda: pkg.fp8_rms_norm(x[:, :24].contiguous(), w[:24]), pkg._lib.MiError),
                     (lambda: pkg.rms_norm(torch.ones((1, 32776), device="cuda"), torch.ones(32776, device="cuda")), pkg._lib.MiError),
                     (lambda: pkg.rms_norm(x.requires_grad_(), w, y=torch.empty_like(x)), RuntimeError),
                     (lambda: pkg.fp8_rms_norm(x.requires_grad_(), w), RuntimeError)):
        with pytest.raises(err):
            bad()
        x = x.detach()
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for f in (lambda: pkg.rms_norm(d, w), lambda: pkg.fp8_rms_norm(d, w), lambda: pkg.rms_norm(x, w, residual=d)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                f()


def _step(pkg, x, w, res, gy, gs):
    x, w, res = [t.detach().requires_grad_() for t in (x, w, res)]
    y, s = pkg.rms_norm(x, w, EPS, residual=res)
    return (y.detach(), s.detach()) + torch.autograd.grad([y, s], [x, w, res], [gy, gs])


def test_training_step_captured(pkg, gpu):
    make = lambda k: [_rand((40, 520), torch.bfloat16, k), _rand((520,), torch.bfloat16, k + 1), *[  # noqa: E731
        _rand((40, 520), torch.bfloat16, k + j) for j in (2, 3, 4)]]
    held = make(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(pkg, *held)
    torch.cuda.current_stream().wait_stream(side)
    g, h = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = _step(pkg, *held)
    with torch.cuda.graph(h):
        outs2 = _step(pkg, *held)
    for k in range(1, 4):
        new = make(10 * k)
        for a, b in zip(held, new):
            a.copy_(b)
        want = _step(pkg, *new)
        g.replay()
        h.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)) and all(torch.equal(a, b) for a, b in zip(outs2, want))


def test_streams_and_threads(pkg, gpu):
    work = [[_rand((T, 256), torch.bfloat16, T + j) if j != 1 else _rand((256,), torch.bfloat16, T) for j in range(5)]
            for T in (1, 60, 300, 7)]
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


def test_rows_past_32_bits(pkg, gpu):
    """More than 2^31 elements: the last rows are those of a small call."""
    T, D = 140000, 16384
    x = torch.empty((T, D), dtype=torch.bfloat16, device="cuda")
    x[:] = _rand((D,), torch.bfloat16, 1)
    x[-3:] = _rand((3, D), torch.bfloat16, 2)
    w = _rand((D,), torch.bfloat16, 3)
    y = pkg.rms_norm(x, w)
    assert torch.equal(y[-3:], pkg.rms_norm(x[-3:].clone(), w)) and torch.equal(y[70000], pkg.rms_norm(x[0], w))
