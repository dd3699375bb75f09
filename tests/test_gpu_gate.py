"""GPU: moe_gate against its definition in 64 bits: scores, bias, groups, ties, experts out of service, rows without one, its
gradient against the formula's and against differences, captured and on several streams."""
import math
import threading

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu
TINY = 1e-20


def _logits(T, E, seed, dtype=torch.float32, spread=1.5):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (spread * torch.randn((T, E), device="cuda", generator=g)).to(dtype)


def _bias(E, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000 + seed)
    return 0.1 * torch.randn((E,), device="cuda", generator=g)


def _scores(l, kind):
    l = l.double()
    if kind == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-l))
    m = l.amax(-1, keepdim=True)
    p = torch.exp(l - torch.where(m == -math.inf, 0.0, m))
    return p / p.sum(-1, keepdim=True).clamp_min(1e-300)


def _want(logits, k, scores="sigmoid", bias=None, n_group=1, topk_group=1, group_top=2, norm_topk=True, scaling=1.0):
    """(idx, w, s, whether a slot has an expert) from the definition."""
    T, E = logits.shape
    s = _scores(logits, scores)
    c = s if bias is None else s + bias.double()
    out = logits.double() == -math.inf
    c = torch.where(out, -math.inf, c)
    order = c if bias is not None else torch.where(out, -math.inf, logits.double())
    if n_group > 1:
        best = torch.sort(c.view(T, n_group, -1), dim=-1, descending=True)[0][..., :group_top]
        score = torch.where(best == -math.inf, 0.0, best).sum(-1)
        score = torch.where(best[..., 0] == -math.inf, -math.inf, score)
        kept = torch.sort(score, dim=-1, descending=True, stable=True)[1][:, :topk_group]
        live = torch.zeros((T, n_group), dtype=torch.bool, device="cuda").scatter_(1, kept, True)
        order = torch.where(live[..., None], order.view(T, n_group, -1), -math.inf).reshape(T, E)
    top, idx = torch.sort(order, dim=-1, descending=True, stable=True)
    has, idx = top[:, :k] > -math.inf, idx[:, :k]
    sel = torch.where(has, s.gather(1, idx), 0.0)
    w = sel / (sel.sum(-1, keepdim=True) + TINY) if norm_topk else sel
    return torch.where(has, idx, -1).int(), w * scaling, s, has


def _grad_want(logits, gw, idx, s, has, scores, norm_topk, scaling):
    """The gradient in 64 bits, and the magnitudes that are added in it."""
    at = idx.long().clamp_min(0)
    sel = torch.where(has, s.gather(1, at), 0.0)
    g = torch.where(has, gw.double() * scaling, 0.0)
    if norm_topk:
        S = sel.sum(-1, keepdim=True) + TINY
        ds, mag = (g - (g * sel).sum(-1, keepdim=True) / S) / S, (g.abs() + (g * sel).abs().sum(-1, keepdim=True) / S) / S
    else:
        ds, mag = g, g.abs()
    full, fmag = [torch.zeros_like(s).scatter_add_(1, at, torch.where(has, v, 0.0)) for v in (ds, mag)]
    if scores == "sigmoid":
        return full * s * (1 - s), fmag * s * (1 - s)
    return s * (full - (full * s).sum(-1, keepdim=True)), s * (fmag + (fmag * s).sum(-1, keepdim=True))


def _check(pkg, logits, k, **kw):
    idx, w = pkg.moe_gate(logits, k, **kw)
    widx, ww, s, has = _want(logits, k, **kw)
    assert idx.dtype is torch.int32 and w.dtype is torch.float32 and idx.shape == w.shape == (logits.shape[0], k)
    assert torch.equal(idx, widx), int((idx != widx).sum())
    # exp, the sum over up to 1024 experts (16 of a lane, 6 levels), the reciprocal, k slots' sum and three more roundings;
    # exp's argument l - m is rounded too: 2^-24 |l - m|
    far = float(logits.float().nan_to_num(neginf=0.0).abs().max()) * 2
    assert bool(((w.double() - ww).abs() <= 2.0 ** -24 * (48 + 2 * far) * ww.abs() + 1e-37).all())
    return idx, w, s, has


CONFIGS = [(1, 64, 8, 1, 1), (3, 64, 8, 1, 1), (5, 1, 1, 1, 1), (17, 9, 9, 1, 1), (33, 33, 32, 1, 1), (40, 40, 5, 1, 1),
           (65, 100, 7, 1, 1), (130, 129, 4, 1, 1), (7, 255, 8, 1, 1), (300, 256, 8, 8, 4), (31, 256, 8, 8, 3), (19, 160, 6, 8, 3),
           (12, 96, 4, 4, 2), (9, 64, 8, 16, 2), (11, 64, 2, 32, 1), (6, 64, 32, 2, 2), (23, 257, 8, 1, 1), (13, 512, 22, 8, 4),
           (5, 1024, 32, 1, 1), (6, 1024, 8, 32, 4), (4, 1000, 8, 8, 4), (2, 32, 1, 32, 1), (20000, 64, 6, 1, 1)]


@pytest.mark.parametrize("T,E,k,G,tg", CONFIGS)
@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_forward_and_gradient(pkg, gpu, T, E, k, G, tg, scores, dtype):
    for n, (bias, norm, scaling, top) in enumerate(((None, True, 1.0, 2), (_bias(E, T), True, 2.5, 2), (_bias(E, E), False, 1.0, 1))):
        logits = _logits(T, E, T + E + n, dtype)
        kw = dict(scores=scores, bias=bias, n_group=G, topk_group=tg, group_top=top, norm_topk=norm, scaling=scaling)
        idx, w, s, has = _check(pkg, logits, k, **kw)
        leaf = logits.detach().requires_grad_()
        i2, w2 = pkg.moe_gate(leaf, k, **kw)
        assert torch.equal(i2, idx) and torch.equal(w2, w) and not i2.requires_grad
        gw = _logits(T, k, 7)
        got, = torch.autograd.grad(w2, leaf, gw)
        want, mag = _grad_want(logits, gw, idx, s, has, scores, norm, scaling)
        half = 2.0 ** -8 if dtype is torch.bfloat16 else 0.0
        assert got.dtype is dtype
        # f32: s to 48 + 2 |l - m| roundings as above, twice, the sums over k, and a few more
        far = 2 * float(logits.float().abs().max())
        assert bool(((got.double() - want).abs() <= (2.0 ** -24 * (128 + 4 * far) + half) * mag + 1e-37).all())


def test_gradient_against_differences(pkg, gpu):
    T, E, k = 4, 20, 5
    logits, gw, h = _logits(T, E, 3), _logits(T, k, 4), 2.0 ** -12
    for kw in (dict(scores="sigmoid"), dict(scores="softmax"), dict(scores="softmax", norm_topk=False, scaling=3.0),
               dict(scores="sigmoid", norm_topk=False)):
        leaf = logits.detach().requires_grad_()
        idx, w = pkg.moe_gate(leaf, k, **kw)
        got, = torch.autograd.grad(w, leaf, gw)
        for t in range(T):
            for e in [int(idx[t, 0]), int(idx[t, k - 1]), *[e for e in range(E) if e not in idx[t].tolist()][:2]]:
                f = []
                for d in (h, -h):
                    l = logits.double().clone()
                    l[t, e] += d
                    s = _scores(l, kw["scores"])[t][idx[t].long()]
                    v = (s / (s.sum() + TINY) if kw.get("norm_topk", True) else s) * kw.get("scaling", 1.0)
                    f.append(float((v * gw[t].double()).sum()))
                # the third derivative's h^2 / 6 and f32
                assert abs(float(got[t, e]) - (f[0] - f[1]) / (2 * h)) <= 1e-6 + 1e-5 * abs(float(got[t, e]))


@pytest.mark.parametrize("E,k,G,tg", [(64, 8, 1, 1), (256, 8, 8, 4), (1024, 32, 1, 1)])
@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
def test_ties_go_to_the_lower_id(pkg, gpu, E, k, G, tg, scores):
    for bias in (None, torch.zeros(E, device="cuda"), torch.full((E,), -3.0, device="cuda")):
        kw = dict(scores=scores, bias=bias, n_group=G, topk_group=tg)
        for logits in (torch.zeros((3, E), device="cuda"), torch.full((2, E), -0.0, device="cuda"),
                       (_logits(50, E, 5) * 2).round() / 2, torch.full((1, E), 5.0, device="cuda")):
            idx, w, _, _ = _check(pkg, logits, k, **kw)
        assert torch.equal(idx, torch.arange(k, device="cuda", dtype=torch.int32)[None])
    mixed = torch.zeros((1, E), device="cuda")
    mixed[0, ::2] = -0.0                                            # the same value
    assert torch.equal(pkg.moe_gate(mixed, k, scores=scores, n_group=G, topk_group=tg)[0][0], torch.arange(k, device="cuda", dtype=torch.int32))


def test_choices_that_f32_scores_would_confuse(pkg, gpu):
    """Choices 2^-33 apart: equal in f32, told apart in 64 bits; the order is that of the definition."""
    E, k = 64, 8
    logits = _logits(400, E, 9)
    c = 0.75
    bias = (c - _scores(logits[:1], "sigmoid")[0]).float()          # row 0: every choice within 2^-25 of 0.75
    _check(pkg, logits, k, bias=bias)
    gaps = torch.sort(_scores(logits[:1], "sigmoid")[0] + bias.double(), descending=True)[0].diff().abs()
    assert float(gaps.min()) > 2.0 ** -42 and float(gaps.max()) < 2.0 ** -23      # (what the definition can tell apart)


@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,k,G,tg", [(64, 8, 1, 1), (256, 8, 8, 4), (100, 7, 1, 1)])
def test_experts_out_of_service(pkg, gpu, scores, E, k, G, tg):
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    logits = _logits(64, E, 11)
    share = torch.rand((64, 1), device="cuda", generator=g)
    logits[torch.rand((64, E), device="cuda", generator=g) < share] = -math.inf
    logits[0] = -math.inf                                           # a row without an expert
    logits[1] = -math.inf
    logits[1, E - 1] = 2.0                                          # one with a single one
    logits[2] = torch.finfo(torch.float32).min                      # the lowest value is a logit like any other
    logits[3, : E // 2] = torch.finfo(torch.float32).min
    for bias in (None, _bias(E, 1) + 0.5):
        for norm in (True, False):
            kw = dict(scores=scores, bias=bias, n_group=G, topk_group=tg, norm_topk=norm)
            idx, w, s, has = _check(pkg, logits, k, **kw)
            assert (idx[0] == -1).all() and (w[0] == 0).all()
            assert int(idx[1, 0]) == E - 1 and (idx[1, 1:] == -1).all() and (w[1, 1:] == 0).all()
            leaf = logits.detach().requires_grad_()
            gw = _logits(64, k, 7)
            got, = torch.autograd.grad(pkg.moe_gate(leaf, k, **kw)[1], leaf, gw)
            want, mag = _grad_want(logits, gw, idx, s, has, scores, norm, 1.0)
            assert torch.isfinite(got).all() and (got[0] == 0).all()
            rows = torch.arange(64, device="cuda") > 3              # (the others: |l - m| is past any bound)
            far = 2 * float(logits[rows].nan_to_num(neginf=0.0).abs().max())
            assert bool(((got.double() - want).abs() <= 2.0 ** -24 * (128 + 4 * far) * mag + 1e-37)[rows].all())
    # a plan and the routed sum take such slots as nothing
    idx, w = pkg.moe_gate(logits, k, scores=scores, n_group=G, topk_group=tg)
    plan = pkg.ragged_plan(idx, w, E, 16)
    x = torch.randn((64, 64), device="cuda")
    out = pkg.moe_combine(pkg.moe_dispatch(x, plan), plan, w)
    assert (out[0] == 0).all() and torch.equal(plan["row_slot"] < 0, idx < 0)


def test_values_that_are_no_numbers(pkg, gpu):
    logits = _logits(6, 64, 13)
    logits[1, 40] = float("nan")
    logits[2, 10] = float("inf")
    logits[3] = float("nan")
    logits[4, :60] = -math.inf
    logits[4, 62] = float("nan")
    clean = [0, 5]
    for scores in ("sigmoid", "softmax"):
        for bias in (None, _bias(64, 3)):
            for G, tg in ((1, 1), (4, 2)):
                kw = dict(scores=scores, bias=bias, n_group=G, topk_group=tg)
                idx, w = pkg.moe_gate(logits, 8, **kw)
                want = pkg.moe_gate(logits[clean].contiguous(), 8, **kw)
                assert torch.equal(idx[clean], want[0]) and torch.equal(w[clean], want[1])
                for t in range(6):                                  # ids stay valid and distinct
                    ids = [i for i in idx[t].tolist() if i >= 0]
                    assert len(set(ids)) == len(ids) and all(i < 64 for i in ids)
                # an infinite logit is the largest; with a bias its choice is 1 + bias (sigmoid), which others may pass
                assert int(idx[2, 0]) == 10 or bias is not None
                assert torch.isnan(w[3]).all() and torch.isnan(w[1]).any() and len([i for i in idx[4].tolist() if i >= 0]) == 4
                if scores == "sigmoid":
                    assert int(idx[1, 0]) == 40 and torch.isfinite(w[2]).all()


def test_strides_and_no_tokens(pkg, gpu):
    wide = _logits(40, 200, 17)
    for view in (wide[:, 3:67], wide[::2, 64:128], _logits(64, 40, 18).t(), wide[:1, :64].expand(5, 64), wide[7:8, 1:65]):
        dense = view.contiguous()
        a, b = pkg.moe_gate(view, 8), pkg.moe_gate(dense, 8)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        x, y = view.detach().requires_grad_(), dense.detach().requires_grad_()
        ga, = torch.autograd.grad(pkg.moe_gate(x, 8)[1][:, 0].sum(), x)
        gb, = torch.autograd.grad(pkg.moe_gate(y, 8)[1][:, 0].sum(), y)
        assert torch.equal(ga, gb)
    none = torch.empty((0, 64), device="cuda", requires_grad=True)
    idx, w = pkg.moe_gate(none, 8)
    g, = torch.autograd.grad(w, none, torch.empty_like(w))
    assert idx.shape == w.shape == (0, 8) and g.shape == (0, 64)
    bias = _bias(128, 3)[::2]
    assert torch.equal(pkg.moe_gate(wide[:, :64], 8, bias=bias)[0], pkg.moe_gate(wide[:, :64], 8, bias=bias.contiguous())[0])


def test_same_choice_as_the_router(pkg, gpu):
    """route's experts and weights, from the logits that its product gives (f32 sums in another order: no near ties here)."""
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    x = torch.randn((16, 512), device="cuda", generator=g).bfloat16()
    rw = torch.randn((512, 64), device="cuda", generator=g) * 0.05
    bias = _bias(64, 5)
    idx, w = pkg.route(x, rw, bias, 8, True, 2.5)
    logits = (x.double() @ rw.double()).float()
    i2, w2 = pkg.moe_gate(logits, 8, bias=bias, scaling=2.5)
    assert torch.equal(idx, i2) and torch.allclose(w, w2, rtol=1e-5, atol=0)


def test_refusals(pkg, gpu):
    l = _logits(4, 64, 1)
    for bad, err in ((lambda: pkg.moe_gate(l.half(), 8), TypeError), (lambda: pkg.moe_gate(l[0], 8), ValueError),
                     (lambda: pkg.moe_gate(l, 0), ValueError), (lambda: pkg.moe_gate(l, 33), ValueError),
                     (lambda: pkg.moe_gate(l[:, :4], 5), ValueError), (lambda: pkg.moe_gate(l, 8, scores="relu"), ValueError),
                     (lambda: pkg.moe_gate(l, 8, n_group=3), ValueError), (lambda: pkg.moe_gate(l, 8, n_group=64), ValueError),
                     (lambda: pkg.moe_gate(l, 8, n_group=4, topk_group=5), ValueError),
                     (lambda: pkg.moe_gate(l, 17, n_group=4, topk_group=1), ValueError),
                     (lambda: pkg.moe_gate(l, 8, n_group=4, topk_group=2, group_top=3), ValueError),
                     (lambda: pkg.moe_gate(l, 8, bias=torch.zeros(63, device="cuda")), ValueError),
                     (lambda: pkg.moe_gate(l, 8, bias=torch.zeros(64, device="cuda").bfloat16()), ValueError),
                     (lambda: pkg.moe_gate(l, 8, bias=torch.zeros(64, device="cuda", requires_grad=True)), RuntimeError),
                     (lambda: pkg.moe_gate(l, 8, bias=torch.zeros(64)), ValueError),
                     (lambda: pkg.moe_gate(l, 8, scaling=float("inf")), pkg._lib.MiError),
                     (lambda: pkg.moe_gate(torch.zeros((2, 1025), device="cuda"), 8), ValueError)):
        with pytest.raises(err):
            bad()
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            pkg.moe_gate(forward_ad.make_dual(l, torch.ones_like(l)), 8)
    leaf = l.detach().requires_grad_()
    g, = torch.autograd.grad(pkg.moe_gate(leaf, 8)[1].square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):                               # first order only
        g.sum().backward()
    with torch.no_grad():
        assert not pkg.moe_gate(leaf, 8)[1].requires_grad


def _step(pkg, logits, gw):
    leaf = logits.detach().requires_grad_()
    idx, w = pkg.moe_gate(leaf, 8, scores="softmax", bias=None, n_group=8, topk_group=4)
    return (idx, w.detach()) + torch.autograd.grad(w, leaf, gw)


def test_training_step_captured(pkg, gpu):
    l, gw = _logits(60, 256, 1), _logits(60, 8, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(pkg, l, gw)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = _step(pkg, l, gw)
    for k in range(3):
        a, b = _logits(60, 256, 10 + k), _logits(60, 8, 20 + k)
        l.copy_(a), gw.copy_(b)
        want = _step(pkg, a, b)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outs, want))


def test_threads(pkg, gpu):
    work = [(_logits(T, 256, T), _logits(T, 8, T)) for T in (1, 500, 30)]
    want = [_step(pkg, *a) for a in work]
    torch.cuda.synchronize()
    wrong, gate = [], threading.Barrier(2)

    def body(first):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                gate.wait(30)
                for n in range(9):
                    at = (n + first) % 3
                    got = _step(pkg, *work[at])
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[at])):
                        wrong.append((first, n))
        except Exception as e:                                     # noqa: BLE001 (a thread's error would be lost)
            wrong.append(e)

    threads = [threading.Thread(target=body, args=(j,)) for j in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not wrong, wrong
