"""CPU: the fp8 oracle against torch's own e4m3 conversion and against the definition by hand, and the host side of the
fp8 and sort entry points: every call here is refused, or returns, before anything is launched."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import fp8 as of8

F8 = torch.float8_e4m3fn


def test_values_match_torch():
    bits = np.arange(256, dtype=np.uint8)
    want = torch.from_numpy(bits).view(F8).to(torch.float64).numpy()
    assert np.array_equal(of8.decode(bits), want, equal_nan=True)


def test_rounding_matches_torch():
    rng = np.random.default_rng(1)
    t = np.concatenate([rng.uniform(-448, 448, 4000), rng.standard_normal(4000) * 0.01,
                        np.repeat(of8.VALUES[:126], 3) + np.tile([-2.0 ** -20, 0.0, 2.0 ** -20], 126),
                        (of8.VALUES[:125] + of8.VALUES[1:126]) / 2]).astype(np.float32)   # the ties
    t = t[np.abs(t) <= 448]
    want = torch.from_numpy(t).to(F8).to(torch.float64).numpy()
    assert np.array_equal(of8.round_e4m3(t.astype(np.float64)), want)


def test_scales_by_definition():
    a = np.array([0.0, 448.0, np.nextafter(np.float32(448), np.float32(1e9)), 1.75, 224.0, 1e-38, 3e38, 2.0 ** -93])
    s = of8.scales(a)
    assert s[0] == 2.0 ** -100 and s[5] == 2.0 ** -100 and s[7] == 2.0 ** -100
    assert list(s[1:5]) == [1.0, 2.0, 2.0 ** -8, 0.5]
    for v, sc in zip(a[[1, 2, 3, 4, 6]], s[[1, 2, 3, 4, 6]]):
        assert v <= 448 * sc and v > 224 * sc


def test_quantize_groups_and_nonfinite():
    x = np.zeros((2, 144))
    x[0, 5], x[0, 130], x[1, 3], x[1, 4], x[1, 5] = 448.0, 1.0, np.inf, np.nan, 2.0
    q, s = of8.quantize(x)
    assert s.shape == (2, 2) and s[0, 0] == 1.0 and s[0, 1] == 2.0 ** -8
    assert q[0, 5] == 448.0 and q[0, 130] == 256.0
    assert np.isnan(q[1, 3]) and np.isnan(q[1, 4]) and q[1, 5] * s[1, 0] == 2.0


def test_mlp_bound_covers_f32():
    """The bound holds for a plain f32 evaluation, with room (a check of the oracle, not of a kernel)."""
    rng = np.random.default_rng(3)
    D, I, B = 256, 144, 9
    ws = [of8.weights_dense(*of8.random_weights(rng, R, K)) for R, K in ((I, D), (I, D), (D, I))]
    xd = of8.rows_dense(*of8.quantize(rng.standard_normal((B, D))))
    y, bound = of8.mlp(xd, *ws, 10.0)
    f = [w.astype(np.float32) for w in ws]
    xf = xd.astype(np.float32)
    h = of8.swiglu(xf @ f[0].T, xf @ f[1].T, np.float32(10.0))
    got = of8.rows_dense(*of8.quantize(h)).astype(np.float32) @ f[2].T
    assert np.all(np.abs(got - y) <= bound)
    assert bound.max() < 0.5 * np.abs(y).max()


# ------------------------------------------------------------------------------------------------ the C ABI's refusals
P = ctypes.c_void_p
X, Q, S, Y, WS, BIG = P(0x10000), P(0x20000), P(0x30000), P(0x40000), P(0x50000), 1 << 40


@pytest.fixture(scope="module")
def L(pkg):
    return pkg._lib.lib()


def test_quantize_refusals(L):
    call = lambda x=X, dt=0, n=4, K=256, st=256, q=Q, s=S: L.mi_fp8_quantize(x, dt, n, K, st, q, s, None)
    assert call(x=None) == 1 and call(q=None) == 1 and call(s=None) == 1
    assert call(dt=2) == 8 and call(dt=7) == 8
    assert call(n=0) == 4 and call(n=(1 << 22) + 1) == 4
    assert call(K=250) == 3 and call(K=0) == 3 and call(K=(1 << 16) + 16) == 3
    assert call(st=240) == 8 and call(st=260) == 8                          # shorter than a row; not whole 8 elements
    assert call(x=P(0x10008)) == 8 and call(q=P(0x20004)) == 8 and call(s=P(0x30002)) == 8


def test_project_refusals(L):
    need = L.mi_fp8_project_workspace(40, 256, 100)
    assert need > 0 and L.mi_fp8_project_workspace(32, 256, 100) == 0        # few rows need no workspace
    call = lambda x=X, dt=0, xs=None, B=40, wq=Q, ws=S, K=256, R=100, y=Y, yf=None, w=WS, wb=BIG: L.mi_fp8_project(
        x, dt, xs, B, wq, ws, K, R, y, yf, w, wb, None)
    assert call(x=None) == 1 and call(wq=None) == 1 and call(ws=None) == 1 and call(y=None) == 1
    assert call(dt=2) == 1                                                     # quantised rows without their scales
    assert call(dt=3) == 8
    assert call(B=0) == 4 and call(B=-1) == 4 and call(B=1 << 22, K=4096) == 4
    assert call(K=248) == 3 and call(R=0) == 3 and call(R=(1 << 16) + 1) == 3
    assert call(x=P(0x10004)) == 8 and call(wq=P(0x20008)) == 8 and call(ws=P(0x30001)) == 8 and call(y=P(0x40001)) == 8
    assert call(w=None) == 5 and call(wb=need - 1) == 5 and call(w=P(0x50008)) == 8
    sizes = [L.mi_fp8_project_workspace(b, 6144, 6144) for b in (1, 2, 8, 16, 17, 32, 33, 64, 100, 128, 200, 512, 1000, 4096)]
    assert sizes == sorted(sizes)                                              # a larger batch's serves every smaller
    assert L.mi_fp8_project_workspace(0, 256, 100) == 0 and L.mi_fp8_project_workspace(4, 250, 100) == 0


def test_mlp_refusals(L):
    need = L.mi_fp8_mlp_workspace(5, 256, 144)
    call = lambda x=X, dt=0, B=5, D=256, I=144, g=Q, lim=7.0, y=Y, w=WS, wb=BIG: L.mi_fp8_mlp(
        x, dt, None, B, D, I, g, S, Q, S, Q, S, lim, y, None, w, wb, None)
    assert call(x=None) == 1 and call(g=None) == 1 and call(y=None) == 1
    assert call(B=0) == 4 and call(D=250) == 3 and call(I=100) == 3
    assert call(lim=0.0) == 8 and call(lim=float("nan")) == 8 and call(g=P(0x20008)) == 8
    assert call(wb=need - 1) == 5 and call(w=None) == 5
    sizes = [L.mi_fp8_mlp_workspace(b, 6144, 2048) for b in (1, 2, 8, 16, 17, 32, 33, 64, 100, 128, 200, 512, 1000, 2048)]
    assert sizes == sorted(sizes) and L.mi_fp8_mlp_workspace(4, 256, 100) == 0


def test_grouped_refusals(L):
    need = L.mi_fp8_grouped_workspace(8 * 32, 256, 100)
    call = lambda x=X, n=8, tm=32, be=P(0x60000), nb=P(0x70000), E=4, K=256, R=100, y=Y, wb=BIG: L.mi_fp8_grouped(
        x, 0, None, n, tm, be, nb, P(0x80000), Q, S, E, K, R, y, None, WS, wb, None)
    assert call(tm=48) == 8 and call(tm=0) == 8 and call(tm=256) == 8
    assert call(n=0) == 4 and call(n=1 << 20) == 4
    assert call(E=0) == 3 and call(E=1025) == 3 and call(K=24) == 3
    assert call(be=None) == 1 and call(nb=None) == 1 and call(x=None) == 1 and call(y=None) == 1
    assert call(be=P(0x60002)) == 8 and call(wb=need - 1) == 5
    assert L.mi_fp8_grouped_workspace(0, 256, 100) == 0


def test_moe_refusals(L):
    need = L.mi_fp8_moe_workspace(5, 2, 8, 256, 144)
    call = lambda x=X, dt=0, T=5, k=2, E=8, D=256, I=144, idx=P(0x60000), w=P(0x70000), lim=7.0, o=Y, wb=BIG, g=Q: \
        L.mi_fp8_moe(g, S, Q, S, Q, S, E, D, I, x, dt, T, k, idx, w, lim, o, None, WS, wb, None)
    assert call(x=None) == 1 and call(idx=None) == 1 and call(w=None) == 1 and call(o=None) == 1 and call(g=None) == 1
    assert call(dt=2) == 8 and call(lim=-1.0) == 8
    assert call(T=0) == 4 and call(k=0) == 4 and call(T=1 << 20, k=8) == 4
    assert call(E=0) == 3 and call(E=1025) == 3 and call(D=250) == 3 and call(I=100) == 3
    assert call(x=P(0x10008)) == 8 and call(idx=P(0x60001)) == 8 and call(wb=need - 1) == 5
    for E, k in ((64, 8), (8, 2), (96, 4), (1, 1)):
        sizes = [L.mi_fp8_moe_workspace(t, k, E, 2048, 768) for t in list(range(1, 70)) + [128, 300, 512, 1000, 1999, 4000]]
        assert sizes == sorted(sizes) and sizes[0] > 0


def test_rows_refusals(L):
    disp = lambda x=X, dt=0, T=4, k=2, D=64, sl=P(0x60000), tr=P(0x70000), n=32, y=Y: L.mi_moe_dispatch(
        x, dt, T, k, D, sl, tr, n, y, None)
    comb = lambda x=X, dt=0, T=4, k=2, D=64, sl=P(0x60000), n=32, y=Y: L.mi_moe_combine(
        x, dt, T, k, D, sl, P(0x80000), n, y, None)
    grad = lambda x=X, dt=0, T=4, k=2, D=64, sl=P(0x60000), n=32, y=Y: L.mi_moe_combine_grad(
        x, P(0x90000), dt, T, k, D, sl, P(0x70000), P(0x80000), n, y, P(0xa0000), None)
    for f in (disp, comb, grad):
        assert f(x=None) == 1 and f(sl=None) == 1 and f(y=None) == 1
        assert f(dt=2) == 8 and f(x=P(0x10008)) == 8 and f(y=P(0x40004)) == 8 and f(sl=P(0x60002)) == 8
        assert f(T=0) == 4 and f(k=0) == 4 and f(T=1 << 21, k=4) == 4 and f(n=0) == 4
        assert f(D=0) == 3 and f(D=60) == 3 and f(D=(1 << 17) + 8) == 3
    assert disp(tr=None) == 1


# ------------------------------------------------------------------------------------------------ the Python side's refusals
def _leaf(pkg, R, K, E=None):
    lead = () if E is None else (E,)
    return pkg.Fp8Leaf(torch.zeros(lead + (R, K)).to(F8), torch.zeros(lead + (-(-R // 128), -(-K // 128))))


def test_python_refusals(pkg):
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    leaf = _leaf(pkg, 100, 256)
    with pytest.raises(TypeError, match="bf16 or f32"):
        pkg.fp8_quantize(torch.zeros(2, 32, dtype=torch.float16))
    with pytest.raises(ValueError, match="columns"):
        pkg.fp8_project(bf(2, 128), leaf)
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        pkg.fp8_project(bf(2, 256), pkg.Fp8Leaf(torch.zeros(100, 256, dtype=torch.int8), leaf.s))
    with pytest.raises(ValueError, match="do not fit"):
        pkg.fp8_project(bf(2, 256), pkg.Fp8Leaf(leaf.q, torch.zeros(1, 1)))
    with pytest.raises(ValueError, match="contiguous"):
        pkg.fp8_project(bf(2, 256), pkg.Fp8Leaf(_leaf(pkg, 256, 256).q.t(), torch.zeros(2, 2)))
    with pytest.raises(ValueError, match="one matrix"):
        pkg.fp8_project(bf(2, 256), _leaf(pkg, 100, 256, 3))
    with pytest.raises(TypeError):
        pkg.fp8_project((torch.zeros(2, 256), torch.zeros(2, 2)), leaf)
    with pytest.raises(ValueError, match="quantised activations"):
        pkg.fp8_project((torch.zeros(2, 256).to(F8), torch.zeros(2, 3)), leaf)
    with pytest.raises(RuntimeError, match="no gradient"):
        pkg.fp8_project(torch.zeros(2, 256, requires_grad=True), leaf)
    with pytest.raises(ValueError, match="an output must be"):
        pkg.fp8_project(bf(2, 256), leaf, y_bf16=bf(2, 99))
    with pytest.raises(ValueError, match="gate and up"):
        pkg.fp8_mlp(bf(2, 256), leaf, leaf, leaf, 7.0)
    with pytest.raises(ValueError, match="all fp8"):
        pkg.mlp_partial({"gate": leaf, "up": leaf, "down": bf(256, 100)}, bf(2, 256), 7.0)
    plan = {"blk_expert": torch.zeros(4, dtype=torch.int32), "n_blocks": torch.ones(1, dtype=torch.int32),
            "tok_row": torch.zeros(64, dtype=torch.int32), "row_slot": torch.zeros((5, 2), dtype=torch.int32)}
    with pytest.raises(ValueError, match="do not fit the plan"):
        pkg.fp8_grouped(bf(60, 256), plan, _leaf(pkg, 100, 256, 3))
    with pytest.raises(ValueError, match=r"\[E, R, K\]"):
        pkg.fp8_grouped(bf(64, 256), plan, leaf)
    g, d = _leaf(pkg, 144, 256, 3), _leaf(pkg, 256, 144, 3)
    with pytest.raises(ValueError, match="idx and w"):
        pkg.fp8_moe(g, g, d, bf(4, 256), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2), 7.0)
    with pytest.raises(TypeError):
        pkg.fp8_moe(g, g, d, (torch.zeros(2, 256).to(F8), torch.zeros(2, 2)), torch.zeros(2, 2, dtype=torch.int32),
                    torch.zeros(2, 2), 7.0)
    with pytest.raises(RuntimeError, match="no gradient"):
        pkg.fp8_moe(g, g, d, bf(2, 256), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 2, requires_grad=True), 7.0)
    with pytest.raises(TypeError, match="bf16 or f32"):
        pkg.moe_dispatch(torch.zeros(5, 64, dtype=torch.float16), plan)
    with pytest.raises(ValueError, match="of 5 tokens"):
        pkg.moe_dispatch(torch.zeros(4, 64), plan)
    with pytest.raises(ValueError, match="64 rows"):
        pkg.moe_combine(torch.zeros(63, 64), plan, torch.zeros(5, 2))
    with pytest.raises(ValueError, match="w must be"):
        pkg.moe_combine(torch.zeros(64, 64), plan, torch.zeros(5, 3))


# ------------------------------------------------------------------------------------------------ a call's own scratch
class _Lib:
    """Stands for the library: notes the scratch of every call, and has a second call arrive within the first."""

    def __init__(self, name, arg):
        self.name, self.arg, self.seen, self.again = name, arg, [], None

    def __getattr__(self, attr):
        if attr == self.name:
            return self._call
        if attr == self.name + "_workspace":
            return lambda *a: 1 << 16
        raise AttributeError(attr)

    def _call(self, *args):
        self.seen.append(args[self.arg])
        if self.again is not None:
            again, self.again = self.again, None
            again()
        return 0


@pytest.mark.parametrize("name,arg", [("mi_fp8_project", 10), ("mi_fp8_mlp", 15), ("mi_fp8_moe", 18),
                                      ("mi_fp8_grouped", 15)])
def test_a_call_within_a_call_has_other_scratch(pkg, monkeypatch, name, arg):
    """The scratch that a call's launches hand each other is held until they are queued: a call from another host thread
    in between must not be given the same memory."""
    fake = _Lib(name, arg)
    monkeypatch.setattr(pkg.fp8, "lib", lambda: fake)
    monkeypatch.setattr(pkg.fp8, "_stream_of", lambda *a: 0)
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    g, d = _leaf(pkg, 144, 256, 3), _leaf(pkg, 256, 144, 3)
    one = [pkg.Fp8Leaf(l.q[0], l.s[0]) for l in (g, g, d)]
    plan = {"blk_expert": torch.zeros(4, dtype=torch.int32), "n_blocks": torch.ones(1, dtype=torch.int32),
            "tok_row": torch.zeros(64, dtype=torch.int32), "row_slot": torch.zeros((5, 2), dtype=torch.int32)}
    call = {"mi_fp8_project": lambda: pkg.fp8_project(bf(40, 256), one[0]),
            "mi_fp8_mlp": lambda: pkg.fp8_mlp(bf(40, 256), *one, 7.0),
            "mi_fp8_moe": lambda: pkg.fp8_moe(g, g, d, bf(4, 256), torch.zeros((4, 2), dtype=torch.int32),
                                              torch.zeros(4, 2), 7.0),
            "mi_fp8_grouped": lambda: pkg.fp8_grouped(bf(64, 256), plan, g)}[name]
    fake.again = call
    call()
    assert len(fake.seen) == 2 and fake.seen[0] != fake.seen[1]


def test_scales_that_require_a_gradient_are_refused(pkg):
    leaf = _leaf(pkg, 100, 256)
    with_grad = pkg.Fp8Leaf(leaf.q, leaf.s.clone().requires_grad_())
    x = torch.zeros((2, 256), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no gradient"):
        pkg.fp8_project(x, with_grad)
    with pytest.raises(RuntimeError, match="no gradient"):
        pkg.fp8_project((x.to(F8), torch.ones((2, 2), requires_grad=True)), leaf)
    with torch.no_grad():
        assert pkg.fp8._leaf_dims(with_grad, "fp8_project") == (0, 100, 256)
    assert not pkg.fp8_leaf({"q": leaf.q, "s": torch.nn.Parameter(leaf.s)}, device="cpu").s.requires_grad


@pytest.mark.parametrize("name,arg", [("mi_fp8_project", 10), ("mi_fp8_mlp", 15), ("mi_fp8_moe", 18),
                                      ("mi_fp8_grouped", 15)])
def test_a_workspace_is_as_long_as_its_memory(pkg, monkeypatch, name, arg):
    """The bytes that a call is told of lie behind the address that it is given: an expanded or strided view has more
    elements, or a wider span, than memory of its own."""
    fake = _Lib(name, arg + 1)
    monkeypatch.setattr(pkg.fp8, "lib", lambda: fake)
    monkeypatch.setattr(pkg.fp8, "_stream_of", lambda *a: 0)
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    g, d = _leaf(pkg, 144, 256, 3), _leaf(pkg, 256, 144, 3)
    one = [pkg.Fp8Leaf(l.q[0], l.s[0]) for l in (g, g, d)]
    plan = {"blk_expert": torch.zeros(4, dtype=torch.int32), "n_blocks": torch.ones(1, dtype=torch.int32),
            "tok_row": torch.zeros(64, dtype=torch.int32), "row_slot": torch.zeros((5, 2), dtype=torch.int32)}
    call = {"mi_fp8_project": lambda ws: pkg.fp8_project(bf(40, 256), one[0], workspace=ws),
            "mi_fp8_mlp": lambda ws: pkg.fp8_mlp(bf(40, 256), *one, 7.0, workspace=ws),
            "mi_fp8_moe": lambda ws: pkg.fp8_moe(g, g, d, bf(4, 256), torch.zeros((4, 2), dtype=torch.int32),
                                                 torch.zeros(4, 2), 7.0, workspace=ws),
            "mi_fp8_grouped": lambda ws: pkg.fp8_grouped(bf(64, 256), plan, g, workspace=ws)}[name]
    buf = torch.zeros(1 << 16, dtype=torch.uint8)
    for ws, size in ((buf, 1 << 16), (buf.view(256, 256), 1 << 16), (buf.view(torch.int32), 1 << 16), (buf[256:], 65280)):
        call(ws)
        assert fake.seen.pop() == size
    for ws in (buf[:1].expand(1 << 16), buf[:256].expand(256, 256), buf[::2], buf.view(256, 256).t(), buf.view(256, 256)[:, :128]):
        with pytest.raises(ValueError, match="workspace"):
            call(ws)
    assert not fake.seen
