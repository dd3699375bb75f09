"""The operators around a layer's experts and projections, as measurable cases, each in a plain form of elementary torch
operations and as the calls that a program makes of the framework.

  norm      rms_norm: the residual's addition and the root-mean-square norm of the sum; train: with the gradients
  fp8norm   fp8_rms_norm: the same, straight to the e4m3 values and scales that the fp8 products take
  gate      moe_gate: a router's logits to expert ids and weights, by sigmoid or softmax scores, with a balancing bias, groups
            of experts and renormalised weights; train: with the gradient of the logits
  linear    bf16_linear: a product over bf16 weights with bias, activation and residual; train: with every gradient

Sizes are those of the benchmarked layer (hidden 6144, 64 experts, top-8, intermediate 2048) and of the router tests (256
experts) in the listed cases, with smaller layers and odd sizes among the drawn ones.  Hidden states are N(0, 1) with a few
large channels, weights N(0, 0.02), norm weights near 1, logits N(0, 1.5).
"""
import math

import torch

own = False

EPS = 1e-5                      # of the norms
STD = 0.02                      # spread of the weights
TINY = 1e-20                    # of the gate's renormalisation
DEV = "cuda"
F8 = torch.float8_e4m3fn
_pkg = []


def pkg():
    if not _pkg:
        import __graft_entry__
        _pkg.append(__graft_entry__.load_package())
    return _pkg[0]


def norm(kind, tokens, D=6144, dtype="bf16", residual=True, train=False):
    return dict(kind=kind, tokens=tokens, D=D, dtype=dtype, residual=residual, train=train)


def gate(tokens, E, k, scores, bias, n_group=1, topk_group=1, masked=0, dtype="f32", train=False):
    return dict(kind="gate", tokens=tokens, E=E, k=k, scores=scores, bias=bias, n_group=n_group, topk_group=topk_group,
                masked=masked, dtype=dtype, train=train)


def linear(tokens, D=6144, n_out=6144, bias=False, act="", residual=False, train=False):
    return dict(kind="linear", tokens=tokens, D=D, n_out=n_out, bias=bias, act=act, residual=residual, train=train)


def listed():
    return [
        # the norm before a block in one stream's decode step: the smallest call, all launch and latency
        dict(norm("norm", 1), name="norm_t1"),
        # a training step's tokens: forward and the gradients of the stream and the weight
        dict(norm("norm", 4096, train=True), name="norm_train_t4096"),
        # the norm in front of fp8 projections for a decode batch
        dict(norm("fp8norm", 37), name="fp8norm_t37"),
        # and for a long prompt in one piece
        dict(norm("fp8norm", 4099), name="fp8norm_t4099"),
        # the routing of one decode step of a few streams
        dict(gate(3, 64, 8, "sigmoid", True), name="gate_t3"),
        # of a long prompt over many experts in groups
        dict(gate(16384, 256, 8, "sigmoid", True, 8, 4, dtype="bf16"), name="gate_groups_t16384"),
        # of a training step, with the gradient of the logits
        dict(gate(8191, 64, 8, "softmax", False, train=True), name="gate_train_t8191"),
        # the output projection of one decode step, added to the stream: streams the weights
        dict(linear(1, residual=True), name="linear_t1"),
        # a biased, activated projection of a decode batch with an odd number of outputs
        dict(linear(37, n_out=2051, bias=True, act="silu"), name="linear_t37"),
        # the output projection of a prompt piece of whatever length the prompt left
        dict(linear(517, residual=True), name="linear_t517"),
        # of a long prompt: bound by the matrix cores
        dict(linear(4096, residual=True), name="linear_t4096"),
        # one training step through a biased, activated layer with its residual
        dict(linear(2048, bias=True, act="gelu", residual=True, train=True), name="linear_train_t2048"),
    ]


def _log(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "fp8norm", "gate", "gate", "gate", "linear", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    train = rng.random() < 0.4
    if kind in ("norm", "fp8norm"):
        D = rng.choice([6144, 4096, 2048, 16 * rng.randint(4, 512)])
        return norm(kind, _log(rng, 1, 4099), D, dtype, rng.random() < 0.7, train and kind == "norm")
    if kind == "gate":
        E, k, n_group, topk_group = rng.choice([(64, 8, 1, 1), (256, 8, 8, 4), (256, 6, 1, 1), (96, 4, 4, 2), (160, 6, 8, 3),
                                                (40, 5, 1, 1), (rng.randint(9, 512), rng.randint(1, 9), 1, 1)])
        return gate(_log(rng, 1, 16384), E, k, rng.choice(["sigmoid", "softmax"]), rng.random() < 0.6, n_group, topk_group,
                    rng.choice([0, 0, E // 16]), dtype, train)
    D = rng.choice([6144, 4096, 2048, 8 * rng.randint(8, 768)])
    n_out = rng.choice([6144, 2048, rng.randint(64, 6144), rng.randint(64, 6144)])
    return linear(_log(rng, 1, 2048 if train else 4096), D, n_out, rng.random() < 0.5, rng.choice(["", "silu", "gelu", "gelu_tanh", "relu"]),
                  rng.random() < 0.5, train)


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(0x30A70000 + int(seed))
    return g


def _type(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _randn(g, *shape):
    return torch.randn(shape, device=DEV, generator=g)


def _acts(g, n, K):
    """[n, K] hidden states: N(0, 1), one channel in 256 ten times as large."""
    x = _randn(g, n, K)
    x[:, torch.randperm(K, device=DEV, generator=g)[:K // 256]] *= 10.0
    return x


def prepare(case, seed):
    g = _gen(seed)
    st = {"case": case}
    T = case["tokens"]
    if case["kind"] in ("norm", "fp8norm"):
        D, t = case["D"], _type(case["dtype"])
        st.update(x=_acts(g, T, D).to(t), res=_acts(g, T, D).to(t) if case["residual"] else None,
                  w=(1.0 + 0.1 * _randn(g, D)).to(t))
        if case["train"]:
            st.update(gy=_randn(g, T, D).to(t), gs=_randn(g, T, D).to(t) if case["residual"] else None)
    elif case["kind"] == "gate":
        E, k = case["E"], case["k"]
        logits = 1.5 * _randn(g, T, E)
        if case["masked"]:                      # experts that are out of service
            logits[:, torch.randperm(E, device=DEV, generator=g)[:case["masked"]]] = -math.inf
        st.update(logits=logits.to(_type(case["dtype"])), bias=0.05 * _randn(g, E) if case["bias"] else None)
        if case["train"]:
            st.update(gw=_randn(g, T, k))
    else:
        D, N, t = case["D"], case["n_out"], torch.bfloat16
        st.update(x=_acts(g, T, D).to(t), w=(STD * _randn(g, N, D)).to(t),
                  b=(0.1 * _randn(g, N)).to(t) if case["bias"] else None,
                  res=_acts(g, T, N).to(t) if case["residual"] else None)
        if case["train"]:
            st.update(gy=_randn(g, T, N).to(t))
    if case["train"]:
        for name in ("x", "res", "w", "b", "logits"):
            if st.get(name) is not None:
                st[name].requires_grad_(True)
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_norm(st, to8):
    case, x, w = st["case"], st["x"].detach(), st["w"].detach().float()
    t = x.dtype
    s = x if st["res"] is None else (x.float() + st["res"].detach().float()).to(t)
    v = s.float()
    r = (1.0 / torch.sqrt(v.double().square().mean(-1, keepdim=True) + EPS)).float()
    y = (v * r) * w
    out = {} if st["res"] is None else {"stream": s}
    if to8:
        out["q"], out["s"] = _quantize(y)
        return out
    out["y"] = y.to(t)
    if case["train"]:
        gy = st["gy"].float()
        gw = gy * w
        ds = r * gw - v * (r ** 3 * (gw * v).mean(-1, keepdim=True))
        if st["res"] is not None:
            ds = ds + st["gs"].float()
            out["dres"] = ds.to(t)
        out["dx"] = ds.to(t)
        out["dw"] = (gy * (v * r)).double().sum(0).to(t)
    return out


def _blocks(n):
    return (n + 127) // 128


def _quantize(y):
    """e4m3 values and power-of-two scales of the rows of y: least s = 2^e, e >= -100, with max |y| <= 448 s."""
    n, K = y.shape
    v = torch.nn.functional.pad(y, (0, _blocks(K) * 128 - K)).view(n, -1, 128)
    m, e = torch.frexp(v.abs().amax(-1) / 448.0)         # amax / 448 = m 2^e, m in [0.5, 1)
    s = torch.ldexp(torch.ones_like(m), torch.where(m == 0.0, -100, e - (m == 0.5).int()).clamp_min(-100))
    return (v / s[..., None]).view(n, -1)[:, :K].to(F8), s


def _scores(l, kind):
    if kind == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-l))
    p = torch.exp(l - l.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _plain_gate(st):
    """Scores and choices in 64 bits, since the choice of a border case turns on the last one."""
    case, k = st["case"], st["case"]["k"]
    T, E, G = case["tokens"], case["E"], case["n_group"]
    l = st["logits"].detach().double()
    s = _scores(l, case["scores"])
    c = s if st["bias"] is None else s + st["bias"].double()
    c = torch.where(l == -math.inf, -math.inf, c)
    if G > 1:                                            # a group counts by its two largest choices
        best = torch.sort(c.view(T, G, -1), dim=-1, descending=True)[0][..., :2]
        score = best[..., 0] + torch.where(best[..., 1] == -math.inf, 0.0, best[..., 1])
        kept = torch.sort(score, dim=-1, descending=True, stable=True)[1][:, :case["topk_group"]]
        live = torch.zeros((T, G), dtype=torch.bool, device=DEV).scatter_(1, kept, True)
        c = torch.where(live[..., None], c.view(T, G, -1), -math.inf).view(T, E)
    top, idx = torch.sort(c, dim=-1, descending=True, stable=True)
    top, idx = top[:, :k], idx[:, :k]
    has = top > -math.inf                                # (a slot that no expert is left for)
    sel = torch.where(has, s.gather(1, idx), 0.0)
    total = sel.sum(-1, keepdim=True) + TINY
    out = {"idx": torch.where(has, idx, -1).to(torch.int32), "w": (sel / total).float()}
    if case["train"]:
        gw = st["gw"].double()
        gs = (gw - (gw * sel).sum(-1, keepdim=True) / total) / total
        gs = torch.zeros_like(s).scatter_add_(1, idx, torch.where(has, gs, 0.0))
        gl = gs * s * (1.0 - s) if case["scores"] == "sigmoid" else s * (gs - (gs * s).sum(-1, keepdim=True))
        out["dlogits"] = gl.to(st["logits"].dtype)
    return out


def _act(z, name):
    """The activation and its derivative at z."""
    if name == "relu":
        return z.clamp_min(0.0), (z > 0.0).to(z.dtype)
    if name == "silu":
        p = 1.0 / (1.0 + torch.exp(-z))
        return z * p, p * (1.0 + z * (1.0 - p))
    if name == "gelu":
        p = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * p, p + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if name == "gelu_tanh":
        a = math.sqrt(2.0 / math.pi)
        t = torch.tanh(a * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * a * (1.0 + 3.0 * 0.044715 * z * z)
    return z, torch.ones_like(z)


def _plain_linear(st):
    case, bf = st["case"], torch.bfloat16
    x, w = st["x"].detach().float(), st["w"].detach().float()
    z = x @ w.t()
    if st["b"] is not None:
        z = z + st["b"].detach().float()
    a, d = _act(z, case["act"])
    if st["res"] is not None:
        a = a + st["res"].detach().float()
    out = {"y": a.to(bf)}
    if case["train"]:
        dz = st["gy"].float() * d
        out.update(dx=(dz @ w).to(bf), dw=(dz.t() @ x).to(bf))
        if st["b"] is not None:
            out["db"] = dz.sum(0).to(bf)
        if st["res"] is not None:
            out["dres"] = st["gy"].clone()
    return out


def _plain(st):
    kind = st["case"]["kind"]
    if kind in ("norm", "fp8norm"):
        return _plain_norm(st, kind == "fp8norm")
    return _plain_gate(st) if kind == "gate" else _plain_linear(st)


# ------------------------------------------------------------------------------------------------ the framework's calls
def _grads(out, outputs, gouts, inputs):
    """The gradients of those inputs ({name: leaf}) that there are, beside the outputs."""
    inputs = {n: t for n, t in inputs.items() if t is not None}
    got = torch.autograd.grad(outputs, list(inputs.values()), gouts)
    return {**{n: t.detach() for n, t in out.items()}, **dict(zip(inputs, got))}


def _own(st):
    p, case = pkg(), st["case"]
    kind, train = case["kind"], case["train"]
    if kind == "fp8norm":
        (q, s), stream, _ = p.fp8_rms_norm(st["x"], st["w"], EPS, residual=st["res"])
        return {"q": q, "s": s} if stream is None else {"q": q, "s": s, "stream": stream}
    if kind == "norm":
        got = p.rms_norm(st["x"], st["w"], EPS, residual=st["res"])
        out = {"y": got} if st["res"] is None else {"y": got[0], "stream": got[1]}
        if not train:
            return out
        gouts = [st["gy"]] if st["res"] is None else [st["gy"], st["gs"]]
        return _grads(out, list(out.values()), gouts, {"dx": st["x"], "dres": st["res"], "dw": st["w"]})
    if kind == "gate":
        idx, w = p.moe_gate(st["logits"], case["k"], scores=case["scores"], bias=st["bias"], n_group=case["n_group"],
                            topk_group=case["topk_group"])
        out = {"idx": idx, "w": w}
        return _grads(out, [w], [st["gw"]], {"dlogits": st["logits"]}) if train else out
    y = p.bf16_linear(st["x"], p.Bf16Leaf(st["w"]), bias=st["b"], act=case["act"] or None, residual=st["res"])
    if not train:
        return {"y": y}
    return _grads({"y": y}, [y], [st["gy"]], {"dx": st["x"], "dw": st["w"], "db": st["b"], "dres": st["res"]})


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------ work, exact values
def work(case):
    T, train = case["tokens"], case["train"]
    el = 4 if case.get("dtype") == "f32" else 2
    if case["kind"] in ("norm", "fp8norm"):
        D, res = case["D"], int(case["residual"])
        out = T * D * el if case["kind"] == "norm" else T * D + 4 * T * _blocks(D)
        fwd = T * D * el * (1 + 2 * res) + D * el + out
        # backward: dy and the stream (and its gradient) in, one gradient and the weight's out
        return {"bytes": fwd + train * (T * D * el * (3 + res) + 2 * D * el), "flops": T * D * (5 + 10 * train)}
    if case["kind"] == "gate":
        E, k = case["E"], case["k"]
        fwd = T * E * el + 8 * T * k + 4 * E * case["bias"]
        return {"bytes": fwd + train * (2 * T * E * el + 12 * T * k), "flops": T * E * (8 + 6 * train)}
    D, N = case["D"], case["n_out"]
    fwd = 2 * (T * D + N * D + T * N * (1 + case["residual"]) + N * case["bias"])
    bwd = 2 * (2 * (T * D + N * D) + T * N + N * case["bias"])      # x, w, dy in; dx, dw, db out (dresidual is dy)
    return {"bytes": fwd + train * bwd, "flops": 2 * T * D * N * (3 if train else 1)}


def _norm64(case, st):
    x, w = st["x"].detach().double(), st["w"].detach().double()
    out = {}
    if case["residual"]:
        # the stream is held in its type: the norm is that of the rounded sum
        stream = (x + st["res"].detach().double()).to(_type(case["dtype"]))
        out["stream"] = x + st["res"].detach().double()
        x = stream.double()
    D = case["D"]
    inv = torch.rsqrt((x * x).sum(1) / D + EPS)
    xhat = x * inv[:, None]
    y = xhat * w
    if case["kind"] == "fp8norm":
        n, blocks = y.shape[0], _blocks(D)
        v = torch.zeros((n, blocks * 128), dtype=torch.float64, device=DEV)
        v[:, :D] = y
        v = v.view(n, blocks, 128)
        a = v.abs().max(2).values
        e = torch.ceil(torch.log2(a.clamp_min(1e-300) / 448.0))
        e = torch.where(a > 448.0 * torch.exp2(e), e + 1, e)              # log2 next to a whole number
        e = torch.where(a <= 448.0 * torch.exp2(e - 1), e - 1, e)
        s = torch.exp2(e.clamp_min(-100.0))
        q = v / s[..., None]
        unit = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3.0)   # step of e4m3 at q
        out["q"], out["s"] = (torch.round(q / unit) * unit).view(n, -1)[:, :D], s
        return out
    out["y"] = y
    if case["train"]:
        gy = st["gy"].double()
        g = gy * w
        dx = (g - xhat * (g * xhat).sum(1, keepdim=True) / D) * inv[:, None]
        if case["residual"]:
            dx = dx + st["gs"].double()
            out["dres"] = dx
        out["dx"], out["dw"] = dx, torch.einsum("td,td->d", gy, xhat)
    return out


def _gate64(case, st):
    """Weights and gradients of the chosen experts; the ids are whole numbers and have no such value."""
    idx = _plain_gate({**st, "case": dict(case, train=False)})["idx"].long()
    l = st["logits"].detach().double()
    p = torch.sigmoid(l) if case["scores"] == "sigmoid" else torch.softmax(l, 1)
    chosen = torch.zeros_like(l)
    chosen[torch.arange(l.shape[0], device=DEV)[:, None].expand_as(idx)[idx >= 0], idx[idx >= 0]] = 1.0
    total = (p * chosen).sum(1, keepdim=True)
    weight = p * chosen / total
    at = idx.clamp_min(0)
    out = {"idx": None, "w": torch.where(idx >= 0, torch.take_along_dim(weight, at, 1), 0.0)}
    if case["train"]:
        gw = torch.zeros_like(l).scatter_add_(1, at, torch.where(idx >= 0, st["gw"].double(), 0.0))
        # d weight_i / d l_j = weight_i (f_i [i = j] - weight_j f_j), f = 1 - p (sigmoid) or 1 (softmax)
        f = 1.0 - p if case["scores"] == "sigmoid" else torch.ones_like(p)
        out["dlogits"] = weight * f * (gw - (gw * weight).sum(1, keepdim=True))
    return out


def _linear64(case, st):
    x, w = st["x"].detach().double(), st["w"].detach().double()
    z = torch.mm(x, w.transpose(0, 1))
    if case["bias"]:
        z += st["b"].detach().double()
    name = case["act"]
    a, d = z, torch.ones_like(z)
    if name == "relu":
        a, d = torch.relu(z), (z > 0).double()
    elif name == "silu":
        sig = torch.sigmoid(z)
        a, d = z * sig, sig + z * sig * torch.sigmoid(-z)
    elif name == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        a, d = z * cdf, cdf + z * torch.exp(-z * z / 2.0) / math.sqrt(2.0 * math.pi)
    elif name == "gelu_tanh":
        u = 2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3)
        sig = torch.sigmoid(u)                           # (1 + tanh(u / 2)) / 2
        a, d = z * sig, sig + z * sig * (1.0 - sig) * 2.0 * math.sqrt(2.0 / math.pi) * (1.0 + 0.134145 * z * z)
    out = {"y": a + st["res"].detach().double() if case["residual"] else a}
    if case["train"]:
        gz = st["gy"].double() * d
        out["dx"], out["dw"] = torch.mm(gz, w), torch.mm(gz.transpose(0, 1), x)
        if case["bias"]:
            out["db"] = gz.sum(0)
        if case["residual"]:
            out["dres"] = st["gy"].double()
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return {"norm": _norm64, "fp8norm": _norm64, "gate": _gate64, "linear": _linear64}[case["kind"]](case, st)
