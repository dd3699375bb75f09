"""GPU: moe_gate's weights and gradients in rows of which some experts are out of service or at the type's lowest value, each row
within a bound of its own logits."""
import math

import pytest
import torch

from tests.test_gpu_gate import _bias, _grad_want, _logits, _want

pytestmark = pytest.mark.gpu


def _partly_masked(E, dtype):
    lowest = torch.finfo(dtype).min
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    logits = _logits(64, E, 11)
    share = torch.rand((64, 1), device="cuda", generator=g)
    logits[torch.rand((64, E), device="cuda", generator=g) < share] = -math.inf
    logits[0] = -math.inf                                           # no expert
    logits[1] = -math.inf
    logits[1, E - 1] = 2.0                                          # one
    logits[2] = lowest                                              # equal ones, at the lowest value
    logits[3] = _logits(1, E, 12)
    logits[3, : E // 2] = lowest                                    # half of them there
    logits[4, 1:] = lowest                                          # all but one
    logits[4, 0] = -1.0
    return logits.to(dtype)


def _far(logits, scores):
    """What the rounding of l - m adds to e^(l - m), per row: |l - m| of the experts whose e^(l - m) is not 0 in f32.  (The
    sigmoid's exponential takes the logit as it is.)"""
    if scores == "sigmoid":
        return torch.zeros((logits.shape[0], 1), dtype=torch.float64, device=logits.device)
    l = logits.double()
    m = l.amax(-1, keepdim=True)
    d = torch.where(m == -math.inf, 0.0, m - l)
    return torch.where(d < 104.0, d, 0.0).amax(-1, keepdim=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
@pytest.mark.parametrize("E,k,G,tg", [(64, 8, 1, 1), (256, 8, 8, 4), (100, 7, 1, 1), (1024, 32, 4, 2)])
def test_partly_masked_rows(pkg, gpu, dtype, scores, E, k, G, tg):
    logits = _partly_masked(E, dtype)
    far = _far(logits, scores)
    gw = _logits(64, k, 7)
    for bias in (None, _bias(E, 1) + 0.5):
        for norm in (True, False):
            kw = dict(scores=scores, bias=bias, n_group=G, topk_group=tg, norm_topk=norm)
            leaf = logits.detach().requires_grad_()
            idx, w = pkg.moe_gate(leaf, k, **kw)
            widx, ww, s, has = _want(logits, k, **kw)
            assert torch.equal(idx, widx)
            # exp 2, the sum over the experts (16 of a lane, 6 levels), its reciprocal 2, a product, the slots' sum 6 and three more
            steps = 48 + 2 * far
            assert float(steps.max()) < 100                         # (a part that is missing is far outside)
            assert bool(((w.double() - ww).abs() <= 2.0 ** -24 * steps * ww.abs() + 1e-37).all())
            got, = torch.autograd.grad(w, leaf, gw)
            want, mag = _grad_want(logits, gw, idx, s, has, scores, norm, 1.0)
            half = 2.0 ** -8 if dtype is torch.bfloat16 else 0.0
            assert bool(((got.double() - want).abs() <= (2.0 ** -24 * (128 + 4 * far) + half) * mag + 1e-37).all())


@pytest.mark.parametrize("E,k", [(64, 8), (100, 7)])
def test_closed_forms(pkg, gpu, E, k):
    """Equal logits share the weight equally; a single finite one takes it all (softmax), or what its score is (sigmoid)."""
    logits = _partly_masked(E, torch.float32)
    for norm, row2 in ((True, 1.0 / k), (False, 1.0 / E)):
        idx, w = pkg.moe_gate(logits, k, scores="softmax", norm_topk=norm)
        assert idx[2].tolist() == list(range(k)) and bool(((w[2].double() - row2).abs() <= 2.0 ** -24 * 48 * row2).all())
        assert int(idx[1, 0]) == E - 1 and float(w[1, 0]) == 1.0 and int(idx[4, 0]) == 0 and float(w[4, 0]) == 1.0
        assert (w[4, 1:] == 0).all() and idx[4, 1:].tolist() == list(range(1, k))
        idx, w = pkg.moe_gate(logits, k, scores="sigmoid", norm_topk=norm)
        assert idx[2].tolist() == list(range(k)) and (w[2] == 0).all()
        for row, at, l in ((1, E - 1, 2.0), (4, 0, -1.0)):
            want = 1.0 if norm else 1.0 / (1.0 + math.exp(-l))
            assert int(idx[row, 0]) == at and abs(float(w[row, 0]) - want) <= 2.0 ** -24 * 8 * want and (w[row, 1:] == 0).all()
