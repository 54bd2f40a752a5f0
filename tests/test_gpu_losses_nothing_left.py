"""losses.distill_top where no token is left for the rest that a teacher's list leaves, as all tokens are listed or those
that are not are at -inf: the loss lacks the rest's term, and its gradient is the gradient of that loss. The loss does not
change where a row's logits are all moved by the same amount, so the gradient's sum over the row is 0."""
from __future__ import annotations

from importlib import import_module

import pytest

import test_gpu_losses as base
from conftest import gpu_case
from test_gpu_losses import DEV, LP, NINF, STEP, SUM, TINY, TYPES, near, near_grad

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def losses(pkg):
    return import_module(pkg.__name__ + ".losses")


def exact(x, ids, v, w, T=1.0):
    """The loss of rows of which nothing but the listed tokens is left, and its gradient by float64 differentiation; by how
    much both may be off (as base.exact_distill has it, p times the listed probabilities' sum in place of p)."""
    at, v, w = ids.long(), v.double(), w.double()
    q = v.exp()
    z = x.gather(1, at).double().requires_grad_()
    lp = torch.log_softmax(z / T, 1)
    cost = torch.where(q > 0, q * (v - lp), 0.0)
    (g,) = torch.autograd.grad(cost.sum(), z)
    loss, lp = cost.detach().sum(1), lp.detach()
    sp = q.sum(1, keepdim=True) * lp.exp()
    loss_err = (q * (LP * (1 + lp.abs()) + 40 * STEP * (1 + v.abs().clamp(max=1e4)))).sum(1) + 40 * STEP * cost.detach().abs().sum(1)
    err = (2 * SUM + 16 * STEP) * sp + 40 * STEP * (sp + q) + TINY
    full = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
    w = w[:, None]
    return ((loss[:, None] * w)[:, 0], (w.abs() * loss_err[:, None])[:, 0], full.scatter(1, at, g * w),
            full.scatter(1, at, err * w.abs() / T))


def rows(R, V, top, dtype, seed, most=0.9):
    """Finite logits for the listed tokens alone; probabilities that sum to `most` or less, down to 0.1."""
    g = torch.Generator(DEV).manual_seed(seed)
    ids = torch.stack([torch.randperm(V, generator=g, device=DEV)[:top] for _ in range(R)]).int()
    x = torch.full((R, V), NINF, dtype=TYPES[dtype], device=DEV)
    x.scatter_(1, ids.long(), (3 * torch.randn(R, top, generator=g, device=DEV)).to(x.dtype))
    sums = most - (most - 0.1) * torch.rand(R, 1, generator=g, device=DEV, dtype=torch.float64)
    v = (torch.log_softmax(2 * torch.randn(R, top, generator=g, device=DEV, dtype=torch.float64), 1) + sums.log()).float()
    return x, ids, v, torch.rand(R, generator=g, device=DEV) + 0.1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R", [8, 300])
@pytest.mark.parametrize("V,top", [(1, 1), (2, 2), (9, 9), (32, 32), (50, 5), (3000, 20), (70001, 32)])
@pytest.mark.parametrize("T", [1.0, 0.5])
def test_the_gradient_is_the_losses(losses, dtype, R, V, top, T):
    x, ids, v, w = rows(R, V, top, dtype, R + V)
    gpu_case(f"distill, only the listed left, {dtype} R={R} V={V} top={top} T={T}")
    loss, grad = losses.distill_top_grad(x, ids, v, w, temperature=T)
    only = losses.distill_top(x, ids, v, w, temperature=T)
    torch.cuda.synchronize()
    want, loss_err, g, err = exact(x, ids, v, w, T)
    near(loss, want, loss_err, "loss")
    near_grad(grad, g, err)
    assert torch.equal(only, loss)
    assert (grad.scatter(1, ids.long(), 0.0) == 0).all()
    step = torch.finfo(grad.dtype)
    limit = (err + step.eps / 2 * (g.abs() + err) + step.smallest_normal * step.eps / 2).sum(1)
    assert (grad.double().sum(1).abs() <= limit).all()


def test_three_logits(losses):
    """Logits 1, .5, -.3 and nothing else, probabilities .3, .2, .1: (sum q) p - q, by hand."""
    x = torch.full((1, 40), NINF, device=DEV)
    x[0, :3] = torch.tensor([1.0, 0.5, -0.3])
    q = torch.tensor([0.3, 0.2, 0.1], dtype=torch.float64, device=DEV)
    gpu_case("distill of three logits")
    _, grad = losses.distill_top_grad(x, torch.arange(3, device=DEV, dtype=torch.int32)[None], q.log().float()[None])
    torch.cuda.synchronize()
    e = x[0, :3].double().exp()
    torch.testing.assert_close(grad[0, :3].double(), 0.6 * e / e.sum() - q, rtol=0, atol=2 * SUM + 60 * STEP)


@pytest.mark.parametrize("R", [5, 256])
def test_against_differences(losses, R):
    """As base.test_gradients_against_differences, along directions of the listed tokens."""
    x, ids, v, w = rows(R, 37, 6, "f32", 3, 0.6)
    h = 2.0 ** -6
    limit = 8 * LP / h + 10 * h * h / 6 * 4
    g = torch.Generator(DEV).manual_seed(5)
    gpu_case("distill, only the listed left, against differences")
    _, grad = losses.distill_top_grad(x, ids, v, w)
    for _ in range(5):
        d = torch.zeros_like(x).scatter_(1, ids.long(), torch.randn(R, 6, generator=g, device=DEV))
        d /= d.norm(dim=1, keepdim=True)
        by = (losses.distill_top(x + h * d, ids, v, w).double() - losses.distill_top(x - h * d, ids, v, w).double()) / (2 * h)
        got = (grad.double() * d.double()).sum(1)
        assert ((by - got).abs() <= limit * (1 + got.abs())).all(), (by - got).abs().max()


# What base holds for other rows, masks and sizes, with the gradient of the loss where nothing is left.
EXACT = base.exact_distill


def exact_distill(x, ids, v, w, rest, T):
    loss, loss_err, g, err = EXACT(x, ids, v, w, rest, T)
    none = ((x > NINF).scatter(1, ids.long(), False).sum(1) == 0) & bool(rest)
    if none.any():
        _, _, g[none], err[none] = exact(x[none], ids[none], v[none], w[none], T)
    return loss, loss_err, g, err


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,offset", [(8, 50, 0), (8, 3000, 1), (8, 70001, 3), (264, 3000, 1)])
def test_masked_rows(losses, monkeypatch, dtype, R, V, offset):
    monkeypatch.setattr(base, "exact_distill", exact_distill)
    base.test_masked_rows(losses, dtype, R, V, offset)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,pad,offset", [s for s in base.SIZES if s[1] <= 32])
def test_short_vocabularies(losses, monkeypatch, dtype, R, V, pad, offset):
    monkeypatch.setattr(base, "exact_distill", exact_distill)
    base.test_distill(losses, dtype, R, V, pad, offset)
