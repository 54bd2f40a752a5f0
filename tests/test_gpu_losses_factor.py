"""The losses under autograd with an incoming factor other than 1, a loss scale above all: the gradient times the factor
is rounded to the logits' type once, so what 16 bits cannot hold without the factor is there with it."""
from __future__ import annotations

from importlib import import_module

import pytest

from conftest import gpu_case
from test_gpu_losses import (CLIP, DEV, INF, NAN, STEP, TYPES, exact_distill, exact_policy, near_grad, policy_of, rows_of,
                             teacher_of)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def losses(pkg):
    return import_module(pkg.__name__ + ".losses")


def policy_case(losses, x, tok, seed):
    """A loss of logits, and the exact gradient of its sum with its limit."""
    old, adv, ref, w = policy_of(x, tok, seed)
    w = w / x.shape[0]
    want = exact_policy(x, tok, old, adv, ref, w, CLIP, 0.05, 1.0)
    return (lambda t: losses.policy_loss(t, tok, old, adv, ref, w, clip=CLIP, kl=0.05).loss), want[4], want[5], \
        lambda t: losses.policy_loss_grad(t, tok, old, adv, ref, w, clip=CLIP, kl=0.05)[1]


def distill_case(losses, x, tok, seed, rest=True):
    ids, v, w = teacher_of(x, 9, seed)
    w = w / x.shape[0]
    want = exact_distill(x, ids, v, w, rest, 1.0)
    return (lambda t: losses.distill_top(t, ids, v, w, rest=rest)), want[2], want[3], \
        lambda t: losses.distill_top_grad(t, ids, v, w, rest=rest)[1]


CASES = {"policy": policy_case, "distill": distill_case,
         "distill listed": lambda *a: distill_case(*a, rest=False)}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", CASES)
@pytest.mark.parametrize("R,V,pad,offset", [(7, 3001, 1, 1), (300, 50001, 3, 2), (9, 60000, 0, 0), (300, 1500, 0, 0)])
def test_a_loss_scale_meets_the_gradient_before_its_rounding(losses, dtype, kind, R, V, pad, offset):
    """Weights of 1 / R and a scale of 2^16, or 2^10 a row and more: float16 alone would hold few of these at all."""
    x, tok = rows_of(R, V, dtype, R + V, pad, offset)
    f, g, err, by_hand = CASES[kind](losses, x, tok, R)
    gen = torch.Generator(DEV).manual_seed(R)
    rows = torch.exp2(10 + 4 * torch.rand(R, generator=gen, device=DEV)) * (1 - 2 * (torch.arange(R, device=DEV) % 2))
    rows[2], rows[4] = 1.0, 0.0
    gpu_case(f"losses autograd {dtype} {kind} R={R} V={V} with a scale")
    for by in (torch.full((R,), 2.0 ** 16, device=DEV), rows):
        leaf = x.detach().requires_grad_()
        (got,) = torch.autograd.grad(f(leaf), leaf, by)
        torch.cuda.synchronize()
        product = g * by.double()[:, None]
        # (the weight times the factor, or the gradient in float32 times it, is rounded once in float32)
        near_grad(got, product, err * by.double().abs()[:, None] + 2 * STEP * product.abs())
    assert torch.equal(got[2], by_hand(x)[2]) and (got[4] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", CASES)
@pytest.mark.parametrize("R", [7, 300])
def test_sums_and_means(losses, dtype, kind, R):
    """The rows' sum gives the gradient by hand, bit for bit, and adds up; a mean's factor is rounded with it; the
    gradient is handed out once."""
    x, tok = rows_of(R, 3001, dtype, 6, 1, 1)
    f, g, err, by_hand = CASES[kind](losses, x, tok, 6)
    want = by_hand(x)
    gpu_case(f"losses autograd {dtype} {kind} sums")
    leaf = x.detach().requires_grad_()
    f(leaf).sum().backward()
    assert torch.equal(leaf.grad, want)
    f(leaf).sum().backward()
    assert torch.equal(leaf.grad, want + want)
    (got,) = torch.autograd.grad(f(leaf).mean(), leaf)
    near_grad(got, g / R, err / R + 3 * STEP * g.abs() / R)
    loss = f(leaf).sum() * 3.0
    loss.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        loss.backward()
    with torch.no_grad():
        assert not f(leaf).requires_grad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R", [12, 300])
def test_padded_and_broken_rows(losses, dtype, R):
    """A row of weight 0 has no gradient whatever comes in; a NaN row is NaN and the others are as they would be."""
    x, tok = rows_of(R, 3000, dtype, 8)
    ids, v, w = teacher_of(x, 4, 8)
    w = w + 0.1
    x[1, 7], x[2], w[2] = NAN, NAN, 0.0
    by = torch.full((R,), 0.37, device=DEV)
    by[2] = INF if dtype != "f32" else 2.0                           # (float32's zeros are multiplied)
    fine = [r for r in range(R) if r not in (1, 2)]
    gpu_case(f"losses autograd {dtype} NaN rows")
    leaf = x.detach().requires_grad_()
    (got,) = torch.autograd.grad(losses.distill_top(leaf, ids, v, w), leaf, by)
    torch.cuda.synchronize()
    assert got[1].isnan().all() and (got[2] == 0).all()
    _, _, g, err = exact_distill(x[fine], ids[fine], v[fine], w[fine], True, 1.0)
    near_grad(got[fine], 0.37 * g, 0.37 * err + 3 * STEP * g.abs())


def test_logits_written_to_before_the_backward_pass(losses):
    """Autograd keeps 16-bit logits for the factor, and says so when they are no longer there."""
    for dtype in TYPES:
        x, tok = rows_of(6, 500, dtype, 3)
        ids, v, w = teacher_of(x, 4, 3)
        leaf = x.detach().requires_grad_()
        gpu_case(f"losses autograd {dtype}, logits written to")
        loss = losses.distill_top(leaf, ids, v, w).sum()
        with torch.no_grad():
            leaf.zero_()
        if dtype == "f32":
            loss.backward()
        else:
            with pytest.raises(RuntimeError, match="inplace"):
                loss.backward()
    torch.cuda.synchronize()


def test_streams(losses):
    """Forward and backward passes on three streams at once, each with its own factor."""
    x, tok = rows_of(40, 20001, "f16", 1)
    ids, v, w = teacher_of(x, 20, 1)
    by = [torch.full((40,), s, device=DEV) for s in (2.0, 512.0, 1.0)]
    want = []
    for b in by:
        leaf = x.detach().requires_grad_()
        want += torch.autograd.grad(losses.distill_top(leaf, ids, v, w), leaf, b)
    gpu_case("losses autograd on three streams")
    torch.cuda.synchronize()
    got = []
    for st, b in zip([torch.cuda.Stream() for _ in range(3)], by):
        with torch.cuda.stream(st):
            leaf = x.detach().requires_grad_()
            got += torch.autograd.grad(losses.distill_top(leaf, ids, v, w), leaf, b)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
