"""CPU: the adapters and the losses refuse dual tensors of forward-mode differentiation, whose tangents they would drop."""
from __future__ import annotations

from importlib import import_module

import pytest

torch = pytest.importorskip("torch")
from torch._subclasses.fake_tensor import FakeTensorMode  # noqa: E402
from torch.autograd import forward_ad  # noqa: E402

BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32


@pytest.fixture
def fake():
    """Tensors "on the GPU" without one: their data is never touched by a refused call."""
    with FakeTensorMode(), forward_ad.dual_level():
        yield lambda *s, dtype=F32: torch.empty(*s, dtype=dtype, device="cuda")


def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


def test_has_tangent(pkg):
    lib = import_module(pkg.__name__ + "._lib")
    t = torch.zeros(3)
    assert not lib.has_tangent(t, None)
    with forward_ad.dual_level():
        d = dual(t)
        assert not d.requires_grad and lib.has_tangent(t, None, d) and not lib.has_tangent(t, None)
        with torch.no_grad():
            assert lib.has_tangent(d)
    assert not lib.has_tangent(d)


@pytest.mark.parametrize("which", ["logits", "old", "adv", "ref", "weight", "out"])
def test_policy(pkg, fake, which):
    losses = import_module(pkg.__name__ + ".losses")
    t = dict(logits=fake(4, 100), tokens=fake(4, dtype=I32), old=fake(4), adv=fake(4), ref=fake(4), weight=fake(4))
    out = fake(4, 100)
    if which == "out":
        out = dual(out)
    else:
        t[which] = dual(t[which])
        with pytest.raises(ValueError, match="policy_loss"):
            losses.policy_loss(*t.values(), kl=0.1)
    with pytest.raises(ValueError, match="policy_loss_grad"):
        losses.policy_loss_grad(*t.values(), kl=0.1, out=out)


@pytest.mark.parametrize("which", ["logits", "v", "weight", "out"])
def test_distill(pkg, fake, which):
    losses = import_module(pkg.__name__ + ".losses")
    t = dict(logits=fake(4, 100), ids=fake(4, 5, dtype=I32), v=fake(4, 5), weight=fake(4))
    out = fake(4, 100)
    if which == "out":
        out = dual(out)
    else:
        t[which] = dual(t[which])
        with pytest.raises(ValueError, match="distill_top"):
            losses.distill_top(*t.values())
    with pytest.raises(ValueError, match="distill_top_grad"):
        losses.distill_top_grad(*t.values(), out=out)


@pytest.mark.parametrize("which", ["y", "x", "a", "b", "scale", "out", "hidden"])
def test_lora(pkg, fake, which, monkeypatch):
    lora = import_module(pkg.__name__ + ".lora")
    monkeypatch.setattr(lora, "_overlap", lambda s, t: False)        # (no addresses here)
    t = dict(y=fake(5, 40, dtype=BF), x=fake(5, 32, dtype=BF), a=fake(3, 8, 32, dtype=BF), b=fake(3, 40, 8, dtype=BF),
             scale=fake(3), out=fake(5, 40, dtype=BF), hidden=fake(5, 8))
    t[which] = dual(t[which])
    rows = lora.LoraRows(fake(5, dtype=I32), fake(5, 4, dtype=I32), fake(8, dtype=I32), 5, 3, 16)
    w = lora.LoraStack(t["a"], t["b"], t["scale"])
    with pytest.raises(ValueError, match="add_lora has no forward"):
        lora.add_lora(t["y"], t["x"], w, rows, t["out"], t["hidden"])
    if which != "out":
        with pytest.raises(ValueError, match="add_lora_grad"):
            lora.add_lora_grad(t["y"], t["x"], w, rows, t["hidden"])
