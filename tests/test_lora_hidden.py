"""add_lora's hidden, which it writes as it does out: apart from the other operands (CPU), and told to autograd."""
from __future__ import annotations

from importlib import import_module

import pytest

from conftest import gpu_case

torch = pytest.importorskip("torch")
BF = torch.bfloat16


@pytest.fixture
def lora(pkg):
    return import_module(pkg.__name__ + ".lora")


class Stack:
    """What add_lora reads of a stack before it launches anything."""

    def __init__(self, n, R, K, N):
        self.a, self.b, self.scale = torch.zeros(n, R, K, dtype=BF), torch.zeros(n, N, R, dtype=BF), torch.ones(n)
        self.n, self.rank = n, R


@pytest.mark.parametrize("which", ["x", "y", "out"])
def test_hidden_must_lie_apart(lora, monkeypatch, which):
    monkeypatch.setattr(lora, "_forward", lambda *a: None)           # (the tensors are on the CPU)
    i32 = dict(dtype=torch.int32)
    rows = lora.LoraRows(torch.zeros(5, **i32), torch.zeros(5, 4, **i32), torch.zeros(8, **i32), 5, 3, 16)
    t = dict(x=torch.zeros(5, 32, dtype=BF), y=torch.zeros(5, 40, dtype=BF), out=torch.zeros(5, 40, dtype=BF))
    w = Stack(3, 8, 32, 40)
    assert lora.add_lora(t["y"], t["x"], w, rows, t["out"], torch.empty(5, 8)) is t["out"]
    buf = torch.empty(5 * 20)
    cols = t[which].shape[1]
    t[which] = buf.view(BF)[:5 * cols].view(5, cols)                 # 80 or 100 of the 100 floats
    with pytest.raises(ValueError, match="hidden overlaps"):
        lora.add_lora(t["y"], t["x"], w, rows, t["out"], buf[60:].view(5, 8))
    assert lora.add_lora(t["y"], t["x"], w, rows, t["out"], torch.empty(5, 8)) is t["out"]


@pytest.mark.gpu
def test_autograd_notices_a_hidden_that_was_written_over(lora):
    g = torch.Generator("cuda").manual_seed(1)
    e = lambda *s: torch.randn(*s, generator=g, device="cuda").to(BF)                  # noqa: E731
    w = lora.LoraStack(e(2, 8, 64), e(2, 72, 8), torch.ones(2, device="cuda"))
    rows = lora.plan_rows(torch.arange(20, device="cuda") % 2, 2)
    x, y = e(20, 64), e(20, 72)
    leaf = torch.randn(20, 8, generator=g, device="cuda", requires_grad=True)
    hidden = torch.sigmoid(leaf)                                     # (whose backward pass asks for it)
    gpu_case("lora into a hidden beside autograd")
    lora.add_lora(y, x, w, rows, hidden=hidden.detach())
    with pytest.raises(RuntimeError, match="inplace"):
        hidden.sum().backward()
    torch.cuda.synchronize()
