"""CPU: what the adapters refuse, without a GPU: the Python checks on tensors that have a shape and a device but
no memory, the library's own on its return codes."""
from __future__ import annotations

import ctypes
from importlib import import_module

import pytest

torch = pytest.importorskip("torch")
from torch._subclasses.fake_tensor import FakeTensorMode  # noqa: E402

P = ctypes.c_void_p
BF, F16, I32, I64 = torch.bfloat16, torch.float16, torch.int32, torch.int64


@pytest.fixture
def lora(pkg):
    return import_module(pkg.__name__ + ".lora")


@pytest.fixture
def fake():
    """Tensors "on the GPU" without one: their data is never touched by a refused call."""
    with FakeTensorMode():
        yield lambda *s, dtype=BF, device="cuda": torch.empty(*s, dtype=dtype, device=device)


@pytest.fixture
def lib(pkg):
    if not pkg.LIB_PATH.exists():
        pytest.skip("librlu.so not built")
    return pkg.lib()


def stack(lora, e, n=3, R=8, K=32, N=40, dtype=BF):
    return lora.LoraStack(e(n, R, K, dtype=dtype), e(n, N, R, dtype=dtype), e(n, dtype=torch.float32))


def planned(lora, e, rows=5, n=3):
    return lora.LoraRows(e(rows, dtype=I32), e(rows, 4, dtype=I32), e(n + 5, dtype=I32), rows, n, 16)


@pytest.mark.parametrize("bad", [
    dict(a=lambda e: e(3, 8)), dict(a=lambda e: e(3, 8, 32, dtype=torch.float32)),
    dict(a=lambda e: e(3, 8, 32, dtype=F16)), dict(a=lambda e: e(3, 8, 32, device="cpu")),
    dict(a=lambda e: e(3, 32, 8).transpose(1, 2)), dict(a=lambda e: e(2, 8, 32)),
    dict(a=lambda e: e(3, 9, 32)), dict(b=lambda e: e(3, 40, 9)), dict(b=lambda e: e(4, 40, 8)),
    dict(b=lambda e: e(3, 0, 8)), dict(a=lambda e: e(3, 8, 0)),
    dict(a=lambda e: e(3, 129, 32), b=lambda e: e(3, 40, 129)),
    dict(a=lambda e: e(3, 0, 32), b=lambda e: e(3, 40, 0)),
    dict(a=lambda e: e(1025, 8, 32), b=lambda e: e(1025, 40, 8), s=lambda e: e(1025, dtype=torch.float32)),
    dict(a=lambda e: e(0, 8, 32), b=lambda e: e(0, 40, 8), s=lambda e: e(0, dtype=torch.float32)),
    dict(s=lambda e: e(3)), dict(s=lambda e: e(2, dtype=torch.float32)),
    dict(s=lambda e: e(3, dtype=torch.float32, device="cpu")),
    dict(s=lambda e: e(3, dtype=torch.float32).requires_grad_())])
def test_a_stack_refuses(lora, fake, bad):
    kw = dict(a=lambda e: e(3, 8, 32), b=lambda e: e(3, 40, 8), s=lambda e: e(3, dtype=torch.float32))
    kw.update(bad)
    with pytest.raises(ValueError, match="LoraStack"):
        lora.LoraStack(*[kw[k](fake) for k in ("a", "b", "s")])


@pytest.mark.parametrize("ids,n", [
    (lambda e: e(5, dtype=torch.float32), 3), (lambda e: e(5, 1, dtype=I32), 3),
    (lambda e: e(10, dtype=I32)[::2], 3), (lambda e: e(5, dtype=I32, device="cpu"), 3),
    (lambda e: e(5, dtype=I32), 0), (lambda e: e(5, dtype=I64), 1025),
    (lambda e: e((1 << 24) + 1, dtype=I32), 3)])
def test_plan_rows_refuses(lora, fake, ids, n):
    with pytest.raises(ValueError, match="plan_rows"):
        lora.plan_rows(ids(fake), n)


ROWS = [dict(x=lambda e: e(5, 33)), dict(x=lambda e: e(4, 32)), dict(x=lambda e: e(5, 32, dtype=F16)),
        dict(x=lambda e: e(5, 32, device="cpu")), dict(x=lambda e: e(32, 5).T), dict(x=lambda e: e(5, 64)[:, ::2]),
        dict(x=lambda e: e(160)),
        dict(y=lambda e: e(5, 41)), dict(y=lambda e: e(6, 40)), dict(y=lambda e: e(5, 40, dtype=torch.float32)),
        dict(y=lambda e: e(40, 5).T),
        dict(hidden=lambda e: e(5, 9, dtype=torch.float32)), dict(hidden=lambda e: e(5, 8)),
        dict(hidden=lambda e: e(5, 16, dtype=torch.float32)[:, :8]),
        dict(hidden=lambda e: e(5, 8, dtype=torch.float32).requires_grad_()),
        dict(rows=4), dict(n=2)]


@pytest.mark.parametrize("bad", ROWS + [
    dict(out=lambda e: e(5, 41)), dict(out=lambda e: e(5, 40, dtype=F16)), dict(out=lambda e: e(40, 5).T),
    dict(out=lambda e: e(1, 40).expand(5, 40)), dict(out=lambda e: e(5, 40, device="cpu")),
    dict(x=lambda e: e(5, 32).requires_grad_(), out=lambda e: e(5, 40)),
    dict(x=lambda e: e(5, 32).requires_grad_())])
def test_add_lora_refuses(lora, fake, bad, monkeypatch):
    monkeypatch.setattr(lora, "_overlap", lambda s, t: False)        # (no addresses here)
    kw = dict(y=lambda e: e(5, 40), x=lambda e: e(5, 32), out=lambda e: None,
              hidden=lambda e: e(5, 8, dtype=torch.float32), rows=5, n=3)
    kw.update(bad)
    with pytest.raises(ValueError, match="add_lora"):
        lora.add_lora(kw["y"](fake), kw["x"](fake), stack(lora, fake),
                      planned(lora, fake, kw["rows"], kw["n"]), kw["out"](fake), kw["hidden"](fake))


@pytest.mark.parametrize("bad", ROWS + [dict(x=lambda e: e(5, 32).requires_grad_()),
                                        dict(y=lambda e: e(5, 40).requires_grad_()), dict(need=(True, False))])
def test_add_lora_grad_refuses(lora, fake, bad):
    kw = dict(y=lambda e: e(5, 40), x=lambda e: e(5, 32), hidden=lambda e: e(5, 8, dtype=torch.float32),
              rows=5, n=3, need=(True, True, True))
    kw.update(bad)
    with pytest.raises(ValueError, match="add_lora_grad"):
        lora.add_lora_grad(kw["y"](fake), kw["x"](fake), stack(lora, fake),
                           planned(lora, fake, kw["rows"], kw["n"]), kw["hidden"](fake), kw["need"])


def test_overlap(lora):
    buf = torch.zeros(4, 32)
    assert lora._overlap(buf[:, :10], buf[:, 5:15]) and lora._overlap(buf[:, :10], buf[:, 20:])
    assert not lora._overlap(buf[:2], buf[2:]) and not lora._overlap(buf, torch.zeros(4, 32))
    assert not lora._overlap(buf[:0], buf)


def test_return_codes(lib):
    a = P(4096)

    def plan(ids=a, wide=0, rows=20, n=3, size=16, cap=6, order=a, tiles=a, first=a):
        return lib.rlu_lora_plan(ids, wide, rows, n, size, cap, order, tiles, first, P(0))
    assert plan(rows=0, cap=0) == 0
    for kw in (dict(wide=2), dict(rows=-1), dict(n=0), dict(n=1025), dict(size=32), dict(cap=5),
               dict(cap=7), dict(ids=P(0)), dict(order=P(0)), dict(tiles=P(0)), dict(first=P(0))):
        assert plan(**kw) == -1, kw
    for kw in (dict(tiles=P(4104)), dict(order=P(4098)), dict(first=P(4098))):
        assert plan(**kw) == -4, kw

    def add(x=a, ldx=32, A=a, b=a, s=a, dtype=0, order=a, tiles=a, first=a, rows=20, n=3, size=16, cap=6, K=32,
            N=40, R=8, hidden=a, y=a, ldy=40, out=a, ldo=40):
        return lib.rlu_lora_add(x, ldx, A, b, s, dtype, order, tiles, first, rows, n, size, cap, K, N, R,
                                hidden, y, ldy, out, ldo, P(0))
    assert add(rows=0, cap=0) == 0
    wrong = (dict(dtype=1), dict(dtype=3), dict(R=0), dict(R=129), dict(K=0), dict(N=0), dict(K=(1 << 24) + 1),
             dict(N=(1 << 24) + 1), dict(cap=7), dict(n=0), dict(ldx=-1), dict(x=P(0)), dict(A=P(0)),
             dict(b=P(0)), dict(s=P(0)), dict(order=P(0)), dict(tiles=P(0)), dict(first=P(0)), dict(hidden=P(0)))
    for kw in wrong + (dict(y=P(0)), dict(out=P(0)), dict(ldo=39), dict(ldy=-1),
                       dict(rows=1 << 24, size=16, cap=(1 << 20) + 5, N=1 << 24, ldo=1 << 24)):
        assert add(**kw) == -1, kw
    odd = (dict(x=P(4097)), dict(A=P(4097)), dict(b=P(4097)), dict(s=P(4098)), dict(hidden=P(4098)),
           dict(order=P(4098)), dict(tiles=P(4104)))
    for kw in odd + (dict(y=P(4097)), dict(out=P(4097))):
        assert add(**kw) == -4, kw

    def grad(dy=a, lddy=40, x=a, ldx=32, A=a, b=a, s=a, dtype=0, order=a, tiles=a, first=a, rows=20, n=3, size=16,
             cap=6, K=32, N=40, R=8, hidden=a, dx=a, lddx=32, da=a, db=a, ws=a):
        return lib.rlu_lora_grad(dy, lddy, x, ldx, A, b, s, dtype, order, tiles, first, rows, n, size, cap, K,
                                 N, R, hidden, dx, lddx, da, db, ws, P(0))
    assert grad(rows=0, cap=0) == 0
    for kw in wrong + (dict(dy=P(0)), dict(ws=P(0)), dict(lddy=-1), dict(lddx=31)):
        assert grad(**kw) == -1, kw
    for kw in odd + (dict(dy=P(4097)), dict(dx=P(4097)), dict(da=P(4097)), dict(db=P(4097)), dict(ws=P(4104))):
        assert grad(**kw) == -4, kw
    n = ctypes.c_longlong(-7)
    assert lib.rlu_lora_grad_workspace(0, 20, 3, 16, 6, 32, 40, 8, ctypes.byref(n)) == 0 and n.value > 0
    assert lib.rlu_lora_grad_workspace(0, 20, 3, 16, 6, 32, 40, 129, ctypes.byref(n)) == -1
    assert lib.rlu_lora_grad_workspace(0, 20, 3, 16, 6, 32, 40, 8, P(0)) == -1
