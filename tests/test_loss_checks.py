"""CPU: what the losses refuse, without a GPU: the Python checks on tensors that have a shape and a device but
no memory, the library's own on its return codes."""
from __future__ import annotations

import ctypes
from importlib import import_module

import pytest

torch = pytest.importorskip("torch")
from torch._subclasses.fake_tensor import FakeTensorMode  # noqa: E402

P = ctypes.c_void_p
I64, I32, F64, BF = torch.int64, torch.int32, torch.float64, torch.bfloat16


@pytest.fixture
def losses(pkg):
    return import_module(pkg.__name__ + ".losses")


@pytest.fixture
def fake():
    """Tensors "on the GPU" without one: their data is never touched by a refused call."""
    with FakeTensorMode():
        yield lambda *s, dtype=torch.float32, device="cuda": torch.empty(*s, dtype=dtype,
                                                                        device=device)


@pytest.fixture
def lib(pkg):
    if not pkg.LIB_PATH.exists():
        pytest.skip("librlu.so not built")
    return pkg.lib()


LOGITS = [
    dict(logits=lambda e: e(4, 100, device="cpu")),
    dict(logits=lambda e: e(4, 100, dtype=F64)),
    dict(logits=lambda e: e(400)),
    dict(logits=lambda e: e(4, 0)),
    dict(logits=lambda e: e(4, 500001)),
    dict(logits=lambda e: e(100, 4).T),
    dict(logits=lambda e: e(4, 200)[:, ::2]),
    dict(weight=lambda e: e(4, dtype=BF)),
    dict(weight=lambda e: e(3)),
    dict(weight=lambda e: e(1).expand(4)),
    dict(weight=lambda e: e(4).requires_grad_()),
    dict(temperature=lambda e: 0.0), dict(temperature=lambda e: -1.0),
    dict(temperature=lambda e: float("nan")), dict(temperature=lambda e: float("inf")),
]
OUT = [
    dict(logits=lambda e: e(4, 100).requires_grad_()),
    dict(out=lambda e: e(4, 99)), dict(out=lambda e: e(4, 100, dtype=BF)),
    dict(out=lambda e: e(4, 100, device="cpu")), dict(out=lambda e: e(100, 4).T),
    dict(out=lambda e: e(1, 100).expand(4, 100)), dict(out=lambda e: e(4, 100).requires_grad_())]


@pytest.mark.parametrize("bad", LOGITS + [
    dict(tokens=lambda e: e(3, dtype=I64)), dict(tokens=lambda e: e(4, 1, dtype=I64)),
    dict(tokens=lambda e: e(4)), dict(tokens=lambda e: e(8, dtype=I64)[::2]),
    dict(tokens=lambda e: e(4, dtype=I64, device="cpu")),
    dict(old=lambda e: e(5)), dict(old=lambda e: e(4, dtype=F64)),
    dict(old=lambda e: e(4).requires_grad_()),
    dict(adv=lambda e: e(4, device="cpu")), dict(adv=lambda e: e(8)[::2]),
    dict(ref=lambda e: e(4, 1)), dict(kl=lambda e: 0.1, ref=lambda e: None),
    dict(kl=lambda e: -0.1), dict(kl=lambda e: float("nan")), dict(kl=lambda e: float("inf")),
    dict(clip=lambda e: (0.1,)), dict(clip=lambda e: (1.1, 0.2)), dict(clip=lambda e: (-0.1, 0.2)),
    dict(clip=lambda e: (0.1, -0.2)), dict(clip=lambda e: (float("nan"), 0.2))])
def test_policy_refuses(losses, fake, bad):
    kw = dict(logits=fake(4, 100), tokens=fake(4, dtype=I64), old=fake(4), adv=fake(4), ref=fake(4),
              weight=fake(4), clip=(0.2, 0.2), kl=0.0, temperature=1.0)
    kw.update({k: f(fake) for k, f in bad.items()})
    more = {k: kw[k] for k in ("clip", "kl", "temperature")}
    args = [kw[k] for k in ("logits", "tokens", "old", "adv", "ref", "weight")]
    for name in ("policy_loss", "policy_loss_grad"):
        with pytest.raises(ValueError, match=name):
            getattr(losses, name)(*args, **more)


@pytest.mark.parametrize("bad", LOGITS + [
    dict(ids=lambda e: e(4, 0, dtype=I32), v=lambda e: e(4, 0)),
    dict(ids=lambda e: e(4, 33, dtype=I32), v=lambda e: e(4, 33)),
    dict(ids=lambda e: e(4, dtype=I32)), dict(ids=lambda e: e(3, 5, dtype=I32)),
    dict(ids=lambda e: e(4, 5, dtype=I64)), dict(ids=lambda e: e(4, 10, dtype=I32)[:, :5]),
    dict(v=lambda e: e(4, 6)), dict(v=lambda e: e(4, 5, dtype=BF)),
    dict(v=lambda e: e(5, 4).T), dict(v=lambda e: e(4, 5).requires_grad_())])
def test_distill_refuses(losses, fake, bad):
    kw = dict(logits=fake(4, 100), ids=fake(4, 5, dtype=I32), v=fake(4, 5), weight=fake(4),
              temperature=1.0)
    kw.update({k: f(fake) for k, f in bad.items()})
    args = [kw[k] for k in ("logits", "ids", "v", "weight")]
    for name in ("distill_top", "distill_top_grad"):
        with pytest.raises(ValueError, match=name):
            getattr(losses, name)(*args, temperature=kw["temperature"])


@pytest.mark.parametrize("bad", OUT)
def test_gradients_by_hand_refuse(losses, fake, bad):
    kw = dict(logits=fake(4, 100), out=None)
    kw.update({k: f(fake) for k, f in bad.items()})
    with pytest.raises(ValueError, match="policy_loss_grad"):
        losses.policy_loss_grad(kw["logits"], fake(4, dtype=I64), fake(4), fake(4), out=kw["out"])
    with pytest.raises(ValueError, match="distill_top_grad"):
        losses.distill_top_grad(kw["logits"], fake(4, 3, dtype=I32), fake(4, 3), out=kw["out"])


def test_out_may_be_the_logits_but_not_overlap_them(losses):
    buf = torch.zeros(4, 32)
    x = buf[:, :10]
    losses._check_out("f", x, x)
    losses._check_out("f", torch.zeros(4, 10), x)
    losses._check_out("f", buf.view(8, 16)[4:, :10], buf.view(8, 16)[:4, :10])
    for out in (buf[:, 1:11], buf[:, 16:26], buf.view(8, 16)[:4, :10], buf.view(8, 16)[1:5, :10]):
        with pytest.raises(ValueError, match="overlaps"):
            losses._check_out("f", out, x)


def test_the_gradients_buffer_starts_where_the_logits_do(losses):
    for rows, vocab, pad, off in ((3, 10, 0, 0), (3, 10, 5, 1), (1, 7, 0, 3), (4, 9, 13, 7), (2, 8, 0, 0)):
        for dtype in (torch.float32, BF):
            x = torch.zeros(rows * (vocab + pad) + off, dtype=dtype)[off:].view(rows, -1)[:, :vocab]
            g = losses._grad_like(x)
            assert g.shape == x.shape and g.dtype == dtype and (rows == 1 or g.stride(0) >= vocab)
            for r in range(rows):
                assert (g[r].data_ptr() - x[r].data_ptr()) % 16 == 0


def test_return_codes(lib):
    n, a = ctypes.c_longlong(-7), P(4096)
    ws = lib.rlu_loss_workspace
    assert ws(0, 3, 10, 1, ctypes.byref(n)) == 0 and n.value >= 0
    for bad in ((3, 3, 10, 1), (-1, 3, 10, 1), (0, -1, 10, 1), (0, 3, 0, 1), (0, 3, 500001, 1),
                (0, 3, 10, 0), (0, 3, 10, 33), (0, 2 ** 23, 10, 1)):
        assert ws(*bad, ctypes.byref(n)) == -1
    assert ws(0, 3, 10, 1, P(0)) == -1

    def policy(logits=a, dtype=0, ld=10, R=4, V=10, tokens=a, wide=1, old=a, adv=a, ref=a, w=a, lo=0.2,
               hi=0.2, kl=0.1, T=1.0, loss=a, lp=a, grad=a, ldg=10, s=a):
        return lib.rlu_policy_loss(logits, dtype, ld, R, V, tokens, wide, old, adv, ref, w, lo, hi, kl,
                                   T, loss, lp, grad, ldg, s, P(0))
    assert policy(R=0) == 0
    nan, inf = float("nan"), float("inf")
    for kw in (dict(dtype=3), dict(ld=-1), dict(R=-1), dict(V=0), dict(V=500001), dict(wide=2),
               dict(lo=-0.1), dict(lo=1.5), dict(lo=nan), dict(hi=-0.1), dict(hi=nan), dict(kl=-1.0),
               dict(kl=nan), dict(kl=inf), dict(T=0.0), dict(T=nan), dict(T=inf), dict(T=1e-40),
               dict(logits=P(0)), dict(tokens=P(0)), dict(old=P(0)), dict(adv=P(0)), dict(loss=P(0)),
               dict(lp=P(0)), dict(s=P(0)), dict(ldg=9), dict(R=2 ** 23)):
        assert policy(**kw) == -1, kw
    for kw in (dict(logits=P(4097)), dict(grad=P(4097)), dict(s=P(4100)), dict(dtype=1, grad=P(4098))):
        assert policy(**kw) == -4, kw

    def distill(logits=a, dtype=0, ld=10, R=4, V=10, ids=a, v=a, top=3, rest=1, w=a, T=1.0, loss=a,
                grad=a, ldg=10, s=a):
        return lib.rlu_distill_top(logits, dtype, ld, R, V, ids, v, top, rest, w, T, loss, grad, ldg,
                                   s, P(0))
    assert distill(R=0) == 0
    for kw in (dict(top=0), dict(top=33), dict(rest=2), dict(ids=P(0)), dict(v=P(0)), dict(T=-1.0),
               dict(ldg=9), dict(V=0)):
        assert distill(**kw) == -1, kw

    def scale(x=a, dtype=0, ld=10, R=4, V=10, by=a):
        return lib.rlu_scale_rows(x, dtype, ld, R, V, by, 1, P(0))
    assert scale(R=0) == 0
    for kw in (dict(x=P(0)), dict(by=P(0)), dict(dtype=5), dict(ld=9), dict(V=0), dict(R=-1),
               dict(R=2 ** 23)):
        assert scale(**kw) == -1, kw
    assert scale(x=P(4097)) == -4
