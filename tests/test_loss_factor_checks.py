"""CPU: what the losses' gradients with a factor refuse, by the library's return codes."""
from __future__ import annotations

import ctypes

import pytest

P = ctypes.c_void_p


@pytest.fixture
def lib(pkg):
    if not pkg.LIB_PATH.exists():
        pytest.skip("librlu.so not built")
    return pkg.lib()


def test_return_codes(lib):
    a = P(4096)
    nan, inf = float("nan"), float("inf")

    def policy(logits=a, dtype=0, ld=10, R=4, V=10, tokens=a, wide=1, old=a, adv=a, ref=a, w=a, lo=0.2, hi=0.2, kl=0.1,
               T=1.0, by=a, step=1, grad=a, ldg=10, s=a):
        return lib.rlu_policy_grad_by(logits, dtype, ld, R, V, tokens, wide, old, adv, ref, w, lo, hi, kl, T, by, step, grad,
                                      ldg, s, P(0))
    assert policy(R=0) == 0
    for kw in (dict(dtype=1), dict(dtype=3), dict(ld=-1), dict(R=-1), dict(V=0), dict(V=500001), dict(wide=2), dict(lo=1.5),
               dict(hi=nan), dict(kl=inf), dict(T=0.0), dict(logits=P(0)), dict(tokens=P(0)), dict(old=P(0)), dict(adv=P(0)),
               dict(by=P(0)), dict(grad=P(0)), dict(s=P(0)), dict(ldg=9), dict(R=2 ** 23)):
        assert policy(**kw) == -1, kw
    for kw in (dict(logits=P(4097)), dict(grad=P(4097)), dict(s=P(4100))):
        assert policy(**kw) == -4, kw

    def distill(logits=a, dtype=2, ld=10, R=4, V=10, ids=a, v=a, top=3, rest=1, w=a, T=1.0, by=a, step=0, grad=a, ldg=10, s=a):
        return lib.rlu_distill_top_grad_by(logits, dtype, ld, R, V, ids, v, top, rest, w, T, by, step, grad, ldg, s, P(0))
    assert distill(R=0) == 0
    for kw in (dict(dtype=1), dict(top=0), dict(top=33), dict(rest=2), dict(ids=P(0)), dict(v=P(0)), dict(T=-1.0), dict(ldg=9),
               dict(V=0), dict(by=P(0)), dict(grad=P(0)), dict(s=P(0))):
        assert distill(**kw) == -1, kw
    for kw in (dict(logits=P(4097)), dict(grad=P(4097)), dict(s=P(4100))):
        assert distill(**kw) == -4, kw
