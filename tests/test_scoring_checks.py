"""CPU: what gemm_fp8_dense, token_logprobs and their packers refuse, without a GPU: the Python checks on
tensors that have a shape and a device but no memory, the library's own on its return codes."""
from __future__ import annotations

import ctypes
from importlib import import_module

import pytest

torch = pytest.importorskip("torch")
from torch._subclasses.fake_tensor import FakeTensorMode  # noqa: E402

P = ctypes.c_void_p
F8, BF = torch.float8_e4m3fn, torch.bfloat16


@pytest.fixture
def mods(pkg):
    return import_module(pkg.__name__ + ".ops"), import_module(pkg.__name__ + ".logprobs")


@pytest.fixture
def fake(monkeypatch):
    """Tensors "on the GPU" without one: their data is never touched by a refused call."""
    with FakeTensorMode():
        yield lambda *s, dtype=torch.float32, device="cuda": torch.empty(*s, dtype=dtype,
                                                                        device=device)


@pytest.fixture
def lib(pkg):
    if not pkg.LIB_PATH.exists():
        pytest.skip("librlu.so not built")
    return pkg.lib()


@pytest.mark.parametrize("bad", [
    dict(logits=lambda e: e(4, 100, device="cpu")),
    dict(logits=lambda e: e(4, 100, dtype=torch.float64)),
    dict(logits=lambda e: e(400)),
    dict(logits=lambda e: e(4, 0)),
    dict(logits=lambda e: e(4, 500001)),
    dict(logits=lambda e: e(100, 4).T),                              # a row's logits apart
    dict(logits=lambda e: e(4, 200)[:, ::2]),
    dict(logits=lambda e: e(4, 100).requires_grad_()),
    dict(tokens=lambda e: e(3, dtype=torch.int64)),
    dict(tokens=lambda e: e(4, 1, dtype=torch.int64)),
    dict(tokens=lambda e: e(4)),
    dict(tokens=lambda e: e(8, dtype=torch.int64)[::2]),
    dict(tokens=lambda e: e(4, dtype=torch.int64, device="cpu")),
    dict(top_n=lambda e: -1), dict(top_n=lambda e: 33),
    dict(logits=lambda e: e(4, 5), top_n=lambda e: 6)])
def test_token_logprobs_refuses(mods, fake, bad):
    args = dict(logits=fake(4, 100), tokens=fake(4, dtype=torch.int64), top_n=0)
    args.update({k: v(fake) for k, v in bad.items()})
    with pytest.raises(ValueError):
        mods[1].token_logprobs(**args)


@pytest.mark.parametrize("bad", [
    dict(qx=lambda e: e(4, 256, dtype=F8, device="cpu")),
    dict(qx=lambda e: e(4, 256, dtype=BF)),
    dict(qx=lambda e: e(4, 128, dtype=F8), xs=lambda e: e(4, 1)),     # another depth
    dict(qx=lambda e: e(4, 512, dtype=F8)[:, :256]),                 # rows apart
    dict(qx=lambda e: e(1024, dtype=F8)),
    dict(xs=lambda e: e(4, 1)), dict(xs=lambda e: e(3, 2)),
    dict(xs=lambda e: e(2, 4).T), dict(xs=lambda e: e(4, 2, dtype=BF)),
    dict(xs=lambda e: e(4, 2, device="cpu")), dict(xs=lambda e: e(4, 2).requires_grad_()),
    dict(out=lambda e: e(4, 101, dtype=BF)), dict(out=lambda e: e(4, 100)),
    dict(out=lambda e: e(100, 4, dtype=BF).T), dict(out=lambda e: e(4, 100, dtype=BF).requires_grad_()),
    dict(out=lambda e: e(1, 100, dtype=BF).expand(4, 100)),          # rows on top of each other
    dict(out=lambda e: e(4, 100, dtype=BF, device="cpu"))])
def test_gemm_fp8_dense_refuses(mods, fake, bad):
    w = mods[0].PackedFp8(wq=fake(128, 256, dtype=F8), ws=fake(1, 2), n=100, k=256)
    args = dict(qx=fake(4, 256, dtype=F8), xs=fake(4, 2), w=w, out=None)
    args.update({k: v(fake) for k, v in bad.items()})
    with pytest.raises(ValueError):
        mods[0].gemm_fp8_dense(**args)


@pytest.mark.parametrize("which", ["qx", "wq"])
def test_gemm_fp8_dense_refuses_fp8_operands_that_ask_for_a_gradient(mods, fake, which):
    """A tensor that asks for one still does when it is cast to e4m3."""
    t = dict(qx=fake(4, 256, dtype=F8), wq=fake(128, 256, dtype=F8))
    t[which] = torch.empty(t[which].shape, device="cuda").requires_grad_().to(F8)
    assert t[which].requires_grad
    w = mods[0].PackedFp8(wq=t["wq"], ws=fake(1, 2), n=100, k=256)
    with pytest.raises(ValueError, match="gradient"):
        mods[0].gemm_fp8_dense(t["qx"], fake(4, 2), w)


@pytest.mark.parametrize("w,ws", [((100, 256), (1, 1)), ((129, 256), (1, 2)), ((100, 200), (1, 2)),
                                  ((0, 256), (0, 2)), ((100, 0), (1, 0)), ((100,), (1, 2))])
def test_pack_fp8_dense_refuses(mods, fake, w, ws):
    with pytest.raises(ValueError):
        mods[0].pack_fp8_dense(fake(*w, dtype=F8), fake(*ws))


def test_pack_fp8_dense_refuses_types_and_devices(mods, fake):
    for w, ws in ((fake(100, 256, dtype=BF), fake(1, 2)), (fake(100, 256, dtype=F8), fake(1, 2, dtype=BF)),
                  (fake(100, 256, dtype=F8, device="cpu"), fake(1, 2)),
                  (fake(100, 256, dtype=F8), fake(1, 2, device="cpu"))):
        with pytest.raises(ValueError):
            mods[0].pack_fp8_dense(w, ws)


@pytest.mark.parametrize("bad", [
    dict(wq=lambda e: e(100, 256, dtype=F8)), dict(wq=lambda e: e(128, 512, dtype=F8)),
    dict(wq=lambda e: e(128, 256, dtype=BF)), dict(wq=lambda e: e(256, 128, dtype=F8).T),
    dict(ws=lambda e: e(2, 2)), dict(ws=lambda e: e(1, 2, dtype=BF)), dict(ws=lambda e: e(1, 4)[:, ::2]),
    dict(n=lambda e: 129), dict(n=lambda e: 0), dict(k=lambda e: 200)])
def test_a_packed_weight_fits_its_sizes(mods, fake, bad):
    args = dict(wq=fake(128, 256, dtype=F8), ws=fake(1, 2), n=100, k=256)
    mods[0].PackedFp8(**args)
    args.update({k: v(fake) for k, v in bad.items()})
    with pytest.raises(ValueError):
        mods[0].PackedFp8(**args)


def test_head_logprobs_refuses(mods, fake):
    ops = mods[0]
    head = ops.Fp8TargetHead.__new__(ops.Fp8TargetHead)
    head.wq, head.ws = fake(128, 256, dtype=F8), fake(1, 2)
    x, t = fake(2, 3, 256, dtype=BF), fake(2, 3, dtype=torch.int64)
    for a in ((fake(2, 3, 256), t), (fake(2, 3, 128, dtype=BF), t), (x, fake(6, dtype=torch.int64)),
              (x, fake(2, dtype=torch.int64)), (fake(2, 3, 256, dtype=BF).requires_grad_(), t),
              (fake(2, 3, 256, dtype=BF, device="cpu"), fake(2, 3, dtype=torch.int64, device="cpu"))):
        with pytest.raises(ValueError):
            head.logprobs(*a)


def test_gemm_return_codes(lib):
    p, n = P(4096), P(0)               # (refused before anything is launched or read)
    call = lib.rlu_gemm_fp8blk_dense
    assert call(p, p, p, p, p, 100, 0, 100, 256, n) == 0             # no rows
    assert call(p, p, p, p, p, 100, -1, 100, 256, n) == -1
    assert call(p, p, p, p, p, 100, 4, 0, 256, n) == -1
    assert call(p, p, p, p, p, 99, 4, 100, 256, n) == -1             # rows on top of each other
    assert call(p, p, p, p, p, 100, 4, 100, 0, n) == -1
    assert call(p, p, p, p, p, 100, 4, 100, 200, n) == -2
    assert call(p, p, p, p, p, 2 ** 31 - 1, 4, 2 ** 31 - 1, 256, n) == -1
    for i in range(5):
        assert call(*[n if j == i else p for j in range(5)], 100, 4, 100, 256, n) == -1
    for i, off in enumerate((8, 2, 8, 2, 1)):                        # qx, xs, w, ws, y
        assert call(*[P(4096 + off) if j == i else p for j in range(5)], 100, 4, 100, 256, n) == -4


def test_logprobs_return_codes(lib):
    p, n = P(4096), P(0)
    size = ctypes.c_longlong()
    ws = lib.rlu_token_logprobs_workspace
    b = ctypes.byref(size)
    assert ws(0, 4, 151936, 20, b) == 0 and size.value > 0
    assert ws(0, 0, 151936, 20, b) == 0 and size.value == 0
    for a in ((3, 4, 100, 0), (-1, 4, 100, 0), (0, -1, 100, 0), (0, 4, 0, 0), (0, 4, 500001, 0),
              (0, 4, 100, -1), (0, 4, 100, 33), (0, 4, 5, 6), (0, 2 ** 31 - 1, 151936, 0),
              (0, 2 ** 24, 100, 0)):                                  # past 2^32 threads
        assert ws(*a, b) == -1
    assert ws(0, 4, 100, 0, n) == -1 and ws(0, 2 ** 24 - 1, 100, 0, b) == 0

    def call(x=p, dtype=0, ld=100, rows=4, vocab=100, tok=p, wide=1, top=2, out=(p,) * 5, work=p):
        return lib.rlu_token_logprobs(x, dtype, ld, rows, vocab, tok, wide, top, *out, work, n)
    assert call(rows=0) == 0
    assert call(ld=-1) == -1 and call(wide=2) == -1 and call(top=33) == -1 and call(dtype=3) == -1
    assert call(x=n) == -1 and call(tok=n) == -1 and call(work=n) == -1
    for i in range(5):
        assert call(out=[n if j == i else p for j in range(5)]) == -1
    assert call(x=P(4097)) == -4 and call(x=P(4098), dtype=1) == -4
    assert call(work=P(4100)) == -4


@pytest.mark.parametrize("dtype,elems", [(0, 8), (1, 4), (2, 8)])
def test_a_row_has_at_most_64_segments(lib, dtype, elems):
    """The joining wave has a lane a segment: over every row count's choice, the workspace says how many."""
    size = ctypes.c_longlong()
    for vocab in (1, 7, 2048, 32003, 151936, 262144, 500000):
        for rows in (1, 2, 5, 20, 64, 300, 4096):
            assert lib.rlu_token_logprobs_workspace(dtype, rows, vocab, 0, ctypes.byref(size)) == 0
            segs = size.value // 16 // rows
            assert size.value == 16 * segs * rows and 1 <= segs <= 64
            # wherever in 16 bytes the row starts, the segments hold it
            assert segs * 8 * 256 * elems >= vocab + elems - 1
