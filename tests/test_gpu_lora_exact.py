"""The adapters' products on whole numbers: every product and every sum of them, in whatever order, has fewer than 24 bits,
so float32 holds each of them as it is and the outputs are the exact results, rounded once. h and u have 18 bits."""
from __future__ import annotations

from importlib import import_module

import pytest

from conftest import gpu_case

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
# a few of float16's bits less, whose largest value is 65504
TOP = {"bf16": 2.0 ** 10, "f16": 2.0 ** 3}


@pytest.fixture(scope="module")
def lora(pkg):
    return import_module(pkg.__name__ + ".lora")


SIZES = [  # rows, K, N, R, n: at most 30 rows an adapter
    (1, 24, 600, 16, 1), (20, 40, 64, 8, 1), (30, 33, 35, 3, 2), (100, 64, 256, 16, 5), (100, 72, 1031, 64, 7), (90, 48, 130, 100, 4),
    (600, 40, 2100, 24, 30), (1100, 64, 520, 16, 60), (1100, 65, 130, 40, 50), (1200, 72, 72, 128, 64)]


def whole(g, most, *shape, some=1.0):
    """Whole numbers from -most to most; `some` of them, the others 0."""
    t = torch.randint(-most, most + 1, shape, generator=g, device=DEV).double()
    return t * (torch.rand(shape, generator=g, device=DEV) < some)


def large(g, top, rows):
    """Eight bits, the lowest of which is top."""
    sign = torch.randint(2, (rows,), generator=g, device=DEV) * 2 - 1
    return sign * torch.randint(128, 256, (rows,), generator=g, device=DEV) * top


def inputs(rows, K, N, R, n, dtype, wide):
    """wide "h": x's first element is large and meets a 1 in every rank, the others are small; "u": so is dy's. What the
    wide value is multiplied with has 24 elements other than 0 on average at most, and is -1, 0 or 1; its large part leaves
    the outputs again, so that their own rounding hides none of its last bits: y is out's negative, rounded, and rows or
    ranks come in pairs of which one takes back the other's."""
    g = torch.Generator(DEV).manual_seed(rows + K + N + R)
    some = min(1.0, 24 / R)
    ids = torch.arange(rows, device=DEV) % n
    ids[3::17] = -1
    t = TYPES[dtype]
    second = torch.arange(rows, device=DEV) // n % 2 == 1            # (of two rows of one adapter)
    first = (torch.arange(rows, device=DEV) - n)[second]
    y = whole(g, 100, rows, N)
    if wide == "h":
        x, a = whole(g, 31, rows, K), whole(g, 7, n, R, K)
        x[:, 0], a[:, :, 0] = large(g, TOP[dtype], rows), 1
        b, dy = whole(g, 1, n, N, R, some=some), whole(g, 1, rows, N)
        x[second, 0], dy[second] = -x[first, 0], dy[first]
        for i in range(n):
            y[ids == i] = -((x[ids == i] @ a[i].T) @ b[i].T).to(t).double()
    else:
        dy, b = whole(g, 31, rows, N), whole(g, 7, n, N, R)
        dy[:, 0], b[:, 0] = large(g, TOP[dtype], rows), 1
        a, x = whole(g, 1, n, R, K, some=some), whole(g, 1, rows, K)
        dy[second, 0], x[second] = -dy[first, 0], x[first]
        a[:, 1::2] = -a[:, 0:R - 1:2]
        a[:, R - R % 2:] = 0
    return ids, x, y, dy, a, b


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,K,N,R,n", SIZES)
@pytest.mark.parametrize("wide", ["h", "u"])
def test_whole_numbers(lora, dtype, rows, K, N, R, n, wide):
    ids, x, y, dy, a, b = inputs(rows, K, N, R, n, dtype, wide)
    t = TYPES[dtype]
    w = lora.LoraStack(a.to(t), b.to(t), torch.ones(n, device=DEV))
    p = lora.plan_rows(ids, n)
    hidden = torch.empty(rows, R, device=DEV)
    gpu_case(f"lora whole numbers {dtype} rows={rows} K={K} N={N} R={R} n={n} {wide}")
    out = lora.add_lora(y.to(t), x.to(t), w, p, hidden=hidden)
    dx, da, db = lora.add_lora_grad(dy.to(t), x.to(t), w, p, hidden)
    torch.cuda.synchronize()

    def same(got, want, size, what):
        assert size.max() < 2 ** 24, (what, size.max())
        assert torch.equal(got, want.to(t)), (what, (got != want.to(t)).sum(), got.numel())
    for i in range(n):
        at = (ids == i).nonzero()[:, 0]
        h, u = x[at] @ a[i].T, dy[at] @ b[i]
        assert torch.equal(hidden[at].double(), h)
        if wide == "h":
            assert h.abs().max() >= 2 ** 17 or dtype == "f16"
            same(out[at], y[at] + h @ b[i].T, y[at].abs() + h.abs() @ b[i].abs().T, "out")
            same(db[i], dy[at].T @ h, dy[at].abs().T @ h.abs(), "db")
        else:
            assert u.abs().max() >= 2 ** 17 or dtype == "f16"
            same(dx[at], u @ a[i], u.abs() @ a[i].abs(), "dx")
            same(da[i], u.T @ x[at], u.abs().T @ x[at].abs(), "da")
