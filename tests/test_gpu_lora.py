"""lora.add_lora and lora.add_lora_grad against float64 within derived limits, over types, ranks, sizes, strides and
batches; plan_rows exactly."""
from __future__ import annotations

from importlib import import_module

import pytest

from conftest import gpu_case

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DEV = "cuda"
NAN, INF = float("nan"), float("inf")
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
STEP = 2.0 ** -24


@pytest.fixture(scope="module")
def lora(pkg):
    return import_module(pkg.__name__ + ".lora")


def apart(rows, cols, dtype, g, pad=0, offset=0, std=1.0):
    """[rows, cols] with pad columns of NaN between its rows, from an offset on; and the whole buffer."""
    buf = torch.full((rows * (cols + pad) + offset + 8,), NAN, dtype=dtype, device=DEV)
    t = buf[offset:offset + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    t.copy_(std * torch.randn(rows, cols, generator=g, device=DEV))
    return t, buf


class Case:
    def __init__(self, lora, rows, K, N, R, n, dtype, ids=None, pad=0, offset=0, seed=0, bare=0.2):
        g = torch.Generator(DEV).manual_seed(seed + rows + K + N + R + n)
        dt = TYPES[dtype]
        self.x, _ = apart(rows, K, dt, g, pad, offset)
        self.y, _ = apart(rows, N, dt, g, pad + 1 if pad else 0, offset)
        self.dy, _ = apart(rows, N, dt, g, pad, offset and offset + 1, 2.0 ** -4)
        a = (torch.randn(n, R, K, generator=g, device=DEV) * K ** -0.5).to(dt)
        b = (torch.randn(n, N, R, generator=g, device=DEV) * 0.3).to(dt)
        s = 0.5 + torch.rand(n, generator=g, device=DEV)
        if ids is None:
            ids = torch.randint(n, (rows,), generator=g, device=DEV, dtype=torch.int32)
            ids[torch.rand(rows, generator=g, device=DEV) < bare] = -1
        self.ids = ids
        self.w = lora.LoraStack(a, b, s)
        self.rows = lora.plan_rows(ids, n)
        self.eps = torch.finfo(dt).eps / 2
        self.tiny = torch.finfo(dt).smallest_normal * self.eps
        # h and u go in as two values of the type, the second rounded: half a step of the first's
        self.split = self.eps * self.eps

    def of(self, t):
        """Each row's own adapter's t, in float64; zeros without one."""
        live = (self.ids >= 0) & (self.ids < self.w.n)
        return torch.where(live.view(-1, *[1] * (t.ndim - 1)), t.double()[self.ids.clamp(0, self.w.n - 1).long()],
                           0.0)

    def hidden(self):
        """scale x a^T and how far a sum of float32 products may be from it: each addition by a step of what
        has been added up."""
        xa, s = self.x.double(), self.of(self.w.scale)[:, None]
        A = self.of(self.w.a)
        h = torch.bmm(A, xa[:, :, None])[:, :, 0]
        size = torch.bmm(A.abs(), xa.abs()[:, :, None])[:, :, 0]
        K = xa.shape[1]
        return s * h, s * ((2 * K + 4) * STEP * size)

    def near(self, got, want, limit, what):
        assert got.dtype == self.x.dtype
        limit = limit + self.eps * (want.abs() + limit) + self.tiny
        bad = ~((got.double() - want).abs() <= limit)
        assert not bad.any(), (what, got[bad][:4], want[bad][:4], limit[bad][:4], bad.sum(), bad.nonzero()[:4])

    def check_out(self, out):
        h, e = self.hidden()
        B = self.of(self.w.b)
        R = h.shape[1]
        by = lambda t: torch.bmm(B.abs(), t.abs()[:, :, None])[:, :, 0]                # noqa: E731
        want = self.y.double() + torch.bmm(B, h[:, :, None])[:, :, 0]
        # f16: a row's h are scaled so that none is below 2^-34 of the largest's step
        limit = by(e) + (self.split + 4 * (R + 1) * STEP) * by(h) + 2 * STEP * self.y.double().abs()
        limit = limit + B.abs().sum(2) * h.abs().amax(1, keepdim=True) * 2.0 ** -34
        self.near(out, want, limit, "out")
        bare = self.ids < 0
        assert torch.equal(out[bare], self.y[bare])


    def check_grad(self, dx, da, db, hidden=None):
        """Against the float64 formulas; a gradient over an adapter's rows adds up those rows."""
        d, x = self.dy.double(), self.x.double()
        A, B = self.of(self.w.a), self.of(self.w.b)
        s = self.of(self.w.scale)[:, None]
        N, R = B.shape[1:]
        h, he = self.hidden()
        u = s * torch.bmm(d[:, None, :], B)[:, 0]
        ue = s * torch.bmm(d.abs()[:, None, :], B.abs())[:, 0] * (2 * N + 8) * STEP
        # a value in two parts: split; float16's tiles are scaled to their largest, 2^-34 of which is the last step
        part = lambda t: self.split * t.abs() + t.abs().amax() * 2.0 ** -34          # noqa: E731
        up, hp = part(u) + ue, part(h) + he
        if dx is not None:
            want = torch.bmm(u[:, None, :], A)[:, 0]
            size = torch.bmm(u.abs()[:, None, :], A.abs())[:, 0]
            self.near(dx, want, torch.bmm(up[:, None, :], A.abs())[:, 0] + 4 * (R + 1) * STEP * size, "dx")
            assert (dx[self.ids < 0] == 0).all()
        for got, v, by, by_err, what in ((da, x, u, up, "da"), (db, d, h, hp, "db")):
            if got is None:
                continue
            for i in range(self.w.n):
                at = self.ids == i
                want, size = by[at].T @ v[at], by[at].abs().T @ v[at].abs()
                limit = by_err[at].T @ v[at].abs() + 4 * (int(at.sum()) + 8) * STEP * size
                if what == "db":
                    want, limit = want.T, limit.T
                self.near(got[i], want, limit, f"{what}[{i}]")


SIZES = [  # rows, K, N, R, n
    (1, 2560, 2560, 16, 1), (1, 1, 1, 1, 1), (2, 7, 5, 3, 2), (5, 33, 31, 8, 3), (16, 128, 512, 16, 1),
    (17, 100, 513, 17, 40), (63, 768, 1543, 8, 12), (64, 256, 100, 24, 2), (100, 31, 33, 33, 5),
    (200, 512, 640, 64, 64), (300, 129, 257, 100, 7), (129, 264, 1030, 128, 3), (1023, 136, 72, 16, 1000),
    (600, 136, 700, 16, 300), (500, 72, 1030, 40, 400), (40, 200, 150000, 24, 3),
    (1024, 136, 72, 16, 1024), (1100, 65, 515, 32, 9), (2050, 128, 130, 128, 1), (3000, 40, 48, 65, 30)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,K,N,R,n", SIZES)
@pytest.mark.parametrize("pad,offset", [(0, 0), (3, 5)])
def test_values(lora, dtype, rows, K, N, R, n, pad, offset):
    c = Case(lora, rows, K, N, R, n, dtype, pad=pad, offset=offset)
    gpu_case(f"lora {dtype} rows={rows} K={K} N={N} R={R} n={n} pad={pad}")
    hidden = torch.full((rows, R), NAN, device=DEV)
    out = lora.add_lora(c.y, c.x, c.w, c.rows, hidden=hidden)
    torch.cuda.synchronize()
    c.check_out(out)
    h, e = c.hidden()
    assert ((hidden.double() - h).abs() <= e + 4 * STEP * h.abs()).all()
    assert (hidden[c.ids < 0] == 0).all()


@pytest.mark.parametrize("ids64", [False, True])
@pytest.mark.parametrize("rows,n", [(1, 1), (5, 1), (16, 3), (50, 70), (1000, 1024), (1024, 5), (4097, 1024),
                                    (20000, 64)])
def test_plan(lora, rows, n, ids64):
    """The rows of each adapter in order, in tiles of one adapter each, then those without and those past the last."""
    for kind in ("any", "runs", "one", "none", "bad"):
        g = torch.Generator(DEV).manual_seed(rows + n)
        ids = torch.randint(-1, n + 1, (rows,), generator=g, device=DEV)
        if kind == "runs":
            ids = ids.sort(descending=True).values
        elif kind != "any":
            ids.fill_({"one": n - 1, "none": -7, "bad": n + 5}[kind])
        if kind == "any" and ids64:
            ids[0], ids[-1] = 2 ** 40, -2 ** 40
        ids = ids if ids64 else ids.int()
        gpu_case(f"lora plan rows={rows} n={n} {kind}")
        p = lora.plan_rows(ids, n)
        torch.cuda.synchronize()
        key = torch.where(ids < 0, n, torch.where(ids >= n, n + 1, ids)).cpu()
        order = key.sort(stable=True).indices
        assert torch.equal(p.order.cpu().long(), order)
        count = torch.bincount(key, minlength=n + 2)
        tiles = (count + p.size - 1) // p.size
        first = torch.cat([torch.zeros(1, dtype=tiles.dtype), tiles.cumsum(0)])
        live = (count[:n] > 0).sum().view(1)
        assert torch.equal(p.first.cpu().long(), torch.cat([first, live, count[:n].sum().view(1)])) and first[-1] <= p.tiles.shape[0]
        start, want = 0, []
        for k in range(n + 2):
            for at in range(0, int(count[k]), p.size):
                want.append([k if k < n else n - 1 - k, start + at, min(p.size, int(count[k]) - at), 0])
            start += int(count[k])
        assert p.tiles[:len(want)].tolist() == want


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [40, 1500])
def test_ids_past_the_last(lora, dtype, rows):
    ids = torch.arange(rows, device=DEV) % 5 - 1                     # -1 .. 3 of a stack of 3
    c = Case(lora, rows, 72, 100, 8, 3, dtype, ids=ids)
    gpu_case(f"lora ids past the last {dtype}")
    out = lora.add_lora(c.y, c.x, c.w, c.rows)
    torch.cuda.synchronize()
    bad = ids == 3
    assert out[bad].isnan().all()
    out[bad] = c.y[bad]
    c.check_out(out)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [50, 1200])
def test_in_place_and_into_a_buffer(lora, dtype, rows):
    """Only the outputs' own elements are written; rows without an adapter stay in place."""
    c = Case(lora, rows, 136, 517, 16, 4, dtype, pad=3, offset=1)
    gpu_case(f"lora out= {dtype} rows={rows}")
    want = lora.add_lora(c.y, c.x, c.w, c.rows)
    for pad, off in ((0, 0), (1, 3), (8, 8)):
        g = torch.Generator(DEV).manual_seed(1)
        out, buf = apart(rows, 517, c.y.dtype, g, pad, off)
        own = torch.zeros_like(buf, dtype=torch.bool)
        own[off:off + rows * (517 + pad)].view(rows, -1)[:, :517] = True
        buf.fill_(3.0)
        assert lora.add_lora(c.y, c.x, c.w, c.rows, out=out) is out
        torch.cuda.synchronize()
        assert torch.equal(out, want) and (buf[~own] == 3.0).all()
        out.copy_(c.y)
        lora.add_lora(out, c.x, c.w, c.rows, out=out)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and (buf[~own] == 3.0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_large_and_small_values(lora, dtype):
    """Hidden values past float16's range and below its smallest, where the output is in range; bf16's likewise."""
    big = 300.0 if dtype == "f16" else 1e12
    c = Case(lora, 33, 512, 96, 16, 2, dtype, bare=0.0)
    c.x.mul_(big)
    c.w.a.mul_(big)                                                  # h near 1e5, and 1e24
    c.w.b.mul_(1e-3 if dtype == "f16" else 1e-20)
    gpu_case(f"lora large {dtype}")
    out = lora.add_lora(c.y, c.x, c.w, c.rows)
    torch.cuda.synchronize()
    assert torch.isfinite(out).all()
    c.check_out(out)
    c.x.mul_(1e-3 / big)
    c.w.a.mul_(1e-2 / big)
    c.w.b.mul_(1e3 if dtype == "f16" else 1e20)
    c.y.mul_(1e-4)
    out = lora.add_lora(c.y, c.x, c.w, c.rows)
    torch.cuda.synchronize()
    c.check_out(out)


def test_nan_and_inf_stay_in_their_rows(lora):
    c = Case(lora, 70, 100, 90, 16, 3, "bf16", bare=0.0)
    want = lora.add_lora(c.y, c.x, c.w, c.rows)
    c.x[3, 7], c.x[60, 99], c.y[5, 1] = NAN, INF, NAN
    gpu_case("lora NaN")
    out = lora.add_lora(c.y, c.x, c.w, c.rows)
    torch.cuda.synchronize()
    assert out[3].isnan().all() and not torch.isfinite(out[60]).any()
    assert out[5, 1].isnan()
    keep = [r for r in range(70) if r not in (3, 5, 60)]
    assert torch.equal(out[keep], want[keep])


def test_no_rows(lora):
    w = lora.LoraStack(torch.zeros(2, 8, 16, dtype=torch.bfloat16, device=DEV),
                       torch.zeros(2, 24, 8, dtype=torch.bfloat16, device=DEV), torch.ones(2, device=DEV))
    rows = lora.plan_rows(torch.empty(0, dtype=torch.int32, device=DEV), 2)
    x = torch.empty(0, 16, dtype=torch.bfloat16, device=DEV)
    y = torch.empty(0, 24, dtype=torch.bfloat16, device=DEV)
    assert lora.add_lora(y, x, w, rows).shape == (0, 24)
    assert lora.add_lora(y, x, w, rows, out=y) is y


def test_outputs_past_2_to_31_elements(lora):
    rows, N = 14200, 151936                                          # 2.16e9 of them, 4.3 GB
    ids = torch.zeros(rows, dtype=torch.int32, device=DEV)
    ids[100:-40] = -1
    g = torch.Generator(DEV).manual_seed(1)
    x = torch.randn(rows, 32, generator=g, device=DEV).bfloat16()
    y = torch.zeros(rows, N, dtype=torch.bfloat16, device=DEV)
    w = lora.LoraStack(torch.randn(1, 8, 32, generator=g, device=DEV).bfloat16(),
                       torch.randn(1, N, 8, generator=g, device=DEV).bfloat16(), torch.ones(1, device=DEV))
    gpu_case("lora past 2^31 elements")
    lora.add_lora(y, x, w, lora.plan_rows(ids, 1), out=y)
    torch.cuda.synchronize()
    at = torch.cat([torch.arange(100), torch.arange(rows - 40, rows)]).to(DEV)
    few = lora.add_lora(torch.zeros(140, N, dtype=torch.bfloat16, device=DEV), x[at], w,
                        lora.plan_rows(torch.zeros(140, dtype=torch.int32, device=DEV), 1))
    torch.cuda.synchronize()
    # (two ways of tiling the same rows: sums of 32 and of 8 products in other orders, rounded once)
    torch.testing.assert_close(y[at], few, rtol=2.0 ** -7, atol=1e-4)
    assert (y[100:200] == 0).all() and (y[-200:-40] == 0).all()


def test_streams_bit_for_bit(lora):
    for rows in (60, 1300):
        c = Case(lora, rows, 264, 1030, 16, 9, "bf16")
        gpu_case(f"lora on three streams at once rows={rows}")
        torch.cuda.synchronize()
        got = []
        for st in [torch.cuda.Stream() for _ in range(3)]:
            with torch.cuda.stream(st):
                got += [lora.add_lora(c.y, c.x, c.w, lora.plan_rows(c.ids, 9)) for _ in range(3)]
        torch.cuda.synchronize()
        for t in got[1:]:
            assert torch.equal(got[0], t)


@pytest.mark.parametrize("rows", [60, 1300])
def test_graphs_replayed_with_new_rows(lora, rows):
    """The plan and two projections in a graph, in place; two graphs at once; eager calls between."""
    cases = [Case(lora, rows, 264, 130, 16, 9, "bf16", seed=s) for s in range(3)]
    w = cases[0].w
    ins = [(cases[0].ids.clone(), cases[0].x.clone(), cases[0].y.clone()) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []

    def step(ids, x, y):
        p = lora.plan_rows(ids, 9)
        first = lora.add_lora(y, x, w, p)
        second = lora.add_lora(y, x, w, p)
        return first, lora.add_lora(second, x, w, p, out=second)
    gpu_case(f"lora graphs rows={rows}")
    torch.cuda.synchronize()
    for args, st in zip(ins, streams):
        with torch.cuda.stream(st):
            step(*args)
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(step(*args))
        graphs.append(g)
    for i in (1, 2, 0, 1):
        for j, st in enumerate(streams):
            c = cases[(i + j) % 3]
            with torch.cuda.stream(st):
                for t, s in zip(ins[j], (c.ids, c.x, c.y)):
                    t.copy_(s)
                graphs[j].replay()
        lora.add_lora(cases[i].y, cases[i].x, w, cases[i].rows)
        torch.cuda.synchronize()
        for j in range(2):
            c = cases[(i + j) % 3]
            want = step(c.ids, c.x, c.y)
            torch.cuda.synchronize()
            assert torch.equal(outs[j][0], want[0]) and torch.equal(outs[j][1], want[1])


# ---- the backward pass --------------------------------------------------------------------------
def both(lora, c, need=(True, True, True)):
    hidden = torch.full((c.x.shape[0], c.w.rank), NAN, device=DEV)
    lora.add_lora(c.y, c.x, c.w, c.rows, hidden=hidden)
    return lora.add_lora_grad(c.dy, c.x, c.w, c.rows, hidden, need)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,K,N,R,n", SIZES)
@pytest.mark.parametrize("pad,offset", [(0, 0), (3, 5)])
def test_gradients(lora, dtype, rows, K, N, R, n, pad, offset):
    c = Case(lora, rows, K, N, R, n, dtype, pad=pad, offset=offset)
    gpu_case(f"lora grad {dtype} rows={rows} K={K} N={N} R={R} n={n} pad={pad}")
    got = both(lora, c)
    torch.cuda.synchronize()
    c.check_grad(*got)


@pytest.mark.parametrize("rows,n,ids", [
    (2000, 3, "one"), (2000, 70, "few"), (64, 64, "each"), (300, 64, "each"), (1500, 2, "none"), (90, 5, "runs"), (5000, 6, "runs"), (700, 1024, "few"),
    (129, 2, "one")])
def test_gradients_of_uneven_batches(lora, rows, n, ids):
    """One adapter with every row, over many runs of tiles; most without any; no row with one; ids in runs."""
    g = torch.Generator(DEV).manual_seed(rows)
    of = {"one": torch.full((rows,), n - 1, device=DEV), "none": torch.full((rows,), -1, device=DEV),
          "each": torch.arange(rows, device=DEV) % n, "few": torch.randint(3, (rows,), generator=g, device=DEV) * (n // 3),
          "runs": torch.randint(-1, n, (rows,), generator=g, device=DEV).sort().values}[ids].int()
    for K, N, R in ((200, 264, 16), (72, 40, 40)):
        c = Case(lora, rows, K, N, R, n, "bf16", ids=of)
        gpu_case(f"lora grad rows={rows} n={n} {ids} K={K}")
        got = both(lora, c)
        torch.cuda.synchronize()
        c.check_grad(*got)
        empty = [i for i in range(n) if not (of == i).any()]
        assert (got[1][empty] == 0).all() and (got[2][empty] == 0).all()


@pytest.mark.parametrize("counts", [
    [10, 600, 200, 1, 0, 7], [0, 256, 257, 16, 17, 300], [10, 900, 250, 1, 0, 300, 256, 257, 64, 65], [1200, 0, 1, 700, 192, 193]])
def test_gradients_of_small_beside_large_adapters(lora, counts):
    """Adapters on both sides of the rows that one workgroup takes alone, in any order of the rows."""
    ids = torch.cat([torch.full((c,), i) for i, c in enumerate(counts)] + [torch.full((9,), -1)]).int()
    ids = ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(len(ids)))].to(DEV)
    c = Case(lora, len(ids), 264, 200, 24, len(counts), "bf16", ids=ids)
    gpu_case(f"lora grad rows of {counts}")
    got = both(lora, c)
    torch.cuda.synchronize()
    c.check_grad(*got)


@pytest.mark.parametrize("rows,K,N,R", [(96, 2560, 2560, 16), (40, 136, 50000, 16), (1030, 512, 20000, 64)])
def test_gradients_of_long_products(lora, rows, K, N, R):
    c = Case(lora, rows, K, N, R, 2, "bf16")
    gpu_case(f"lora grad long rows={rows} K={K} N={N}")
    got = both(lora, c)
    torch.cuda.synchronize()
    c.check_grad(*got)


def test_gradients_asked_for_one_by_one(lora):
    for rows in (70, 1100):
        c = Case(lora, rows, 136, 200, 16, 3, "f16")
        gpu_case(f"lora grad need rows={rows}")
        want = both(lora, c)
        for need in ((True, False, False), (False, True, False), (False, False, True), (False, True, True),
                     (False, False, False)):
            got = both(lora, c, need)
            torch.cuda.synchronize()
            for t, u, n in zip(got, want, need):
                assert torch.equal(t, u) if n else t is None


@pytest.mark.parametrize("R", [65, 128])
@pytest.mark.parametrize("rows,n", [(70, 40), (1100, 3)])
def test_gradients_of_high_ranks_one_by_one(lora, rows, n, R):
    """Over 64 ranks, where dx has a launch of its own."""
    c = Case(lora, rows, 264, 520, R, n, "bf16")
    gpu_case(f"lora grad need rows={rows} R={R}")
    want = both(lora, c)
    torch.cuda.synchronize()
    c.check_grad(*want)
    for need in ((True, False, False), (False, True, False), (False, False, True)):
        got = both(lora, c, need)
        torch.cuda.synchronize()
        for t, u, n in zip(got, want, need):
            assert torch.equal(t, u) if n else t is None


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,K,N,R", [(30, 256, 320, 16), (1100, 129, 65, 40), (1100, 128, 264, 8)])
def test_factors_at_any_address(lora, dtype, rows, K, N, R):
    """Adapters, their scale and hidden one element behind an aligned address: the same bits."""
    c = Case(lora, rows, K, N, R, 3, dtype)
    off = lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)     # noqa: E731
    w = lora.LoraStack(off(c.w.a), off(c.w.b), off(c.w.scale))
    assert w.a.data_ptr() % 16 and w.b.data_ptr() % 16 and w.scale.data_ptr() % 16
    h, g = torch.empty(rows, R, device=DEV), off(torch.full((rows, R), NAN, device=DEV))
    gpu_case(f"lora {dtype} factors at odd addresses rows={rows}")
    want = lora.add_lora(c.y, c.x, c.w, c.rows, hidden=h)
    got = lora.add_lora(c.y, c.x, w, c.rows, hidden=g)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(g, h)
    for t, u in zip(lora.add_lora_grad(c.dy, c.x, w, c.rows, g), lora.add_lora_grad(c.dy, c.x, c.w, c.rows, h)):
        assert torch.equal(t, u)


@pytest.mark.parametrize("rows", [45, 1300])
def test_gradients_of_ids_past_the_last_and_nan(lora, rows):
    """A bad row has no part in the adapters' gradients; a NaN in a row goes to that row and to its adapter alone;
    rows without an adapter have 0, whatever adapter 0 holds."""
    ids = (torch.arange(rows, device=DEV) % 5 - 1).int()             # -1 .. 3 of a stack of 3
    c = Case(lora, rows, 72, 100, 8, 3, "bf16", ids=ids)
    gpu_case("lora grad ids past the last")
    dx, da, db = both(lora, c)
    bad = ids == 3
    torch.cuda.synchronize()
    assert dx[bad].isnan().all()
    dx[bad] = 0
    c.check_grad(dx, da, db)
    c.x[1, 3] = NAN                                                  # (adapter 0's row)
    c.w.a[0, 2, 5] = INF
    got = both(lora, c)
    torch.cuda.synchronize()
    assert (got[0][ids < 0] == 0).all() and got[1][0, :, 3].isnan().all()
    keep = [r for r in range(rows) if ids[r] in (1, 2)]
    assert torch.equal(got[0][keep], dx[keep])
    assert torch.equal(got[1][1:], da[1:]) and torch.equal(got[2][1:], db[1:])


@pytest.mark.parametrize("dtype", TYPES)
def test_large_and_small_gradients(lora, dtype):
    """u past float16's range and below its smallest; bf16's likewise."""
    for big in ((2.0 ** 11, 2.0 ** -12) if dtype == "f16" else (2.0 ** 60, 2.0 ** -60)):
        c = Case(lora, 100, 136, 96, 16, 2, dtype, bare=0.0)
        c.w.b.mul_(big)
        c.w.a.mul_(1 / big)
        c.dy.mul_(16.0 if big > 1 else 0.25)
        c.x.mul_(2.0 ** -8 if big > 1 else 4.0)
        gpu_case(f"lora grad scale {big} {dtype}")
        got = both(lora, c)
        torch.cuda.synchronize()
        assert all(torch.isfinite(t).all() for t in got)
        c.check_grad(*got)


def test_gradients_against_differences(lora):
    """Of L = sum dy (y + h B^T) along random directions, with operands that are exact in bf16 before and after a step.
    L is linear in x, in a and in b alone, so its central difference has no error but the outputs' roundings."""
    g = torch.Generator(DEV).manual_seed(1)
    c = Case(lora, 40, 64, 48, 8, 3, "bf16")
    for t in (c.x, c.w.a, c.w.b, c.dy, c.y):
        t.copy_((torch.randint(-8, 9, t.shape, generator=g, device=DEV)) / 8)
    dx, da, db = both(lora, c)
    gpu_case("lora against differences")

    def loss():
        # in float32, whose hidden part is exact enough: the output's rounding is what a difference would see
        h = torch.empty(40, 8, device=DEV)
        lora.add_lora(c.y, c.x, c.w, c.rows, hidden=h)
        return (c.dy.double() * torch.bmm(c.of(c.w.b), h.double()[:, :, None])[:, :, 0]).sum()
    for t, grad in ((c.x, dx), (c.w.a, da)):
        for _ in range(3):
            step = torch.randint(-1, 2, t.shape, generator=g, device=DEV).to(t.dtype)
            keep = t.clone()
            t.copy_(keep + step)
            up = loss()
            t.copy_(keep - step)
            by = (up - loss()) / 2
            t.copy_(keep)
            got = (grad.double() * step.double()).sum()
            size = (grad.double().abs() * step.double().abs()).sum()
            assert (by - got).abs() <= (c.eps + 600 * STEP) * size + 600 * STEP * up.abs(), (by, got)
    # and in b, whose product the output adds up: hidden stays, the difference is the gradient's own sum
    h = torch.empty(40, 8, device=DEV)
    lora.add_lora(c.y, c.x, c.w, c.rows, hidden=h)
    step = torch.randint(-1, 2, c.w.b.shape, generator=g, device=DEV).double()
    by = (c.dy.double() * torch.bmm(c.of(step), h.double()[:, :, None])[:, :, 0]).sum()
    size = (db.double().abs() * step.abs()).sum()
    assert (by - (db.double() * step).sum()).abs() <= (c.eps + 600 * STEP) * size


def test_autograd_notices_an_output_that_was_written_over(lora):
    c = Case(lora, 20, 64, 72, 8, 2, "bf16")
    leaf = c.y.detach().clone().requires_grad_()
    for out in (None, "y"):
        y = torch.sigmoid(leaf)                                      # (whose backward pass asks for y)
        gpu_case(f"lora into {out} beside autograd")
        with torch.no_grad():
            lora.add_lora(y, c.x, c.w, c.rows, out=out and y)
        if out:
            with pytest.raises(RuntimeError, match="inplace"):
                y.sum().backward()
        else:
            y.sum().backward()
    torch.cuda.synchronize()


def test_autograd_refuses_operands_written_to(lora):
    for which in ("a", "b", "scale"):
        c = Case(lora, 20, 64, 72, 8, 2, "bf16")
        a, b, scale = c.w.a.clone().requires_grad_(), c.w.b.clone(), c.w.scale.clone()
        w = lora.LoraStack(a, b, scale)
        gpu_case(f"lora autograd, {which} written to")
        out = lora.add_lora(c.y, c.x, w, c.rows)
        with torch.no_grad():
            getattr(w, which).mul_(2)
        with pytest.raises(RuntimeError, match="inplace"):
            out.sum().backward()
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [30, 1100])
def test_autograd(lora, dtype, rows):
    c = Case(lora, rows, 72, 130, 16, 3, dtype, pad=2, offset=1)
    want = both(lora, c)
    y, x, a, b = (t.detach().requires_grad_() for t in (c.y, c.x, c.w.a, c.w.b))
    w = lora.LoraStack(a, b, c.w.scale)
    gpu_case(f"lora autograd {dtype} rows={rows}")
    out = lora.add_lora(y, x, w, c.rows)
    assert torch.equal(out, lora.add_lora(c.y, c.x, c.w, c.rows))
    got = torch.autograd.grad(out, (y, x, a, b), c.dy, retain_graph=True)
    for t, u in zip(got, (c.dy, *want)):
        assert torch.equal(t, u)
    again = torch.autograd.grad(out, (x, b), c.dy)
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[2])
    (lora.add_lora(c.y, c.x, w, c.rows).sum() * 2.0).backward()       # (an expanded gradient)
    c.dy = torch.full_like(c.dy, 2.0)
    for t, u in zip((a.grad, b.grad), both(lora, c)[1:]):
        assert torch.equal(t, u)
    out = lora.add_lora(y, x, w, c.rows)
    with torch.no_grad():
        a.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.backward(c.dy)


def test_gradients_on_streams_and_in_graphs(lora):
    for rows in (60, 1300):
        c = Case(lora, rows, 264, 530, 16, 9, "bf16")
        gpu_case(f"lora grad on three streams at once rows={rows}")
        torch.cuda.synchronize()
        got = []
        for st in [torch.cuda.Stream() for _ in range(3)]:
            with torch.cuda.stream(st):
                got += [both(lora, c) for _ in range(3)]
        torch.cuda.synchronize()
        for t in got[1:]:
            assert all(torch.equal(a, b) for a, b in zip(got[0], t))
        others = Case(lora, rows, 264, 530, 16, 9, "bf16", seed=7)
        others.w = c.w
        ids, x, dy = c.ids.clone(), c.x.clone(), c.dy.clone()
        graph = torch.cuda.CUDAGraph()
        leaf = lora.LoraStack(c.w.a.detach().requires_grad_(), c.w.b, c.w.scale)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            p = lora.plan_rows(ids, 9)
            hidden = torch.empty(rows, 16, device=DEV)
            lora.add_lora(c.y, x, c.w, p, hidden=hidden)
            outs = lora.add_lora_grad(dy, x, c.w, p, hidden)
            with pytest.raises(ValueError, match="add_lora_grad"):
                lora.add_lora(c.y, x, leaf, p)
        for case in (others, c, others, c):
            for t, s in zip((ids, x, dy), (case.ids, case.x, case.dy)):
                t.copy_(s)
            graph.replay()
            want = both(lora, case)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_no_rows_have_zero_gradients(lora):
    w = lora.LoraStack(torch.ones(2, 8, 16, dtype=torch.bfloat16, device=DEV),
                       torch.ones(2, 24, 8, dtype=torch.bfloat16, device=DEV), torch.ones(2, device=DEV))
    rows = lora.plan_rows(torch.empty(0, dtype=torch.int64, device=DEV), 2)
    e = lambda n: torch.empty(0, n, dtype=torch.bfloat16, device=DEV)                  # noqa: E731
    dx, da, db = lora.add_lora_grad(e(24), e(16), w, rows, torch.empty(0, 8, device=DEV))
    assert dx.shape == (0, 16) and (da == 0).all() and (db == 0).all()
