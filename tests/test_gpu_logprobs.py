"""logprobs.token_logprobs against float64: ranks and ids exactly, values within derived limits; and the
head's scoring as a whole."""
from __future__ import annotations

from importlib import import_module

import pytest

from conftest import gpu_case

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DEV = "cuda"
NINF, INF, NAN = float("-inf"), float("inf"), float("nan")
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@pytest.fixture(scope="module")
def mods(pkg):
    return import_module(pkg.__name__ + ".logprobs"), import_module(pkg.__name__ + ".ops")


@pytest.fixture(scope="module")
def score(mods):
    return mods[0].token_logprobs


def exact(x, tokens, top):
    """In float64, by a stable sort, for rows of finite and -inf logits and tokens in range. Also rest, the
    sum of e^(x - max) without the maximum's own term."""
    x = x.double()
    s, at = torch.sort(x, dim=1, descending=True, stable=True)
    m = s[:, :1]
    none = m == NINF
    d = s - torch.where(none, 0.0, m)
    e = torch.exp(d)
    rest = torch.where(none[:, 0], 0.0, e[:, 1:].sum(1))
    lz = torch.log1p(rest)
    t = torch.where(e > 0, d * e, 0.0).sum(1) / (1 + rest)
    lp = d - lz[:, None]
    place = (at == tokens[:, None].long()).to(torch.uint8).argmax(1, keepdim=True)
    return (lp.gather(1, place)[:, 0], place[:, 0] + 1, lz - t, lp[:, :top], at[:, :top], rest)


# A thread adds 64 terms one after the other, then 4 + 2 over a wave, 2 over its workgroup and 6 over the
# segments: 78 roundings of 2^-24. A term's own error: the exponential's (2^-23) and its argument's, half a
# step of at most 150, times ln 2. 190 2^-24 in all, relative to a sum of positive terms.
SUM = 190 * 2.0 ** -24
STEP = 2.0 ** -24


def check(got, x, tokens, top):
    lp, rank, h, tlp, tids, rest = exact(x, tokens, top)
    assert got.rank.dtype == torch.int32 and torch.equal(got.rank.long(), rank)
    assert got.top_ids.dtype == torch.int32 and torch.equal(got.top_ids.long(), tids)
    log_z = SUM * rest / (1 + rest)                  # ln(1 + rest) of a rest off by SUM

    def near(a, b, extra):
        fine = torch.isfinite(b)
        assert a.dtype == torch.float32 and torch.equal(a.double()[~fine], b[~fine])
        err = (a.double() - b).abs()
        bad = fine & ~(err <= extra + 4 * STEP * b.abs())
        assert not bad.any(), (err[bad], b[bad])
    # x - m and the subtraction of ln Z, rounded, are both within the steps of |logprob| + 2 ln Z
    lz = torch.log1p(rest)
    near(got.logprob, lp, log_z + 4 * STEP * lz)
    near(got.top_logprobs, tlp, (log_z + 4 * STEP * lz)[:, None])
    near(got.entropy, h, 3 * SUM * h)                # two sums of one sign each, and their quotient


def rows_of(R, V, dtype, seed, pad=0, offset=0):
    """Logits with a few high ones a row, every fourth row nearly certain, between columns of NaN."""
    g = torch.Generator(DEV).manual_seed(seed)
    buf = torch.full((R * (V + pad) + offset,), NAN, dtype=TYPES[dtype], device=DEV)
    x = buf[offset:].view(R, V + pad)[:, :V]
    f = 2.5 * torch.randn(R, V, generator=g, device=DEV)
    f.scatter_add_(1, torch.randint(V, (R, 5), generator=g, device=DEV),
                   8 + 4 * torch.rand(R, 5, generator=g, device=DEV))
    f[::4, V // 2] = 40.0
    x.copy_(f)
    t = torch.randint(V, (R,), generator=g, device=DEV)
    return x, torch.where(torch.rand(R, generator=g, device=DEV) < 0.5, x.argmax(1), t)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,top,pad,offset", [
    (3, 1, 1, 0, 0), (5, 2, 2, 1, 1), (4, 5, 5, 0, 3), (7, 33, 20, 2, 0), (9, 255, 32, 0, 1),
    (2, 256, 0, 0, 0), (6, 2047, 1, 3, 2), (6, 2049, 7, 7, 1), (4, 4096, 32, 0, 0), (3, 8191, 20, 5, 3),
    (5, 16385, 5, 1, 7), (17, 32003, 20, 2, 5), (2, 65537, 32, 0, 1), (1, 151936, 0, 0, 0),
    (20, 151936, 20, 0, 0), (300, 50001, 3, 3, 1), (520, 33000, 32, 0, 0), (2, 499999, 32, 1, 1),
    (1, 500000, 20, 0, 0), (70000, 9, 2, 0, 0)])
def test_values_ranks_and_ids(score, dtype, R, V, top, pad, offset):
    x, t = rows_of(R, V, dtype, R + V + top, pad, offset)
    gpu_case(f"logprobs {dtype} R={R} V={V} top={top} pad={pad} offset={offset}")
    got = score(x, t, top)
    torch.cuda.synchronize()
    check(got, x, t, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [40, 5000, 70001])
def test_equal_logits_go_by_index(score, dtype, V):
    """Runs of equal logits longer than any list holds, the two zeros among them, and sorted rows."""
    g = torch.Generator(DEV).manual_seed(V)
    x = torch.zeros(8, V, device=DEV)
    x[0] = 3.0
    x[1] = -torch.randint(0, 2, (V,), generator=g, device=DEV).float()
    x[2] = torch.where(torch.rand(V, generator=g, device=DEV) < 0.5, 0.0, -0.0)
    x[3] = torch.linspace(-20, 20, V, device=DEV)
    x[4] = torch.linspace(20, -20, V, device=DEV)
    x[5, V // 3:V // 3 + 30] = 5.0
    x[6] = torch.randint(-2, 3, (V,), generator=g, device=DEV).float()
    x[7] = -7.25
    x = x.to(TYPES[dtype])
    gpu_case(f"logprobs ties {dtype} V={V}")
    for top in (1, 20, 32):
        for t in (0, 1, V // 3 + 7, V - 1):
            tok = torch.full((8,), t, device=DEV)
            got = score(x, tok, top)
            torch.cuda.synchronize()
            check(got, x, tok, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V", [(7, 3001), (16, 16387), (40, 33001), (200, 33001)])
def test_candidates_around_a_lists_length(score, dtype, R, V):
    """So many elements at the highest value that a wave lists from none to all of its threads, and up to and past
    the 256 that its list holds; a few higher ones in every other row."""
    g = torch.Generator(DEV).manual_seed(R + V)
    share = torch.tensor([0.001, 0.004, 0.01, 0.02, 0.04, 0.06, 0.0625, 0.07, 0.1, 0.2], device=DEV)
    f = 2.0 * torch.rand(R, V, generator=g, device=DEV)
    many = torch.rand(R, V, generator=g, device=DEV) < share.repeat(-(-R // 10))[:R, None]
    f[many] = 4.0
    f[::2].scatter_(1, torch.randint(V, (len(f[::2]), 4), generator=g, device=DEV), 6.0)
    f[::3] -= 9.0
    x = f.to(TYPES[dtype])
    tok = torch.randint(V, (R,), generator=g, device=DEV)
    gpu_case(f"logprobs candidates {dtype} R={R} V={V}")
    for top in (1, 3, 20, 32):
        got = score(x, tok, top)
        torch.cuda.synchronize()
        check(got, x, tok, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,offset", [(50, 0), (3000, 1), (70001, 3)])
def test_masked_rows(score, dtype, V, offset):
    """-inf everywhere, but for one, for fewer than the alternatives, for most; the type's lowest value in
    their place, alone and beside -inf; tokens on both sides of the mask."""
    low = torch.finfo(TYPES[dtype]).min
    buf = torch.empty(9 * V + offset, dtype=TYPES[dtype], device=DEV)
    x = buf[offset:].view(9, V)
    g = torch.Generator(DEV).manual_seed(V)
    f = torch.randn(9, V, generator=g, device=DEV) * 3
    x.copy_(f)
    x[0] = NINF
    x[1] = NINF
    x[1, V - 2] = 1.5
    x[2] = NINF
    x[2, 5:12] = f[2, 5:12].to(x.dtype)
    x[3][torch.rand(V, generator=g, device=DEV) < 0.9] = NINF
    x[4] = low
    x[5] = low
    x[5, 7] = 2.0
    x[6] = NINF
    x[6, ::3] = low
    x[7][torch.rand(V, generator=g, device=DEV) < 0.5] = low
    x[8, :V // 2] = NINF
    gpu_case(f"logprobs masks {dtype} V={V}")
    for t in (0, 3, 7, V // 2, V - 1):
        tok = torch.full((9,), t, dtype=torch.int32, device=DEV)
        got = score(x, tok, 20)
        torch.cuda.synchronize()
        check(got, x, tok, 20)
        assert got.entropy[0] == 0 and (got.top_logprobs[0] == NINF).all()
        assert torch.equal(got.top_ids[0].long(), torch.arange(20, device=DEV))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [9, 3000, 70001])
def test_nan_and_inf_rows_and_tokens_out_of_range(score, dtype, V):
    x, t = rows_of(12, V, dtype, V, 1, 1)
    bad = {1: (0, NAN), 3: (V - 1, INF), 4: (V // 2, -NAN), 6: (V // 3, NAN), 8: (V - 1, NAN)}
    for r, (j, v) in bad.items():
        x[r, j] = v
    x[6] = torch.where(torch.isnan(x[6]), x[6], NINF)                # NaN and -inf alone
    x[8] = NAN
    x[9] = INF
    t[10], t[11] = -1, V
    wide = t.clone()
    wide[5] = -2 ** 40
    wide[7] = 2 ** 40
    gpu_case(f"logprobs NaN {dtype} V={V}")
    top = min(V, 5)
    for tok in (t, t.int(), wide):
        got = score(x, tok, top)
        torch.cuda.synchronize()
        broken = sorted(bad) + [9]
        for a in (got.logprob, got.entropy, got.top_logprobs):
            assert a[broken].isnan().all()
        assert (got.rank[broken] == 0).all() and (got.top_ids[broken] == -1).all()
        asks = tok.clone()
        out = (tok < 0) | (tok >= V)
        asks[out] = 0
        fine = [r for r in range(12) if r not in broken]
        for r in fine:
            if tok[r] < 0:
                assert got.logprob[r] == 0 and got.rank[r] == 0
            elif tok[r] >= V:
                assert got.logprob[r].isnan() and got.rank[r] == 0
        want = exact(x[fine], asks[fine], top)
        ok = ~out[fine]
        assert torch.equal(got.rank[fine].long()[ok], want[1][ok])
        assert torch.equal(got.top_ids[fine].long(), want[4])
        torch.testing.assert_close(got.entropy[fine].double(), want[2], rtol=4 * SUM, atol=0)


@pytest.mark.parametrize("scale", [1e-30, 1e4, 1e30, 1e38, 3e38])
def test_large_and_small_logits(score, scale):
    g = torch.Generator(DEV).manual_seed(1)
    x = (torch.rand(6, 9000, generator=g, device=DEV) * 2 - 1) * scale
    x[1] = x[1].abs()
    x[2] = -x[2].abs() - scale * 0.1
    x[3] = scale
    x[4] = -scale
    t = torch.randint(9000, (6,), generator=g, device=DEV)
    gpu_case(f"logprobs scale={scale}")
    got = score(x, t, 20)
    torch.cuda.synchronize()
    lp, rank, h, tlp, tids, _ = exact(x, t, 20)
    assert torch.equal(got.rank.long(), rank) and torch.equal(got.top_ids.long(), tids)
    # a difference past float32's range is -inf
    lp, tlp = lp.float().double(), tlp.float().double()
    torch.testing.assert_close(got.logprob.double(), lp, rtol=8 * STEP, atol=2 * SUM)
    torch.testing.assert_close(got.top_logprobs.double(), tlp, rtol=8 * STEP, atol=2 * SUM)
    torch.testing.assert_close(got.entropy.double(), h, rtol=4 * SUM, atol=1e-37)


def test_no_rows_and_no_alternatives(score):
    out = score(torch.empty(0, 100, device=DEV), torch.empty(0, dtype=torch.int64, device=DEV), 5)
    assert [tuple(a.shape) for a in out] == [(0,), (0,), (0,), (0, 5), (0, 5)]
    out = score(torch.zeros(2, 100, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV))
    assert out.top_ids.shape == (2, 0)


def test_logits_past_2_to_31_elements(score):
    R, V = 14200, 151936                                             # 2.16e9 of them, 4.3 GB
    x = torch.zeros(R, V, dtype=torch.bfloat16, device=DEV)
    y, t = rows_of(30, V, "bf16", 3)
    x[-30:] = y
    tok = torch.full((R,), 5, device=DEV)
    tok[-30:] = t
    gpu_case("logprobs past 2^31 elements")
    got = score(x, tok, 20)
    torch.cuda.synchronize()
    check(type(got)(*[a[-30:] for a in got]), y, t, 20)
    check(type(got)(*[a[:30] for a in got]), x[:30], tok[:30], 20)


def test_repeats_and_streams_bit_for_bit(score):
    x, t = rows_of(40, 70001, "bf16", 1)
    gpu_case("logprobs on three streams at once")
    torch.cuda.synchronize()
    got = []
    for st in [torch.cuda.Stream() for _ in range(3)]:
        with torch.cuda.stream(st):
            got += [score(x, t, 20) for _ in range(3)]
    torch.cuda.synchronize()
    for g in got[1:]:
        for a, b in zip(got[0], g):
            assert torch.equal(a, b)


def test_graphs_replayed_with_new_logits(score):
    """Two captured graphs, replayed at once, eager calls between."""
    cases = [rows_of(24, 32003, "f16", s) for s in range(3)]
    ins = [(cases[0][0].clone(), cases[0][1].clone()) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    gpu_case("logprobs graphs")
    torch.cuda.synchronize()
    for (x, t), st in zip(ins, streams):
        with torch.cuda.stream(st):
            score(x, t, 20)
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(score(x, t, 20))
        graphs.append(g)
    for i in (1, 2, 0, 1):
        for j, st in enumerate(streams):
            with torch.cuda.stream(st):
                ins[j][0].copy_(cases[(i + j) % 3][0])
                ins[j][1].copy_(cases[(i + j) % 3][1])
                graphs[j].replay()
        eager = score(*cases[i], 20)
        torch.cuda.synchronize()
        check(eager, *cases[i], 20)
        for j in range(2):
            check(outs[j], *cases[(i + j) % 3], 20)


# ---- the head's scoring: quantized rows, the product, the log probabilities ---------------------
@pytest.mark.parametrize("shape,N", [((5,), 1152), ((2, 33), 2048), ((70,), 1152), ((3, 700), 1280)])
def test_head_logprobs(mods, shape, N):
    """Of the logits that the two calls give (ranks and ids of these bf16 logits exactly), over row chunks."""
    lp, ops = mods
    K = 512
    g = torch.Generator(DEV).manual_seed(N + len(shape))
    weight = (torch.randn(N, K, generator=g, device=DEV) * 0.1).bfloat16()

    class Orig:
        def apply(self, layer, x, bias=None):
            raise AssertionError("not for scoring")
    head = ops.Fp8TargetHead(Orig(), weight)
    x = torch.randn(*shape, K, generator=g, device=DEV).bfloat16()
    t = torch.randint(N, shape, generator=g, device=DEV)
    t.view(-1)[0] = -1
    gpu_case(f"head logprobs {shape} N={N}")
    got = head.logprobs(x, t, 7)
    flat = x.reshape(-1, K)
    w = ops.PackedFp8(wq=head.wq, ws=head.ws, n=N, k=K)
    logits = ops.gemm_fp8_dense(*ops.fp8_quant_group(flat), w)
    torch.cuda.synchronize()
    assert got.logprob.shape == shape and got.top_ids.shape == (*shape, 7)
    if flat.shape[0] <= 64:
        assert torch.equal(logits, head.apply(None, x).reshape(-1, N))
    assert got.logprob.view(-1)[0] == 0 and got.rank.view(-1)[0] == 0
    one = lp.TokenLogprobs(*[a.reshape(flat.shape[0], *a.shape[len(shape):])[1:] for a in got])
    check(one, logits[1:], t.reshape(-1)[1:], 7)


def test_head_logprobs_in_chunks_and_of_no_rows(mods, monkeypatch):
    lp, ops = mods
    g = torch.Generator(DEV).manual_seed(9)
    head = ops.Fp8TargetHead(object(), torch.randn(1024, 256, generator=g, device=DEV).bfloat16())
    x = torch.randn(600, 256, generator=g, device=DEV).bfloat16()
    t = torch.randint(1024, (600,), generator=g, device=DEV)
    gpu_case("head logprobs in chunks")
    whole = head.logprobs(x, t, 3)
    monkeypatch.setattr(ops, "LOGPROBS_ROWS", 256)
    parts = head.logprobs(x[:, :], t, 3)
    torch.cuda.synchronize()
    # (a chunk of fewer rows may run another tile, whose sums are taken in another order)
    torch.testing.assert_close(parts.logprob, whole.logprob, rtol=0, atol=0.26)
    assert parts.top_ids.shape == whole.top_ids.shape == (600, 3)
    none = head.logprobs(x[:0], t[:0], 3)
    assert none.logprob.shape == (0,) and none.top_ids.shape == (0, 3)
    wide = torch.randn(600, 512, generator=g, device=DEV).bfloat16()
    wide[:, ::2] = x
    again = head.logprobs(wide[:, ::2], t, 3)
    for a, b in zip(parts, again):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows", [20, 300])
def test_head_logprobs_in_a_replayed_graph(mods, rows):
    _, ops = mods
    g = torch.Generator(DEV).manual_seed(rows)
    head = ops.Fp8TargetHead(object(), torch.randn(1280, 512, generator=g, device=DEV).bfloat16())
    xs = [torch.randn(rows, 512, generator=g, device=DEV).bfloat16() for _ in range(3)]
    ts = [torch.randint(1280, (rows,), generator=g, device=DEV) for _ in range(3)]
    gpu_case(f"head logprobs graph rows={rows}")
    x, t, st = xs[0].clone(), ts[0].clone(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        head.logprobs(x, t, 5)
    st.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        out = head.logprobs(x, t, 5)
    for i in (0, 1, 2, 1):
        with torch.cuda.stream(st):
            x.copy_(xs[i])
            t.copy_(ts[i])
            graph.replay()
        want = head.logprobs(xs[i], ts[i], 5)
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rows", [1, 4])
def test_head_logprobs_of_strided_rows_and_tokens(mods, rows):
    """Rows and tokens apart, at any stride, and one row expanded: as their copies."""
    _, ops = mods
    g = torch.Generator(DEV).manual_seed(rows)
    head = ops.Fp8TargetHead(object(), torch.randn(256, 128, generator=g, device=DEV).bfloat16())
    x = torch.randn(rows, 128, generator=g, device=DEV).bfloat16()
    t = torch.randint(256, (rows,), generator=g, device=DEV)
    gpu_case(f"head logprobs strided rows={rows}")
    odd = torch.zeros(rows, 133, device=DEV).bfloat16()
    odd[:, :128] = x
    apart = torch.zeros(rows, 256, device=DEV).bfloat16()
    apart[:, ::2] = x
    ids = torch.zeros(rows, 3, dtype=torch.int64, device=DEV)
    ids[:, 1] = t
    for a, b, want in ((odd[:, :128], ids[:, 1], (x, t)), (apart[:, ::2], t, (x, t)),
                       (x[:1].expand(rows, 128), t, (x[:1].repeat(rows, 1), t)),
                       (x, t[:1].expand(rows), (x, t[:1].repeat(rows)))):
        for p, q in zip(head.logprobs(a, b, 3), head.logprobs(*want, 3)):
            assert torch.equal(p, q)


@pytest.mark.parametrize("shape,N,K,rows", [((600,), 1024, 256, 256), ((3, 700), 1280, 512, 1024),
                                            ((129,), 2048, 384, 64), ((65,), 1152, 2560, 1),
                                            ((5, 3), 1152, 256, 15)])
def test_head_logprobs_are_those_of_its_chunks(mods, monkeypatch, shape, N, K, rows):
    """Every field, bit for bit, of the two calls on each `rows` rows, joined in order."""
    lp, ops = mods
    g = torch.Generator(DEV).manual_seed(N + K + rows)
    head = ops.Fp8TargetHead(object(), (torch.randn(N, K, generator=g, device=DEV) * 0.1).bfloat16())
    x = torch.randn(*shape, K, generator=g, device=DEV).bfloat16()
    t = torch.randint(N, shape, generator=g, device=DEV)
    monkeypatch.setattr(ops, "LOGPROBS_ROWS", rows)
    gpu_case(f"head logprobs chunks {shape} N={N} K={K} rows={rows}")
    got = head.logprobs(x, t, 6)
    flat, ids = x.reshape(-1, K), t.reshape(-1)
    w = ops.PackedFp8(wq=head.wq, ws=head.ws, n=N, k=K)
    at = 0
    for r in range(0, flat.shape[0], rows):
        logits = ops.gemm_fp8_dense(*ops.fp8_quant_group(flat[r:r + rows]), w)
        want = lp.token_logprobs(logits, ids[r:r + rows], 6)
        torch.cuda.synchronize()
        check(want, logits, ids[r:r + rows], 6)
        for name, a, b in zip(lp.TokenLogprobs._fields, got, want):
            part = a.reshape(flat.shape[0], *a.shape[len(shape):])[at:at + b.shape[0]]
            assert torch.equal(part, b), (name, r)
        at += want.logprob.shape[0]
    assert at == flat.shape[0] and all(a.shape[:len(shape)] == shape for a in got)
