"""ops.gemm_fp8_dense against float64: exactly where every sum is, within derived limits elsewhere."""
from __future__ import annotations

from importlib import import_module

import pytest

from conftest import gpu_case

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DEV = "cuda"
F8, BF = torch.float8_e4m3fn, torch.bfloat16


@pytest.fixture(scope="module")
def ops(pkg):
    return import_module(pkg.__name__ + ".ops")


def whole(M, N, K, seed, density=0.25):
    """Operands of -1, 0 and 1 with scales that are powers of two, block by block: every product and sum
    is exact in the matrix unit and in float32."""
    g = torch.Generator(DEV).manual_seed(seed)
    t = lambda *s: (torch.randint(0, 2, s, generator=g, device=DEV) * 2 - 1).float() * \
        (torch.rand(*s, generator=g, device=DEV) < density)
    p = lambda *s: torch.exp2(torch.randint(-2, 3, s, generator=g, device=DEV).float())
    return (t(M, K).to(F8), p(M, K // 128), t(N, K).to(F8), p(-(-N // 128), K // 128))


def exact(qx, xs, w, ws):
    x = qx.double().view(*xs.shape, 128) * xs.double()[:, :, None]
    s = ws.double().repeat_interleave(128, 0)[:w.shape[0]]
    y = w.double().view(w.shape[0], -1, 128) * s[:, :, None]
    return x.reshape(qx.shape) @ y.reshape(w.shape).T


# Rows and columns around each kernel's tiles: up to 64 rows and few columns the head's kernel, then 128 x
# 128, 192 x 256 and 256 x 256; K / 128 = 1, 2, 3, 9, 16 and 20 steps (the scales are staged by 8).
SHAPES = [(1, 1, 128), (1, 128, 256), (3, 5, 384), (17, 129, 1152), (63, 127, 128), (64, 300, 2560),
          (65, 1, 128), (65, 7, 256), (127, 129, 384), (128, 128, 128), (129, 1543, 1152),
          (200, 4099, 384), (255, 256, 2048), (257, 257, 2560), (300, 9999, 128), (617, 1543, 768),
          (1025, 2600, 1152), (2100, 6145, 384), (4096, 2560, 256), (4100, 2561, 1152),
          (700, 33000, 256), (1500, 40000, 1152), (193, 60000, 2048), (160, 151936, 256),
          # 31 and 97 steps, which the head's kernel does not take
          (1024, 2561, 2560), (7, 300, 3968), (40, 129, 12416)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_whole_numbers_are_exact(ops, M, N, K):
    qx, xs, w, ws = whole(M, N, K, M * 7 + N + K)
    gpu_case(f"dense exact M={M} N={N} K={K}")
    # rows apart in a buffer with 5 more columns and a row before and behind: they stay as they were
    buf = torch.full((M + 2, N + 5), 7.0, dtype=BF, device=DEV)
    y = ops.gemm_fp8_dense(qx, xs, ops.pack_fp8_dense(w, ws), out=buf[1:-1, :N])
    torch.cuda.synchronize()
    want = exact(qx, xs, w, ws).to(BF)
    assert torch.equal(y, want)
    for rest in (buf[0], buf[-1], buf[:, N:]):
        assert (rest == 7.0).all()
    # whole vectors: an aligned buffer
    cols = -(-N // 8) * 8
    buf = torch.full((M, cols), 7.0, dtype=BF, device=DEV)
    ops.gemm_fp8_dense(qx, xs, ops.pack_fp8_dense(w, ws), out=buf[:, :N])
    torch.cuda.synchronize()
    assert torch.equal(buf[:, :N], want) and (buf[:, N:] == 7.0).all()


@pytest.mark.parametrize("M,N,K", [(20, 300, 2560), (65, 129, 1152), (617, 1543, 768), (1500, 9000, 2560),
                                   (4096, 2560, 1152), (2100, 20000, 512), (193, 60000, 1408)])
def test_random_values(ops, M, N, K):
    """Of quantized rows and weights with outlying channels. The limit, from the sum S of the products'
    magnitudes: half a bf16 step of the value (2^-8), the float32 sums over K / 128 steps and their
    scales ((K / 128 + 2) 2^-24 S), and the matrix unit's own sum, 2^-14 S: it brings an instruction's
    products to one exponent before it adds them, which over 512 random 16 x 16 x 128 products came to
    2.3e-5 S at most, 2^-15.4."""
    g = torch.Generator(DEV).manual_seed(M + N + K)
    x = torch.randn(M, K, generator=g, device=DEV) * \
        torch.exp(torch.randn(K, generator=g, device=DEV))
    qx, xs = ops.fp8_quant_group(x.to(BF))
    w = (torch.randn(N, K, generator=g, device=DEV) * 100).clamp(-448, 448).to(F8)
    ws = torch.rand(-(-N // 128), K // 128, generator=g, device=DEV) * 0.01 + 1e-4
    gpu_case(f"dense random M={M} N={N} K={K}")
    y = ops.gemm_fp8_dense(qx, xs, ops.pack_fp8_dense(w, ws)).double()
    torch.cuda.synchronize()
    want = exact(qx, xs, w, ws)
    S = exact(qx.float().abs().to(F8), xs, w.float().abs().to(F8), ws)
    assert ((y - want).abs() <= 2 ** -8 * want.abs() + (2 ** -14 + (K // 128 + 2) * 2 ** -24) * S).all()


@pytest.mark.parametrize("M", [1, 8, 17, 48, 64])
def test_up_to_64_rows_equal_gemm_fp8_block(ops, M):
    """The same bits as the head's product of the same rows, which a server calls at decode."""
    g = torch.Generator(DEV).manual_seed(M)
    w = torch.randn(1152, 2560, generator=g, device=DEV) * 0.02
    wq, ws = ops.pack_fp8_block(w)
    qx, xs = ops.fp8_quant_group(torch.randn(M, 2560, generator=g, device=DEV).to(BF))
    gpu_case(f"dense against head M={M}")
    y = ops.gemm_fp8_dense(qx, xs, ops.PackedFp8(wq=wq, ws=ws, n=1152, k=2560))
    want = ops.gemm_fp8_block_q(qx, xs, wq, ws)
    torch.cuda.synchronize()
    assert torch.equal(y.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("M,N", [(40, 300), (300, 513), (2100, 6145), (4100, 2561)])
def test_nan_and_inf_stay_in_their_row_and_column(ops, M, N):
    K = 512
    qx, xs, w, ws = whole(M, N, K, 3)
    want = exact(qx, xs, w, ws).to(BF)
    row, col, scaled = M // 2, N // 3, M - 1
    qx.view(torch.uint8)[row, 77] = 0x7f                             # e4m3's NaN
    w.view(torch.uint8)[col, 300] = 0xff
    xs[scaled, 1] = float("inf")
    gpu_case(f"dense NaN M={M} N={N}")
    y = ops.gemm_fp8_dense(qx, xs, ops.pack_fp8_dense(w, ws))
    torch.cuda.synchronize()
    assert y[row].isnan().all() and y[:, col].isnan().all()
    assert not y[scaled].isfinite().any()          # (a step's sum of 0 times inf is NaN)
    keep = torch.ones_like(y, dtype=torch.bool)
    keep[row], keep[scaled], keep[:, col] = False, False, False
    assert torch.equal(y[keep], want[keep])


def test_no_rows(ops):
    qx, xs, w, ws = whole(4, 200, 256, 1)
    y = ops.gemm_fp8_dense(qx[:0], xs[:0], ops.pack_fp8_dense(w, ws))
    assert y.shape == (0, 200)


def test_packed_weight_is_padded_with_zeros(ops):
    _, _, w, ws = whole(1, 200, 256, 2)
    p = ops.pack_fp8_dense(w, ws)
    assert (p.n, p.k, p.n_pad, p.wq.shape) == (200, 256, 256, (256, 256))
    rows = torch.zeros(256, 256, dtype=torch.uint8, device=DEV)
    rows[:200] = w.view(torch.uint8)
    assert torch.equal(ops.shuffle_fp8_weight(rows.view(F8)).view(torch.uint8), p.wq.view(torch.uint8))


def test_block_scales_of_a_parameter(ops):
    """A layer's scales may ask for a gradient: the packed ones do not, and the product takes them."""
    qx, xs, w, ws = whole(20, 256, 256, 5)
    gpu_case("dense, a parameter's scales")
    p = ops.pack_fp8_dense(w, torch.nn.Parameter(ws))
    assert not p.ws.requires_grad
    y = ops.gemm_fp8_dense(qx, xs, p)
    torch.cuda.synchronize()
    assert torch.equal(y, exact(qx, xs, w, ws).to(BF))


@pytest.mark.parametrize("M,N,K", [(48, 300, 1152), (300, 1543, 768), (2100, 6145, 384)])
def test_other_streams_and_graph_replays(ops, M, N, K):
    """Two captured graphs replayed at once on two streams with new rows each time, beside eager calls."""
    a = [whole(M, N, K, s) for s in (1, 2, 3)]
    packs = [ops.pack_fp8_dense(w, ws) for _, _, w, ws in a]
    want = [[exact(a[i][0], a[i][1], a[j][2], a[j][3]).to(BF) for i in range(3)] for j in range(2)]
    gpu_case(f"dense graphs M={M} N={N} K={K}")
    streams = [torch.cuda.Stream() for _ in range(2)]
    ins = [(a[2][0].clone(), a[2][1].clone()) for _ in range(2)]
    outs, graphs = [], []
    torch.cuda.synchronize()
    for j, st in enumerate(streams):
        with torch.cuda.stream(st):
            ops.gemm_fp8_dense(*ins[j], packs[j])
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(ops.gemm_fp8_dense(*ins[j], packs[j]))
        graphs.append(g)
    for i in (0, 1, 2, 0):
        for j, st in enumerate(streams):
            with torch.cuda.stream(st):
                ins[j][0].view(torch.uint8).copy_(a[i][0].view(torch.uint8))
                ins[j][1].copy_(a[i][1])
                graphs[j].replay()
        eager = ops.gemm_fp8_dense(a[i][0], a[i][1], packs[0])
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0][i])
        for j in range(2):
            assert torch.equal(outs[j], want[j][i])


def test_output_past_2_to_31_elements(ops):
    M, N, K = 14200, 151936, 128                                     # 2.16e9 of them, 4.3 GB
    qx, xs, w, ws = whole(M, N, K, 5)
    gpu_case(f"dense M={M} N={N}, output past 2^31 elements")
    y = ops.gemm_fp8_dense(qx, xs, ops.pack_fp8_dense(w, ws))
    torch.cuda.synchronize()
    for r in (slice(0, 40), slice(7000, 7040), slice(M - 40, M)):
        assert torch.equal(y[r], exact(qx[r], xs[r], w, ws).to(BF))


def test_repeats_bit_for_bit(ops):
    g = torch.Generator(DEV).manual_seed(0)
    for M, N, K in ((300, 1543, 768), (2100, 6145, 1152)):
        qx, xs = ops.fp8_quant_group(torch.randn(M, K, generator=g, device=DEV).to(BF))
        p = ops.pack_fp8_dense(torch.randn(N, K, generator=g, device=DEV).to(F8),
                               torch.rand(-(-N // 128), K // 128, generator=g, device=DEV))
        gpu_case(f"dense repeats M={M} N={N}")
        a, b = (ops.gemm_fp8_dense(qx, xs, p) for _ in range(2))
        torch.cuda.synchronize()
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
