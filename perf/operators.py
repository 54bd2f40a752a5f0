"""Timed cases of scoring: the fp8 block-scaled product for any number of rows, and the log
probabilities of given tokens with rank, entropy and top alternatives.

A case is a dict of plain values; its "kind" says which operator it runs:

  gemm      y [rows, cols] bf16 = x [rows, depth] w [cols, depth]^T of e4m3 values, x with a float32
            scale per row and 128 columns, w with one per 128 x 128 block.
  logprobs  for each row of logits [rows, vocab]: the given token's log probability and rank, the
            entropy, and the `top` largest log probabilities with their ids, ties to the lowest id.
            `pad` columns of the buffer lie between two rows' logits. `masked` rows have most of the
            vocabulary at -inf, every fifth of them all of it.

    listed()  the cases           draw(rng)  one more of the same ranges
    prepare / run / work / exact  of one case; `own`: run calls the package, else plain torch
"""
from __future__ import annotations

import importlib.util
import pathlib
import sys

import torch

ROOT = pathlib.Path(__file__).resolve().parent.parent
PKG_NAME = "r9700_lru_expert_cache_amd"
DEV = "cuda"
VOCAB = 151936
ROWS = 512                # rows at a time where a whole temporary would be several times the input
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

own = False


def _pkg():
    if PKG_NAME in sys.modules:
        return sys.modules[PKG_NAME]
    d = ROOT / "r9700-lru-expert-cache_amd"
    spec = importlib.util.spec_from_file_location(PKG_NAME, d / "__init__.py",
                                                  submodule_search_locations=[str(d)])
    mod = importlib.util.module_from_spec(spec)
    sys.modules[PKG_NAME] = mod
    spec.loader.exec_module(mod)
    return mod


# ---- the cases ----------------------------------------------------------------------------------
def _gemm(name, rows, cols, depth):
    c = dict(kind="gemm", rows=rows, cols=cols, depth=depth)
    return dict(c, name=name) if name else c


def _logprobs(name, rows, vocab, dtype, top, pad=0, masked=False):
    c = dict(kind="logprobs", rows=rows, vocab=vocab, dtype=dtype, top=top, pad=pad, masked=masked)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token through a projection of the 2560-wide model: launch latency
        _gemm("gemm_1", 1, 2560, 2560),
        # the drafts of 32 streams, 5 rows each, through the target head: still the weights' read
        _gemm("gemm_160_head", 160, VOCAB, 2560),
        # a short ragged prompt through a projection with an odd number of outputs
        _gemm("gemm_617_ragged", 617, 1543, 768),
        # a prompt chunk through a square projection
        _gemm("gemm_4096", 4096, 2560, 2560),
        # a chunk's logits, for the log probabilities of a prompt
        _gemm("gemm_2048_head", 2048, VOCAB, 2560),
        # the largest chunk through a wide projection
        _gemm("gemm_8192_wide", 8192, 10240, 2560),
        # one sampled token, its log probability only: launch latency
        _logprobs("logprobs_1", 1, VOCAB, "bf16", 0),
        # a 4-stream verification step, 5 rows each, with the usual limit of 20 alternatives
        _logprobs("logprobs_20_top20", 20, VOCAB, "bf16", 20),
        # a wide decode batch under grammar masks, float32 logits after penalties
        _logprobs("logprobs_256_masked", 256, VOCAB, "f32", 5, masked=True),
        # a short prompt over a small odd vocabulary, rows that start at odd addresses
        _logprobs("logprobs_617_odd", 617, 32003, "f16", 1, pad=2),
        # a prompt chunk's scores without alternatives
        _logprobs("logprobs_2048", 2048, VOCAB, "f32", 0),
        # the largest chunk with 20 alternatives
        _logprobs("logprobs_4096_top20", 4096, VOCAB, "bf16", 20),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    if rng.random() < 0.5:
        depth = 128 * _log_int(rng, 4, 32)
        cols = VOCAB if rng.random() < 0.25 else _log_int(rng, 100, 16384)
        most = 2048 * VOCAB * 2560 // (cols * depth)
        return _gemm(None, _log_int(rng, 1, min(8192, most)), cols, depth)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    vocab = VOCAB if rng.random() < 0.4 else _log_int(rng, 500, 200000)
    most = 4096 * VOCAB * 2 // ((4 if dtype == "f32" else 2) * vocab)
    return _logprobs(None, _log_int(rng, 1, min(8192, most)), vocab, dtype,
                     rng.choice([0, 1, 5, rng.randint(2, 20), 20]), pad=rng.choice([0, 0, 1, 5, 64]),
                     masked=rng.random() < 0.25)


# ---- inputs -------------------------------------------------------------------------------------
def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed(seed * 16 + salt)


def _quantized(case, seed):
    """Hidden states with a few large channels, e4m3 with a scale per row and 128 columns; weights,
    e4m3 with a scale per 128 x 128 block (the last one of fewer rows where cols ends in it)."""
    m, n, k = case["rows"], case["cols"], case["depth"]
    g = _gen(seed, 1)
    x = torch.randn(m, k, generator=g, device=DEV)
    x *= torch.exp(0.7 * torch.randn(k, generator=g, device=DEV))
    x = x.view(m, k // 128, 128)
    xs = x.abs().amax(2).clamp_(min=1e-5) / 448.0
    qx = (x / xs[:, :, None]).clamp_(-448, 448).view(m, k).to(torch.float8_e4m3fn)
    w = torch.empty(n, k, dtype=torch.float8_e4m3fn, device=DEV)
    ws = torch.empty(-(-n // 128), k // 128, device=DEV)
    for r0 in range(0, n, 16384):
        r1 = min(n, r0 + 16384)
        f = torch.zeros(-(-(r1 - r0) // 128) * 128, k, device=DEV)
        f[:r1 - r0] = 0.02 * torch.randn(r1 - r0, k, generator=g, device=DEV)
        f = f.view(-1, 128, k // 128, 128)
        s = f.abs().amax(dim=(1, 3), keepdim=True) / 448.0
        w[r0:r1] = (f / s).clamp_(-448, 448).view(-1, k)[:r1 - r0].to(torch.float8_e4m3fn)
        ws[r0 // 128:r0 // 128 + s.shape[0]] = s[:, 0, :, 0]
    return qx, xs, w, ws


def _logits(case, seed):
    """Logits of a head: a broad bulk, a few high ones per row, one row in four nearly certain, and
    the tokens to score: half drawn from the high ones, half anywhere."""
    r, v = case["rows"], case["vocab"]
    g = _gen(seed, 2)
    buf = torch.empty(r, v + case["pad"], dtype=DTYPES[case["dtype"]], device=DEV)
    logits = buf[:, :v]
    high = torch.randint(v, (r, 32), generator=g, device=DEV)
    lift = 8.0 + 4.0 * torch.rand(r, 32, generator=g, device=DEV)
    lift[::4, 0] = 24.0
    for r0 in range(0, r, ROWS):
        x = 2.5 * torch.randn(min(r, r0 + ROWS) - r0, v, generator=g, device=DEV)
        x.scatter_add_(1, high[r0:r0 + ROWS], lift[r0:r0 + ROWS])
        if case["masked"]:
            keep = torch.rand(x.shape, generator=g, device=DEV) < 0.002
            keep[::5] = False
            x.masked_fill_(~keep, float("-inf"))
        logits[r0:r0 + ROWS] = x
    tokens = torch.randint(v, (r,), generator=g, device=DEV)
    pick = high.gather(1, torch.randint(32, (r, 1), generator=g, device=DEV))[:, 0]
    tokens = torch.where(torch.rand(r, generator=g, device=DEV) < 0.5, pick, tokens)
    return logits, tokens


def prepare(case, seed):
    if case["kind"] == "logprobs":
        logits, tokens = _logits(case, seed)
        return dict(case=case, logits=logits, tokens=tokens)
    qx, xs, w, ws = _quantized(case, seed)
    if own:
        # as a server holds it: the weight laid out once, at load
        return dict(case=case, qx=qx, xs=xs, packed=_pkg().ops.pack_fp8_dense(w, ws))
    return dict(case=case, qx=qx, xs=xs, w=w, ws=ws)


# ---- one pass -----------------------------------------------------------------------------------
def _dequant(q, s, block, dtype):
    """q [n, k] times its scale per `block` rows and 128 columns."""
    n, k = q.shape
    s = s.to(dtype).repeat_interleave(block, 0)[:n]
    return (q.to(dtype).view(n, k // 128, 128) * s[:, :, None]).view(n, k)


def _plain_gemm(state):
    x = _dequant(state["qx"], state["xs"], 1, torch.float32)
    w = _dequant(state["w"], state["ws"], 128, torch.float32)
    return (x @ w.T).to(torch.bfloat16)


def _order(x):
    """int64 keys that order the values of each row, the lowest index first among equals."""
    b = x.float().view(torch.int32).to(torch.int64)
    b = torch.where(x == 0, 0, b)                       # the two zeros are equal
    b = torch.where(b < 0, -(b + 2 ** 31), b)
    return b * 2 ** 20 + (2 ** 20 - 1 - torch.arange(x.shape[1], device=x.device))


def _plain_logprobs(logits, tokens, top):
    x = logits.float()
    m = x.amax(1, keepdim=True)
    none = torch.isinf(m)                               # nothing left of the row
    d = x - torch.where(none, 0.0, m)
    e = torch.exp(d)
    # the sum without the maximum's own 1, which a nearly certain row's small terms would be lost in
    rest = e.scatter(1, x.argmax(1, keepdim=True), 0.0).sum(1, keepdim=True)
    rest = torch.where(none, 0.0, rest)
    lz = torch.log1p(rest)
    h = lz - torch.where(e > 0, d * e, 0.0).sum(1, keepdim=True) / (1.0 + rest)
    lp = d.gather(1, tokens[:, None]) - lz
    xt = x.gather(1, tokens[:, None])
    before = torch.arange(x.shape[1], device=x.device) < tokens[:, None]
    rank = 1 + (x > xt).sum(1) + ((x == xt) & before).sum(1)
    ids = torch.topk(_order(x), top, dim=1).indices
    return (lp[:, 0], rank.to(torch.int32), h[:, 0], d.gather(1, ids) - lz, ids.to(torch.int32))


def _parts(f, logits, tokens, top):
    """f over ROWS rows at a time, joined."""
    n = logits.shape[0]
    out = [f(logits[r:r + ROWS], tokens[r:r + ROWS], top) for r in range(0, n, ROWS)]
    return out[0] if len(out) == 1 else tuple(torch.cat(t) for t in zip(*out))


NAMES = ("logprob", "rank", "entropy", "top_logprobs", "top_ids")


def run(state):
    if state["case"]["kind"] == "gemm":
        if own:
            return _pkg().ops.gemm_fp8_dense(state["qx"], state["xs"], state["packed"])
        return _plain_gemm(state)
    top = state["case"]["top"]
    if own:
        out = _pkg().logprobs.token_logprobs(state["logits"], state["tokens"], top)
    else:
        out = _parts(_plain_logprobs, state["logits"], state["tokens"], top)
    return {k: t for k, t in zip(NAMES, out) if t.numel()}


# ---- what a pass has to do ----------------------------------------------------------------------
def work(case):
    if case["kind"] == "gemm":
        m, n, k = case["rows"], case["cols"], case["depth"]
        return dict(bytes=m * k + m * k // 32 + n * k + n * k // 4096 + 2 * m * n,
                    flops=2 * m * n * k)
    r, v = case["rows"], case["vocab"]
    size = 4 if case["dtype"] == "f32" else 2
    # an element: the difference to the maximum, the exponential, two sums
    return dict(bytes=r * (v * size + 8 + 12 + 8 * case["top"]), flops=4 * r * v)


# ---- the same in 64 bits ------------------------------------------------------------------------
def _exact_gemm(case, seed):
    qx, xs, w, ws = _quantized(case, seed)
    out = torch.zeros(case["rows"], case["cols"], dtype=torch.float64, device=DEV)
    for kb in range(xs.shape[1]):
        k = slice(128 * kb, 128 * kb + 128)
        wk = w[:, k].double() * ws[:, kb].double().repeat_interleave(128)[:w.shape[0], None]
        out.addmm_(qx[:, k].double() * xs[:, kb, None].double(), wk.T)
    return out


def _exact_rows(logits, tokens, top):
    """By sorting each row: ranks and alternatives are places in a stable descending order."""
    x = logits.double()
    s, at = torch.sort(x, dim=1, descending=True, stable=True)
    lse = torch.logsumexp(x, 1, keepdim=True)
    lp = s - torch.where(torch.isinf(lse), 0.0, lse)
    h = -torch.where(lp > float("-inf"), torch.exp(lp) * lp, 0.0).sum(1)
    place = (at == tokens[:, None]).to(torch.uint8).argmax(1, keepdim=True)
    return (lp.gather(1, place)[:, 0], (place[:, 0] + 1).to(torch.int32), h, lp[:, :top],
            at[:, :top].to(torch.int32))


def exact(case, seed):
    if case["kind"] == "gemm":
        return _exact_gemm(case, seed)
    out = _parts(_exact_rows, *_logits(case, seed), case["top"])
    return {k: t for k, t in zip(NAMES, out) if t.numel()}
