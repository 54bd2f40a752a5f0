"""Timed cases of what learns beside frozen quantized projections: low-rank adapters of many requests,
and the losses that teach them from scored logits, with their gradients.

A case is a dict of plain values; its "kind" says which operator it runs:

  lora       out [rows, cols] = y + s_a (x A_a^T) B_a^T with the adapter a of each row, `adapters` of
             rank `rank` in the stack. Rows come in runs of `run` (a stream's rows, a prompt) or, where
             it is 0, in runs of any length; `bare` leaves some runs without an adapter.
  lora_grad  the same and its backward pass: from dy the gradients of x, A and B.
  distill    for each row the divergence of a student's logits [rows, vocab] from a teacher's `top` log
             probabilities with the rest of the vocabulary as one outcome, and the logits' gradient.
  policy     for each row the clipped policy loss of a sampled token with a KL term against a reference
             policy, the token's log probability, and the logits' gradient. `masked` rows have most of
             the vocabulary at -inf.
             `pad` columns of the buffer lie between two rows' logits.

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
CLIP = (0.2, 0.28)
KL = 0.05

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
def _lora(name, kind, rows, cols, depth, rank, adapters, run, dtype="bf16", bare=False):
    c = dict(kind=kind, rows=rows, cols=cols, depth=depth, rank=rank, adapters=adapters, run=run,
             dtype=dtype, bare=bare)
    return dict(c, name=name) if name else c


def _distill(name, rows, vocab, dtype, top, pad=0):
    c = dict(kind="distill", rows=rows, vocab=vocab, dtype=dtype, top=top, pad=pad)
    return dict(c, name=name) if name else c


def _policy(name, rows, vocab, dtype, pad=0, masked=False):
    c = dict(kind="policy", rows=rows, vocab=vocab, dtype=dtype, pad=pad, masked=masked)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token through a projection of the 2560-wide model, 64 adapters loaded: launch latency
        _lora("lora_1", "lora", 1, 2560, 2560, 16, 64, 1),
        # the drafts of 32 streams, 5 rows each, every stream's own adapter on the target head
        _lora("lora_160_head", "lora", 160, VOCAB, 2560, 16, 32, 5),
        # short ragged prompts through a projection with an odd number of outputs, some without adapter
        _lora("lora_617_ragged", "lora", 617, 1543, 768, 8, 12, 0, "f16", bare=True),
        # the largest prefill chunk through a wide projection, ranks of 64
        _lora("lora_8192_wide", "lora", 8192, 10240, 2560, 64, 8, 0),
        # a small training step of one adapter: launch latency
        _lora("lora_grad_96", "lora_grad", 96, 2560, 2560, 16, 1, 0),
        # a training step of two tenants' adapters on the target head
        _lora("lora_grad_1024_head", "lora_grad", 1024, VOCAB, 2560, 16, 2, 0),
        # a 4-stream verification step, 5 rows each, learned from the usual 20 alternatives
        _distill("distill_20", 20, VOCAB, "bf16", 20),
        # a short prompt over a small odd vocabulary, rows that start at odd addresses
        _distill("distill_617_odd", 617, 32003, "f16", 8, pad=2),
        # the largest chunk
        _distill("distill_4096", 4096, VOCAB, "bf16", 20),
        # a few sampled tokens: launch latency
        _policy("policy_8", 8, VOCAB, "bf16"),
        # tokens sampled under grammar masks, float32 logits
        _policy("policy_256_masked", 256, VOCAB, "f32", masked=True),
        # a chunk of a rollout, float32 logits
        _policy("policy_2048", 2048, VOCAB, "f32"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(["lora", "lora", "lora_grad", "distill", "distill", "policy", "policy"])
    if kind.startswith("lora"):
        grad = kind == "lora_grad"
        depth = 128 * _log_int(rng, 4, 32)
        cols = VOCAB if rng.random() < 0.2 else _log_int(rng, 100, 16384)
        rank = rng.choice([8, 16, 16, 32, 64])
        adapters = rng.choice([1, 2]) if grad else _log_int(rng, 1, 64)
        # no more than the largest case's rows x (columns + depth), and than its rank times that
        size = (1024 * VOCAB if grad else 8192 * 10240) // (cols + depth)
        most = min(8192, size, size * (16 if grad else 64) // rank)
        if not grad and cols == VOCAB:       # the adapters' own bytes
            adapters = min(adapters, 512 // rank)
        return _lora(None, kind, _log_int(rng, 1, max(1, most)), cols, depth, rank, adapters,
                     rng.choice([0, 0, 1, 5]), rng.choice(["bf16", "bf16", "f16"]),
                     bare=rng.random() < 0.3)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    vocab = VOCAB if rng.random() < 0.4 else _log_int(rng, 500, 200000)
    most = 4096 * VOCAB * 2 // ((4 if dtype == "f32" else 2) * vocab)
    rows, pad = _log_int(rng, 1, min(8192, most)), rng.choice([0, 0, 1, 5, 64])
    if kind == "distill":
        return _distill(None, rows, vocab, dtype, rng.choice([1, 5, rng.randint(2, 20), 20, 32]), pad)
    return _policy(None, rows, vocab, dtype, pad, masked=rng.random() < 0.25)


# ---- inputs -------------------------------------------------------------------------------------
def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed(seed * 16 + salt)


def _ids(case, seed):
    """The adapter of each row, on the host: runs of one request's rows."""
    g = torch.Generator().manual_seed(seed * 16 + 3)
    m, n = case["rows"], case["adapters"]
    if case["run"]:
        runs = torch.full((-(-m // case["run"]),), case["run"])
    else:                                    # as many prompts as adapters, twice, of any length
        cuts = torch.randint(1, m + 1, (2 * n,), generator=g).sort().values
        runs = torch.diff(cuts, prepend=torch.zeros(1, dtype=cuts.dtype),
                          append=torch.tensor([m]))
    of = torch.randperm(n, generator=g)[torch.arange(len(runs)) % n]
    if case["bare"]:
        of[torch.rand(len(runs), generator=g) < 0.25] = -1
    return torch.repeat_interleave(of, runs)[:m].to(torch.int32)


def _adapted(case, seed):
    """Hidden states with a few large channels, a projection's output, adapters as they are after some
    training (both factors away from zero), a scale of alpha / rank each, an output's gradient."""
    m, n, k, r, a = (case[x] for x in ("rows", "cols", "depth", "rank", "adapters"))
    dt, g = DTYPES[case["dtype"]], _gen(seed, 1)
    x = torch.randn(m, k, generator=g, device=DEV)
    x *= torch.exp(0.7 * torch.randn(k, generator=g, device=DEV))
    y = torch.randn(m, n, generator=g, device=DEV, dtype=dt)
    A = (torch.randn(a, r, k, generator=g, device=DEV) * k ** -0.5).to(dt)
    B = torch.empty(a, n, r, dtype=dt, device=DEV)
    for i in range(a):
        B[i] = 0.1 * torch.randn(n, r, generator=g, device=DEV)
    s = (16 + 16 * torch.rand(a, generator=g, device=DEV)) / r
    dy = None
    if case["kind"] == "lora_grad":
        dy = torch.randn(m, n, generator=g, device=DEV, dtype=dt) * 2 ** -6
    return x.to(dt), y, A, B, s, _ids(case, seed).to(DEV), dy


def _listed_ids(rows, vocab, g):
    """32 ids of each row, no two the same."""
    wide = vocab // 32
    return torch.randint(wide, (rows, 32), generator=g, device=DEV) + \
        wide * torch.arange(32, device=DEV)


def _logits(case, seed):
    """Logits of a head: a broad bulk, 32 high ones per row, one row in four nearly certain. Returns them with
    the ids of the high ones and by how much those are lifted."""
    r, v = case["rows"], case["vocab"]
    g = _gen(seed, 2)
    buf = torch.empty(r, v + case["pad"], dtype=DTYPES[case["dtype"]], device=DEV)
    logits = buf[:, :v]
    high = _listed_ids(r, v, g)
    lift = 8.0 + 4.0 * torch.rand(r, 32, generator=g, device=DEV)
    lift[::4, 0] = 24.0
    for r0 in range(0, r, ROWS):
        x = 2.5 * torch.randn(min(r, r0 + ROWS) - r0, v, generator=g, device=DEV)
        x.scatter_add_(1, high[r0:r0 + ROWS], lift[r0:r0 + ROWS])
        if case.get("masked"):
            keep = torch.rand(x.shape, generator=g, device=DEV) < 0.002
            keep.scatter_(1, high[r0:r0 + ROWS], True)
            x.masked_fill_(~keep, float("-inf"))
        logits[r0:r0 + ROWS] = x
    return logits, high, lift


def _weight(case, seed):
    """The mean over a batch's tokens with a tenth of them padding; float16 training scales its loss."""
    r = case["rows"]
    live = torch.rand(r, generator=_gen(seed, 4), device=DEV) >= 0.1
    return live.float() * ((2.0 ** 14 if case["dtype"] == "f16" else 1.0) / r)


def _distill_inputs(case, seed):
    logits, high, lift = _logits(case, seed)
    # a teacher that agrees on the high ones, more or less, and has a bulk of its own
    g = _gen(seed, 5)
    t = lift + 1.5 * torch.randn(lift.shape, generator=g, device=DEV)
    bulk = 8.0 + 2.0 * torch.rand(case["rows"], 1, generator=g, device=DEV)
    t = t - torch.logsumexp(torch.cat([t, bulk], 1).double(), 1, keepdim=True).float()
    v, at = torch.sort(t, dim=1, descending=True)
    top = case["top"]
    return (logits, high.gather(1, at)[:, :top].to(torch.int32).contiguous(),
            v[:, :top].contiguous(), _weight(case, seed))


def _lse(logits):
    """logsumexp of each row in 64 bits."""
    return torch.cat([torch.logsumexp(x.double(), 1) for x in logits.split(ROWS)])


def _policy_inputs(case, seed):
    logits, high, _ = _logits(case, seed)
    g = _gen(seed, 6)
    r = case["rows"]
    pick = torch.randint(32, (r, 1), generator=g, device=DEV)
    pick = torch.where(torch.rand(r, 1, generator=g, device=DEV) < 0.4, 0, pick)
    tokens = high.gather(1, pick)[:, 0]
    lp = logits.gather(1, tokens[:, None])[:, 0].double() - _lse(logits)
    # the sampler's policy, a few updates old; a ratio at the very border of the clipped range would
    # go either way by the last bit of a sum, so those few are as they were sampled
    d = 0.15 * torch.randn(r, generator=g, device=DEV, dtype=torch.float64)
    rho = torch.exp(d)
    edge = ((rho - 1 + CLIP[0]).abs() < 1e-3) | ((rho - 1 - CLIP[1]).abs() < 1e-3)
    old = (lp - torch.where(edge, 0.0, d)).float()
    ref = (lp + 0.3 * torch.randn(r, generator=g, device=DEV)).float()
    adv = torch.randn(r, generator=g, device=DEV)
    return logits, tokens, old, adv, ref, _weight(case, seed)


def prepare(case, seed):
    if case["kind"] == "distill":
        return dict(case=case, args=_distill_inputs(case, seed))
    if case["kind"] == "policy":
        return dict(case=case, args=_policy_inputs(case, seed))
    x, y, A, B, s, ids, dy = _adapted(case, seed)
    if own:
        # as a server or a trainer holds them: the stack, and a step's rows laid out once for all layers
        lora = _pkg().lora
        w = lora.LoraStack(A, B, s)
        return dict(case=case, x=x, y=y, dy=dy, w=w, rows=lora.plan_rows(ids, w.n))
    return dict(case=case, x=x, y=y, dy=dy, A=A, B=B, s=s, ids=ids)


# ---- one pass -----------------------------------------------------------------------------------
def _plain_lora(x, y, A, B, s, ids, dy):
    """With every row's product with all adapters, of which its own are kept."""
    n, r, k = A.shape
    xf = x.float()
    keep = torch.where((ids[:, None] == torch.arange(n, device=DEV)), s, 0.0)
    keep = keep.repeat_interleave(r, 1)                              # [rows, n r]
    A2 = A.float().view(n * r, k)
    B2 = B.float().transpose(1, 2).reshape(n * r, -1)
    h = (xf @ A2.T) * keep
    out = (y.float() + h @ B2).to(y.dtype)
    if dy is None:
        return out
    df = dy.float()
    u = (df @ B2.T) * keep
    return dict(out=out, dx=(u @ A2).to(x.dtype), da=(u.T @ xf).view(n, r, k).to(A.dtype),
                db=(h.T @ df).view(n, r, -1).transpose(1, 2).to(B.dtype))


def _softmax(x):
    """Of rows with a finite element: probabilities, and the logarithm of their denominator beside the maximum."""
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(1, keepdim=True)
    return e / z, m + torch.log(z)


def _plain_distill(logits, ids, v, weight):
    x, w, at = logits.float(), weight[:, None], ids.long()
    p, lz = _softmax(x)
    q = torch.exp(v)
    # what is left over is small where a row is nearly certain: by 64 bits, and by the others' own sum
    qr = (1.0 - torch.exp(v.double()).sum(1, keepdim=True)).clamp_(min=0).float()
    lp = x.gather(1, at) - lz
    pr = p.scatter(1, at, 0.0).sum(1, keepdim=True)
    loss = (q * (v - lp)).sum(1, keepdim=True) + \
        torch.where(qr > 0, qr * (torch.log(qr) - torch.log(pr)), 0.0)
    g = p * (1.0 - qr / pr)
    g = g.scatter(1, at, p.gather(1, at) - q)
    return (loss * w)[:, 0], (g * w).to(logits.dtype)


def _plain_policy(logits, tokens, old, adv, ref, weight):
    x, t = logits.float(), tokens[:, None]
    p, lz = _softmax(x)
    lp = (x.gather(1, t) - lz)[:, 0]
    rho = torch.exp(lp - old)
    held = torch.clamp(rho, 1 - CLIP[0], 1 + CLIP[1])
    d = ref - lp
    loss = -torch.minimum(rho * adv, held * adv) + KL * (torch.exp(d) - d - 1)
    g = torch.where(rho * adv <= held * adv, -rho * adv, 0.0) + KL * (1 - torch.exp(d))
    # 1 - p of the token as the others' sum: it is small where the token is nearly certain
    others = p.scatter(1, t, 0.0).sum(1, keepdim=True)
    grad = (-p).scatter(1, t, others) * (g * weight)[:, None]
    # a row of no weight has no log probability either
    return weight * loss, torch.where(weight != 0, lp, 0.0), grad.to(logits.dtype)


def _parts(f, args):
    """f over ROWS rows at a time, joined."""
    n = args[0].shape[0]
    if n <= ROWS:
        return f(*args)
    out = [f(*[a[r:r + ROWS] for a in args]) for r in range(0, n, ROWS)]
    return tuple(torch.cat(t) for t in zip(*out))


def run(state):
    kind = state["case"]["kind"]
    if kind == "distill":
        if own:
            loss, grad = _pkg().losses.distill_top_grad(*state["args"])
        else:
            loss, grad = _parts(_plain_distill, state["args"])
        return dict(loss=loss, grad=grad)
    if kind == "policy":
        if own:
            (loss, lp), grad = _pkg().losses.policy_loss_grad(*state["args"], clip=CLIP, kl=KL)
        else:
            loss, lp, grad = _parts(_plain_policy, state["args"])
        return dict(loss=loss, logprob=lp, grad=grad)
    if not own:
        return _plain_lora(*[state[k] for k in ("x", "y", "A", "B", "s", "ids", "dy")])
    lora, x, w, rows = _pkg().lora, state["x"], state["w"], state["rows"]
    if kind == "lora":
        return lora.add_lora(state["y"], x, w, rows)
    hidden = torch.empty(x.shape[0], w.rank, device=x.device)
    out = lora.add_lora(state["y"], x, w, rows, hidden=hidden)
    dx, da, db = lora.add_lora_grad(state["dy"], x, w, rows, hidden)
    return dict(out=out, dx=dx, da=da, db=db)


# ---- what a pass has to do ----------------------------------------------------------------------
def work(case):
    if case["kind"] in ("distill", "policy"):
        r, v = case["rows"], case["vocab"]
        size = 4 if case["dtype"] == "f32" else 2
        row = 8 * case["top"] + 8 if case["kind"] == "distill" else 8 + 4 * 6
        # an element: the difference to the maximum, the exponential, the sum, the gradient's factor
        return dict(bytes=r * (2 * v * size + row), flops=4 * r * v)
    m, n, k, r = case["rows"], case["cols"], case["depth"], case["rank"]
    used = min(case["adapters"], -(-m // case["run"]) if case["run"] else m)
    nbytes = 2 * m * k + 4 * m * n + 2 * used * r * (n + k) + 4 * m
    flops = 2 * m * r * (n + k)
    if case["kind"] == "lora_grad":          # dy; dx and the gradients of the whole stack
        nbytes += 2 * m * n + 2 * m * k + 2 * case["adapters"] * r * (n + k)
        flops *= 3
    return dict(bytes=nbytes, flops=flops)


# ---- the same in 64 bits ------------------------------------------------------------------------
def _exact_lora(case, seed):
    """An adapter at a time, over its own rows."""
    x, y, A, B, s, ids, dy = _adapted(case, seed)
    out = y.double()
    grads = None
    if dy is not None:
        grads = dict(dx=torch.zeros(x.shape, dtype=torch.float64, device=DEV),
                     da=torch.zeros(A.shape, dtype=torch.float64, device=DEV),
                     db=torch.zeros(B.shape, dtype=torch.float64, device=DEV))
    for a in ids.unique().tolist():
        if a < 0:
            continue
        at = (ids == a).nonzero()[:, 0]
        xa, Aa, Ba = x[at].double(), A[a].double(), B[a].double()
        h = s[a].double() * (xa @ Aa.T)
        out[at] += h @ Ba.T
        if dy is not None:
            d = dy[at].double()
            u = s[a].double() * (d @ Ba)
            grads["dx"][at] = u @ Aa
            grads["da"][a] = u.T @ xa
            grads["db"][a] = d.T @ h
    return out if dy is None else dict(out=out, **grads)


def _exact_distill(logits, ids, v, weight):
    lp = torch.log_softmax(logits.double(), 1)
    v, at, w = v.double(), ids.long(), weight.double()[:, None]
    qr = (1.0 - torch.exp(v).sum(1, keepdim=True)).clamp_(min=0)
    others = lp.scatter(1, at, float("-inf"))
    lr = torch.logsumexp(others, 1, keepdim=True)
    loss = (torch.exp(v) * (v - lp.gather(1, at))).sum(1, keepdim=True) + torch.special.xlogy(qr, qr) - qr * lr
    target = torch.exp(others - lr) * qr
    target.scatter_(1, at, torch.exp(v))
    return (loss * w)[:, 0], (torch.exp(lp) - target) * w


def _exact_policy(logits, tokens, old, adv, ref, weight):
    logp = torch.log_softmax(logits.double(), 1)
    lp = logp.gather(1, tokens[:, None])[:, 0]
    old, adv, ref, w = old.double(), adv.double(), ref.double(), weight.double()
    gain, d = torch.exp(lp - old) * adv, ref - lp
    bound = torch.where(adv >= 0, 1 + CLIP[1], 1 - CLIP[0]) * adv
    loss = torch.maximum(-gain, -bound) + KL * (torch.expm1(d) - d)
    g = w * (torch.where(gain <= bound, -gain, 0.0) - KL * torch.expm1(d))
    grad = -torch.exp(logp)
    grad.scatter_(1, tokens[:, None], -torch.expm1(lp)[:, None])
    return w * loss, torch.where(w != 0, lp, 0.0), grad * g[:, None]


def exact(case, seed):
    if case["kind"] == "distill":
        loss, grad = _parts(_exact_distill, _distill_inputs(case, seed))
        return dict(loss=loss, grad=grad)
    if case["kind"] == "policy":
        loss, lp, grad = _parts(_exact_policy, _policy_inputs(case, seed))
        return dict(loss=loss, logprob=lp, grad=grad)
    return _exact_lora(case, seed)
