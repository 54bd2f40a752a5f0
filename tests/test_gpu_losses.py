"""losses.policy_loss and losses.distill_top against float64: losses, log probabilities and gradients within
derived limits, over types, strides, masks and row counts on both sides of the kernels' choice."""
from __future__ import annotations

from importlib import import_module

import pytest

from conftest import gpu_case

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DEV = "cuda"
NINF, INF, NAN = float("-inf"), float("inf"), float("nan")
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CLIP = (0.2, 0.28)


@pytest.fixture(scope="module")
def losses(pkg):
    return import_module(pkg.__name__ + ".losses")


STEP = 2.0 ** -24
# A sum of exponentials, relative. A term: its argument's rounding and that of log2(e) / T, half a step each of at
# most 150, times ln 2 (208 steps), the exponential (2). A thread's chunk: 32 additions; chunks: at most 62, each
# with a rescaling by an exponential (3, and the 208 once over all, as their arguments add up to 150 at most);
# 6 + 8 additions and two such factors over wave and workgroup, 6 and one over segments.
SUM = (210 + 32 + 62 * 4 + 208 + 14 + 2 * 210 + 6 + 210) * STEP
# a log probability: the sum under a logarithm, (x - m) / T, its product, the logarithm and their difference
LP = SUM + 4 * STEP
# an exponential below the smallest normal float is 0: the instruction gives no smaller ones
TINY = 2.0 ** -126


def softmax(x, T, ids):
    """In float64, of rows with a finite logit: ln p, ln of the sum of p over the unlisted."""
    lp = torch.log_softmax(x.double() / T, 1)
    others = lp.clone()
    others.scatter_(1, ids, NINF)
    return lp, others, torch.logsumexp(others, 1, keepdim=True)


def near(got, want, limit, what):
    assert got.dtype != torch.float64
    bad = ~((got.double() - want).abs() <= limit)
    assert not bad.any(), (what, got[bad][:4], want[bad][:4], bad.sum(), bad.nonzero()[:4])


def near_grad(got, want, limit):
    """limit before the rounding to the type: half a step, or half of the smallest value above 0."""
    t = torch.finfo(got.dtype)
    near(got, want, limit + t.eps / 2 * (want.abs() + limit) + t.smallest_normal * t.eps / 2, "grad")


def exact_policy(x, tok, old, adv, ref, w, clip, kl, T):
    t = tok.long()[:, None]
    logp, _, rest = softmax(x, T, t)
    lp = logp.gather(1, t)[:, 0]
    old, adv, w = old.double(), adv.double(), w.double()
    rho = torch.exp(lp - old)
    gain, bound = rho * adv, rho.clamp(1 - clip[0], 1 + clip[1]) * adv
    loss, g = -torch.minimum(gain, bound), torch.where(gain <= bound, -gain, 0.0)
    err = LP * (1 + lp.abs()) + 4 * STEP * (1 + (lp - old).abs())     # of lp - old, and so of rho
    loss_err, g_err = gain.abs() * err, gain.abs() * err
    if kl:
        d = ref.double() - lp
        loss = loss + kl * (torch.expm1(d) - d)
        g = g - kl * torch.expm1(d)
        e = kl * (torch.exp(d) + 1) * (LP * (1 + lp.abs()) + 6 * STEP * (1 + d.abs()))
        loss_err, g_err = loss_err + e, g_err + e
    grad = -torch.exp(logp)
    grad.scatter_(1, t, torch.exp(rest))
    size = grad.abs()
    f = (w / T)[:, None]
    return (w * loss, w.abs() * (loss_err + 8 * STEP * loss.abs()), torch.where(w != 0, lp, 0.0),
            LP * (1 + lp.abs()), f * g[:, None] * grad,
            f.abs() * (size * ((2 * SUM + 16 * STEP) * g.abs() + g_err)[:, None] + TINY * g.abs()[:, None]))


def exact_distill(x, ids, v, w, rest, T):
    """For ids that differ and lie in range."""
    at = ids.long()
    lp, others, lr = softmax(x, T, at)
    v, w = v.double(), w.double()
    if rest:
        ln_q, q = v, torch.exp(v)
        left = 1 - q.sum(1, keepdim=True)
    else:
        ln_q = torch.log_softmax(v / T, 1)
        q = torch.exp(ln_q)
        left = torch.zeros_like(lr)
    total = torch.where(left < 0, q.sum(1, keepdim=True), 1.0)
    left = left.clamp(min=0)
    left = torch.where(lr == NINF, 0.0, left)
    lpt = lp.gather(1, at)
    cost = torch.where(q > 0, q * (ln_q - lpt), 0.0)
    loss = cost.sum(1, keepdim=True)
    tail = torch.where(left > 0, left * (torch.log(left) - lr), 0.0)
    # the teacher's own sums: the exponential's 2 steps and its argument's, 32 additions, a logarithm
    q_err = 40 * STEP
    loss_err = (q * (LP * (1 + lpt.abs().clamp(max=1e4)) + 40 * STEP * (1 + ln_q.abs().clamp(max=1e4)))).sum(1)
    loss_err = loss_err + 40 * STEP * (cost.abs().sum(1) + tail.abs()[:, 0])
    # what is left may be off by q_err, whatever it is
    loss_err = loss_err + torch.where(lr[:, 0] > NINF, q_err * (30 + lr[:, 0].abs()) + left[:, 0] * LP, 0.0)
    share = torch.where(lr == NINF, 0.0, left / torch.exp(lr))
    p = torch.exp(lp)
    grad = p * (total - share)
    err = p * ((2 * SUM + 16 * STEP) * (total + share) + torch.where(lr == NINF, 0.0, q_err / torch.exp(lr)) + q_err)
    err = err + TINY * (total + share)
    pt = p.gather(1, at)
    grad.scatter_(1, at, total * pt - q)
    # without a rest the exponential's argument (v - max) / T is off by three half steps of itself, which is at
    # most ln q in size
    far = 0.0 if rest else 4 * STEP * ln_q.abs().clamp(max=1e4)
    err.scatter_(1, at, (2 * SUM + 16 * STEP) * pt + q_err * (pt + q) + far * q + TINY)
    f = (w / T)[:, None]
    loss = (loss + tail)[:, 0]
    return w * loss, w.abs() * loss_err, f * grad, f.abs() * err


def rows_of(R, V, dtype, seed, pad=0, offset=0, spread=2.5):
    """Logits with a few high ones a row, every fourth row nearly certain, between columns of NaN."""
    g = torch.Generator(DEV).manual_seed(seed)
    buf = torch.full((R * (V + pad) + offset,), NAN, dtype=TYPES[dtype], device=DEV)
    x = buf[offset:].view(R, V + pad)[:, :V]
    f = spread * torch.randn(R, V, generator=g, device=DEV)
    high = torch.randint(V, (R, 5), generator=g, device=DEV)
    f.scatter_add_(1, high, 8 + 4 * torch.rand(R, 5, generator=g, device=DEV))
    f[::4, V // 2] = 40.0
    x.copy_(f)
    tok = torch.where(torch.rand(R, generator=g, device=DEV) < 0.5, x.argmax(1), high[:, 0])
    return x, tok


def policy_of(x, tok, seed, clip=CLIP, T=1.0):
    """The other inputs, with no ratio next to the clipped range's ends."""
    g = torch.Generator(DEV).manual_seed(seed + 1)
    R = x.shape[0]
    lp = torch.log_softmax(x.double() / T, 1).gather(1, tok.long()[:, None])[:, 0]
    d = 0.3 * torch.randn(R, generator=g, device=DEV, dtype=torch.float64)
    rho = torch.exp(d)
    d[((rho - 1 + clip[0]).abs() < 5e-3) | ((rho - 1 - clip[1]).abs() < 5e-3)] = 0.0
    old = (lp - d).float()
    ref = (lp + 0.3 * torch.randn(R, generator=g, device=DEV)).float()
    adv = torch.randn(R, generator=g, device=DEV)
    w = torch.rand(R, generator=g, device=DEV)
    w[w < 0.1] = 0.0
    return old, adv, ref, w


def teacher_of(x, top, seed):
    """Different ids of each row, half of them its highest, and log probabilities that leave a rest."""
    g = torch.Generator(DEV).manual_seed(seed + 2)
    R, V = x.shape
    score = x.float() + 6 * torch.randn(R, V, generator=g, device=DEV)
    score[score.isnan()] = NINF
    ids = score.topk(top, dim=1).indices.int()
    v = torch.randn(R, top + 1, generator=g, device=DEV) * 2
    v[::3, 0] += 20                                                # a nearly certain teacher
    v = torch.log_softmax(v.double(), 1)[:, :top].float().contiguous()
    w = torch.rand(R, generator=g, device=DEV)
    w[w < 0.1] = 0.0
    return ids.contiguous(), v, w


def check_policy(out, grad, x, tok, old, adv, ref, w, clip=CLIP, kl=0.05, T=1.0):
    loss, loss_err, lp, lp_err, want, err = exact_policy(x, tok, old, adv, ref, w, clip, kl, T)
    near(out.loss, loss, loss_err, "loss")
    near(out.logprob, lp, lp_err, "logprob")
    near_grad(grad, want, err)


def check_distill(loss, grad, x, ids, v, w, rest=True, T=1.0):
    want, loss_err, g, err = exact_distill(x, ids, v, w, rest, T)
    near(loss, want, loss_err, "loss")
    near_grad(grad, g, err)


SIZES = [(3, 1, 0, 0), (5, 2, 1, 1), (4, 5, 0, 3), (7, 33, 2, 0), (9, 255, 0, 1), (2, 256, 0, 0),
         (6, 2047, 3, 2), (6, 4097, 7, 1), (4, 16384, 0, 0), (3, 16391, 5, 3), (17, 32003, 2, 5),
         (2, 65537, 0, 1), (1, 151936, 0, 0), (20, 151936, 0, 0), (255, 9001, 0, 0), (256, 9001, 0, 0),
         (300, 50001, 3, 1), (2, 499999, 1, 1), (1, 500000, 0, 0), (40000, 9, 0, 0),
         (200, 1020, 1, 1), (200, 1030, 0, 0), (1000, 2040, 3, 7), (1000, 2049, 0, 0), (300, 4093, 5, 2), (400, 8185, 3, 1),
         (200, 8200, 0, 0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,pad,offset", SIZES)
def test_policy(losses, dtype, R, V, pad, offset):
    x, tok = rows_of(R, V, dtype, R + V, pad, offset)
    old, adv, ref, w = policy_of(x, tok, R)
    gpu_case(f"policy {dtype} R={R} V={V} pad={pad} offset={offset}")
    out, grad = losses.policy_loss_grad(x, tok, old, adv, ref, w, clip=CLIP, kl=0.05)
    only = losses.policy_loss(x, tok.int(), old, adv, ref, w, clip=CLIP, kl=0.05)
    torch.cuda.synchronize()
    check_policy(out, grad, x, tok, old, adv, ref, w)
    assert torch.equal(only.loss, out.loss) and torch.equal(only.logprob, out.logprob)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,pad,offset", SIZES)
def test_distill(losses, dtype, R, V, pad, offset):
    for top in sorted({1, min(V, 7), min(V, 20), min(V, 32)}):
        x, _ = rows_of(R, V, dtype, R + V, pad, offset)
        ids, v, w = teacher_of(x, top, R)
        gpu_case(f"distill {dtype} R={R} V={V} pad={pad} offset={offset} top={top}")
        for rest in (True, False):
            loss, grad = losses.distill_top_grad(x, ids, v, w, rest=rest)
            only = losses.distill_top(x, ids, v, w, rest=rest)
            torch.cuda.synchronize()
            check_distill(loss, grad, x, ids, v, w, rest)
            assert torch.equal(only, loss)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [0.3, 0.7, 2.0, 50.0])
@pytest.mark.parametrize("R", [9, 260])
def test_temperatures(losses, dtype, T, R):
    x, tok = rows_of(R, 5003, dtype, 3, 1, 1)
    old, adv, ref, w = policy_of(x, tok, R, T=T)
    gpu_case(f"losses {dtype} T={T} R={R}")
    out, grad = losses.policy_loss_grad(x, tok, old, adv, ref, w, clip=CLIP, kl=0.2, temperature=T)
    torch.cuda.synchronize()
    check_policy(out, grad, x, tok, old, adv, ref, w, kl=0.2, T=T)
    ids, v, w = teacher_of(x, 20, R)
    for rest in (True, False):
        loss, grad = losses.distill_top_grad(x, ids, v, w, rest=rest, temperature=T)
        torch.cuda.synchronize()
        check_distill(loss, grad, x, ids, v, w, rest, T)


@pytest.mark.parametrize("clip", [(0.0, 0.0), (1.0, 5.0), (0.1, 0.1)])
def test_without_kl_weight_or_reference(losses, clip):
    x, tok = rows_of(300, 3001, "f32", 5)
    old, adv, ref, _ = policy_of(x, tok, 5, clip)
    one = torch.ones(300, device=DEV)
    if clip == (0.0, 0.0):                   # every ratio is at the border then, unless it is far from it
        old = old - 0.5
    gpu_case(f"policy clip={clip}")
    out, grad = losses.policy_loss_grad(x, tok, old, adv, clip=clip)
    same, _ = losses.policy_loss_grad(x, tok, old, adv, ref, one, clip=clip)
    torch.cuda.synchronize()
    check_policy(out, grad, x, tok, old, adv, None, one, clip, 0.0)
    assert torch.equal(out.loss, same.loss)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,offset", [(8, 50, 0), (8, 3000, 1), (8, 70001, 3), (264, 3000, 1)])
def test_masked_rows(losses, dtype, R, V, offset):
    """-inf nearly everywhere, the type's lowest value in its place, alone and beside -inf; listed tokens alone
    left, and none."""
    low = torch.finfo(TYPES[dtype]).min
    g = torch.Generator(DEV).manual_seed(V)
    buf = torch.empty(R * V + offset, dtype=TYPES[dtype], device=DEV)
    x = buf[offset:].view(R, V)
    x.copy_(torch.randn(R, V, generator=g, device=DEV) * 3)
    many = torch.rand(R, V, generator=g, device=DEV) < 0.9
    x[0::8] = torch.where(many[0::8], torch.tensor(NINF, dtype=x.dtype, device=DEV), x[0::8])
    x[1::8] = NINF
    x[2::8] = low
    x[3::8] = torch.where(many[3::8], torch.tensor(low, dtype=x.dtype, device=DEV), x[3::8])
    x[4::8, ::2] = NINF
    x[4::8, 1::2] = low
    x[5::8] = low
    x[5::8, 7] = 2.0
    x[6::8] = NINF
    ids = torch.stack([torch.randperm(V, generator=g, device=DEV)[:5] for _ in range(R)]).int()
    ids[4::8] = torch.arange(1, 11, 2, device=DEV, dtype=torch.int32)   # (listed ones at -inf: the next test)
    live = torch.randn(R, 5, generator=g, device=DEV)
    for r in range(R):                                              # the listed ones stay
        if r % 8 not in (2, 4, 5, 6):
            x[r, ids[r].long()] = live[r].to(x.dtype)
    tok = ids[:, 0].long()
    some = [r for r in range(R) if r % 8 != 6]
    none = [r for r in range(R) if r % 8 == 6]
    v = torch.log_softmax(torch.randn(R, 6, generator=g, device=DEV), 1)[:, :5].contiguous()
    lp = torch.log_softmax(x.double(), 1).gather(1, tok[:, None])[:, 0]
    lp[none] = -1.0
    # (a token beside a far higher one has a log probability that leaves no ratio: such rows are sampled so)
    old, adv = (lp.float() - 0.1), torch.randn(R, generator=g, device=DEV)
    w = torch.rand(R, generator=g, device=DEV) + 0.1
    gpu_case(f"losses masks {dtype} R={R} V={V}")
    out, grad = losses.policy_loss_grad(x, tok, old, adv, None, w, clip=CLIP)
    loss, dgrad = losses.distill_top_grad(x, ids, v, w)
    loss2, dgrad2 = losses.distill_top_grad(x, ids, v, w, rest=False)
    torch.cuda.synchronize()
    for t in (grad, dgrad, dgrad2):
        assert (t[none] == 0).all()
    assert (out.logprob[none] == NINF).all() and (loss[none] == INF).all() and (loss2[none] == INF).all()
    sane = [r for r in some if r % 8 != 5]
    pick = lambda *ts: [t[sane] for t in ts]                          # noqa: E731
    out = type(out)(*pick(*out))
    check_policy(out, grad[sane], *pick(x, tok, old, adv), None, w[sane], kl=0.0)
    check_distill(loss[sane], dgrad[sane], *pick(x, ids, v, w))
    check_distill(loss2[sane], dgrad2[sane], *pick(x, ids, v, w), rest=False)
    far = [r for r in some if r % 8 == 5]                           # one token alone has all
    assert torch.isfinite(grad[far]).all() and torch.isfinite(dgrad[far]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R", [12, 300])
def test_listed_tokens_at_minus_infinity(losses, dtype, R):
    """What the formula gives: a ratio of 0; an infinite divergence whose gradient is finite."""
    x, tok = rows_of(R, 3001, dtype, 9, 1, 1)
    ids, v, w = teacher_of(x, 6, 9)
    w = w + 0.1
    tok = ids[:, 2].long()
    x.scatter_(1, tok[:, None], NINF)
    adv = torch.randn(R, device=DEV)
    gpu_case(f"losses listed -inf {dtype}")
    out, grad = losses.policy_loss_grad(x, tok, torch.full((R,), -2.0, device=DEV), adv, None, w, clip=CLIP)
    loss, dgrad = losses.distill_top_grad(x, ids, v, w)
    torch.cuda.synchronize()
    assert (out.logprob == NINF).all() and (grad == 0).all()
    near(out.loss, -(w * torch.minimum(0 * adv, 0.8 * adv)).double(), 4 * STEP * (w * adv).abs(), "loss")
    assert (loss == INF).all()
    want = exact_distill(x, ids, v, w, True, 1.0)
    near_grad(dgrad, want[2], want[3])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R", [16, 300])
@pytest.mark.parametrize("V", [9, 3000, 70001])
def test_nan_inf_padding_and_ids_out_of_range(losses, dtype, R, V):
    x, tok = rows_of(R, V, dtype, V, 1, 1)
    old, adv, ref, w = policy_of(x, tok, V)
    ids, v, _ = teacher_of(x, 4, V)
    w = w + 0.1
    clean = x.clone()
    for r, (j, bad) in {1: (0, NAN), 3: (V - 1, INF), 4: (V // 2, -NAN), 5: (int(tok[5]), NAN),
                        6: (int(ids[6, 1]), INF)}.items():
        x[r, j] = bad
    x[8] = NINF
    x[8, V // 2] = NAN
    broken = [1, 3, 4, 5, 6, 8, 9]
    tok[9] = V
    ids[9, 2] = V + 5
    tok[10], ids[10] = -1, -1                                        # none
    x[11], w[11] = NAN, 0.0                                          # padding may hold anything
    x[12], tok[12], w[12] = INF, -7, 2.0
    ids[13, 1:3], v[13, 1:3] = -1, NAN                               # (as a scored NaN row's alternatives)
    gpu_case(f"losses NaN {dtype} R={R} V={V}")
    out, grad = losses.policy_loss_grad(x, tok, old, adv, ref, w, clip=CLIP, kl=0.05)
    w[12] = 0.0
    loss, dgrad = losses.distill_top_grad(x, ids, v, w)
    torch.cuda.synchronize()
    for t in (out.loss, out.logprob, grad, loss, dgrad):
        assert t[broken].isnan().all()
        assert (t[[11, 12]] == 0).all()
    for t in (out.loss, out.logprob, grad, loss, dgrad):
        assert (t[10] == 0).all()
    fine = [r for r in range(R) if r not in broken + [10, 11, 12, 13]]
    pick = lambda *ts: [t[fine] for t in ts]                          # noqa: E731
    check_policy(type(out)(*pick(*out)), grad[fine], *pick(x, tok, old, adv, ref, w))
    check_distill(loss[fine], dgrad[fine], *pick(x, ids, v, w))
    keep = [0, 3]
    check_distill(loss[13:14], dgrad[13:14], clean[13:14], ids[13:14, keep], v[13:14, keep], w[13:14])


def test_an_id_listed_twice(losses):
    x, _ = rows_of(300, 2001, "f32", 3)
    ids, v, w = teacher_of(x, 6, 3)
    twice = torch.cat([ids, ids[:, 2:3], ids[:, 2:3]], 1).contiguous()
    half = v.clone()
    part = v[:, 2:3].double().exp()
    vs = torch.cat([torch.cat([v[:, :2], (part * 0.5).log().float(), v[:, 3:]], 1),
                    (part * 0.3).log().float(), (part * 0.2).log().float()], 1).contiguous()
    gpu_case("distill with an id listed three times")
    _, want = losses.distill_top_grad(x, ids, half, w)
    for rows in (slice(0, 300), slice(0, 9)):
        loss, grad = losses.distill_top_grad(x[rows], twice[rows].contiguous(), vs[rows].contiguous(),
                                             w[rows].contiguous())
        torch.cuda.synchronize()
        # the same probabilities, summed in another order, of float32 logarithms near -20 at most
        torch.testing.assert_close(grad, want[rows], rtol=2 * SUM, atol=200 * STEP)


@pytest.mark.parametrize("R", [5, 300])
def test_probabilities_of_more_than_one(losses, R):
    """A teacher's certain token at 0 after rounding, or a little above: the gradient is p - q. Above by more: S p - q."""
    x = torch.zeros(R, 2001, device=DEV)
    x[:, 7] = 30.0
    ids = torch.tensor([[7, 3]], dtype=torch.int32, device=DEV).expand(R, 2).contiguous()
    w = torch.ones(R, device=DEV)
    p = torch.softmax(x.double(), 1)[0]
    for top in (0.0, 1e-6, 1e-5, 1e-4, 0.3):
        v = torch.tensor([[top, -12.0]], device=DEV).expand(R, 2).contiguous()
        gpu_case(f"distill R={R} with a log probability of {top}")
        loss, grad = losses.distill_top_grad(x, ids, v, w)
        torch.cuda.synchronize()
        q = v[0].double().exp()
        S = q.sum() if q.sum() > 1 + 2.0 ** -16 else 1.0               # (at 1e-5 it is: e^-12 = 0.6e-5 comes on top)
        want = S * p
        want[7] -= q[0]
        want[3] -= q[1]
        # at 7 an exponential, S, their product and difference (2, 3, 1 and 1 steps of at most 1.4), at 3 the exponential
        # alone, the others an exponential of -30
        limit = 220 * STEP * p
        limit[7], limit[3] = 10 * STEP, 10 * STEP * q[1]
        near(grad, want.expand(R, -1), limit, "grad")
        cost = q * (v[0].double() - torch.log(p[[7, 3]]))
        near(loss, cost.sum().expand(R), 10 * STEP * cost.abs().sum(), "loss")


def test_where_everything_is_listed(losses):
    x, _ = rows_of(300, 20, "f32", 3)
    ids = torch.stack([torch.randperm(20, device=DEV) for _ in range(300)]).int()
    v = torch.log_softmax(torch.randn(300, 20, device=DEV), 1)
    w = torch.rand(300, device=DEV)
    gpu_case("distill with the whole vocabulary listed")
    loss, grad = losses.distill_top_grad(x, ids, v, w)
    torch.cuda.synchronize()
    check_distill(loss, grad, x, ids, v, w)
    lp = torch.log_softmax(x.double(), 1)
    q = torch.zeros_like(lp).scatter_(1, ids.long(), v.double().exp())
    near_grad(grad, w[:, None] * (lp.exp() - q), w[:, None] * (2 * SUM + 60 * STEP) * (lp.exp() + q))


@pytest.mark.parametrize("scale", [1e-30, 1e4, 1e30, 3e38])
@pytest.mark.parametrize("R", [6, 258])
def test_large_and_small_logits(losses, scale, R):
    g = torch.Generator(DEV).manual_seed(1)
    x = (torch.rand(R, 9000, generator=g, device=DEV) * 2 - 1) * scale
    x[1] = x[1].abs()
    x[2] = -x[2].abs() - scale * 0.1
    x[3] = scale
    x[4] = -scale
    tok = x.argmax(1)
    old, adv, ref, w = policy_of(x, tok, 1)
    gpu_case(f"losses scale={scale}")
    out, grad = losses.policy_loss_grad(x, tok, old, adv, ref, w, clip=CLIP, kl=0.05)
    torch.cuda.synchronize()
    check_policy(out, grad, x, tok, old, adv, ref, w)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R", [20, 300])
def test_into_a_buffer_and_in_place(losses, dtype, R):
    """Rows of another stride and phase, nothing written beside them; the logits' own place; expanded logits."""
    x, tok = rows_of(R, 20001, dtype, 2, 3, 1)
    old, adv, ref, w = policy_of(x, tok, 2)
    ids, v, _ = teacher_of(x, 20, 2)
    gpu_case(f"losses out= {dtype} R={R}")
    want = losses.policy_loss_grad(x, tok, old, adv, ref, w, kl=0.1)
    wantd = losses.distill_top_grad(x, ids, v, w)
    for off, pad in ((0, 0), (1, 2), (5, 3), (7, 0)):
        buf = torch.full((R * (20001 + pad) + off + 16,), 7.0, dtype=x.dtype, device=DEV)
        out = buf[off:off + R * (20001 + pad)].view(R, -1)[:, :20001]
        rest = torch.ones_like(buf, dtype=torch.bool)
        rest[off:off + R * (20001 + pad)].view(R, -1)[:, :20001] = False
        got = losses.policy_loss_grad(x, tok, old, adv, ref, w, kl=0.1, out=out)
        assert got[1] is out and torch.equal(out, want[1]) and torch.equal(got[0].loss, want[0].loss)
        losses.distill_top_grad(x, ids, v, w, out=out)
        assert torch.equal(out, wantd[1]) and (buf[rest] == 7.0).all()
    for fn, args, kw in ((losses.policy_loss_grad, (tok, old, adv, ref, w), dict(kl=0.1)),
                         (losses.distill_top_grad, (ids, v, w), {})):
        buf = torch.full((R, 20005), 3.0, dtype=x.dtype, device=DEV)
        y = buf[:, 1:20002]
        y.copy_(x)
        want = fn(y, *args, **kw)
        assert torch.equal(y, x)
        got = fn(y, *args, out=y, **kw)
        torch.cuda.synchronize()
        assert torch.equal(y, want[1])
        assert torch.equal(got[0].loss, want[0].loss) if kw else torch.equal(got[0], want[0])
        assert (buf[:, 0] == 3.0).all() and (buf[:, 20002:] == 3.0).all()
    one = x[:1].expand(R, -1)
    o2, a2, r2, w2 = policy_of(one, tok, 2)
    out, grad = losses.policy_loss_grad(one, tok, o2, a2, r2, w2, clip=CLIP, kl=0.05)
    torch.cuda.synchronize()
    check_policy(out, grad, one, tok, o2, a2, r2, w2)


def test_no_rows(losses):
    x = torch.empty(0, 100, device=DEV)
    e, i = torch.empty(0, device=DEV), torch.empty(0, dtype=torch.int64, device=DEV)
    out, grad = losses.policy_loss_grad(x, i, e, e)
    assert out.loss.shape == (0,) and grad.shape == (0, 100)
    loss = losses.distill_top(x.requires_grad_(), torch.empty(0, 3, dtype=torch.int32, device=DEV),
                              torch.empty(0, 3, device=DEV))
    loss.sum().backward()
    assert x.grad.shape == (0, 100)


def test_logits_past_2_to_31_elements(losses):
    R, V = 14200, 151936                                             # 2.16e9 of them, 4.3 GB
    x = torch.zeros(R, V, dtype=torch.bfloat16, device=DEV)
    y, tok = rows_of(30, V, "bf16", 3)
    x[-30:] = y
    old, adv, ref, w = policy_of(y, tok, 3)
    full = lambda t, v=0: torch.cat([torch.full((R - 30,), v, dtype=t.dtype, device=DEV), t])   # noqa: E731
    gpu_case("losses past 2^31 elements")
    out, grad = losses.policy_loss_grad(x, full(tok, 5), full(old), full(adv), full(ref), full(w, 0),
                                        clip=CLIP, kl=0.05)
    torch.cuda.synchronize()
    check_policy(type(out)(*[t[-30:] for t in out]), grad[-30:], y, tok, old, adv, ref, w)
    assert (grad[:1000] == 0).all()


@pytest.mark.parametrize("R", [5, 256])
def test_gradients_against_differences(losses, R):
    """Central differences of the losses along random directions, float32 of 37 logits. The loss's own error (LP
    of some 5) over a step of 2^-6, and the third derivative's (below 10 on unit directions) times h^2 / 6."""
    x, tok = rows_of(R, 37, "f32", 4, spread=1.0)
    x[::4, 18] = 3.0
    old, adv, ref, w = policy_of(x, tok, 4, (0.5, 0.5))
    w = w + 0.2
    ids, v, _ = teacher_of(x, 6, 4)
    h = 2.0 ** -6
    limit = 8 * LP / h + 10 * h * h / 6 * 4
    g = torch.Generator(DEV).manual_seed(5)
    kw = dict(clip=(1.0, 1e4), kl=0.3)                               # (no border within a step)
    gpu_case("losses against differences")
    _, pg = losses.policy_loss_grad(x, tok, old, adv, ref, w, **kw)
    dg = [losses.distill_top_grad(x, ids, v, w, rest=rest)[1] for rest in (True, False)]
    for _ in range(5):
        d = torch.randn(R, 37, generator=g, device=DEV)
        d /= d.norm(dim=1, keepdim=True)
        for grad, f in ((pg, lambda y: losses.policy_loss(y, tok, old, adv, ref, w, **kw).loss),
                        (dg[0], lambda y: losses.distill_top(y, ids, v, w)),
                        (dg[1], lambda y: losses.distill_top(y, ids, v, w, rest=False))):
            by = (f(x + h * d).double() - f(x - h * d).double()) / (2 * h)
            got = (grad.double() * d.double()).sum(1)
            assert ((by - got).abs() <= limit * (1 + got.abs())).all(), (by - got).abs().max()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R", [7, 300])
def test_autograd(losses, dtype, R):
    x, tok = rows_of(R, 3001, dtype, 6, 1, 1)
    old, adv, ref, w = policy_of(x, tok, 6)
    ids, v, _ = teacher_of(x, 9, 6)
    want = losses.policy_loss_grad(x, tok, old, adv, ref, w, kl=0.1)[1]
    wantd = losses.distill_top_grad(x, ids, v, w)[1]
    gpu_case(f"losses autograd {dtype}")
    leaf = x.detach().requires_grad_()
    out = losses.policy_loss(leaf, tok, old, adv, ref, w, kl=0.1)
    assert not out.logprob.requires_grad
    out.loss.sum().backward()
    assert torch.equal(leaf.grad, want)
    losses.distill_top(leaf, ids, v, w).sum().backward()             # adds to what is there
    assert torch.equal(leaf.grad, want + wantd)
    # other gradients than 1, row by row, and a mean's
    by = torch.randn(R, device=DEV)
    by[0], by[1] = 1.0, 0.0
    (got,) = torch.autograd.grad(losses.distill_top(leaf, ids, v, w), leaf, by)
    # (one rounding to the type, with or without one to float32 before it)
    product = wantd.double() * by.double()[:, None]
    near_grad(got, product, STEP * product.abs())
    assert torch.equal(got[0], wantd[0]) and (got[1] == 0).all()
    (got,) = torch.autograd.grad(losses.distill_top(leaf, ids, v, w).mean(), leaf)
    near_grad(got, wantd.double() / R, 2 * STEP * wantd.double().abs() / R)
    loss = losses.distill_top(leaf, ids, v, w).sum()
    loss.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        loss.backward()
    with torch.no_grad():
        assert not losses.distill_top(leaf, ids, v, w).requires_grad


def test_autograd_notices_logits_that_were_written_over(losses):
    h = torch.randn(5, 500, device=DEV, requires_grad=True)
    tok = torch.randint(500, (5,), device=DEV)
    old, adv = torch.full((5,), -6.0, device=DEV), torch.ones(5, device=DEV)
    gpu_case("losses' gradient in place of logits that autograd has saved")
    x = torch.tanh(h)                                                # (whose backward pass asks for x)
    lg = x.detach()
    _, g = losses.policy_loss_grad(lg, tok, old, adv, out=lg)
    with pytest.raises(RuntimeError, match="inplace"):
        x.backward(g)
    x = 2 * h
    lg = x.detach()
    _, want = losses.policy_loss_grad(lg, tok, old, adv)
    _, g = losses.policy_loss_grad(lg, tok, old, adv, out=lg)
    x.backward(g)
    torch.cuda.synchronize()
    assert torch.equal(h.grad, 2 * want)


def test_autograd_through_a_head(losses):
    """The loss's gradient goes on to a trainable head, as float32 autograd has it."""
    g = torch.Generator(DEV).manual_seed(1)
    h = torch.randn(40, 64, generator=g, device=DEV)
    W = (torch.randn(500, 64, generator=g, device=DEV) * 0.2).requires_grad_()
    ids, v, w = teacher_of(h @ W.detach().T, 8, 1)
    gpu_case("losses through a head")
    losses.distill_top(h @ W.T, ids, v, w).sum().backward()
    got, W.grad = W.grad, None
    lp = torch.log_softmax((h.double() @ W.double().T), 1)
    at = ids.long()
    q = v.double().exp()
    left = 1 - q.sum(1)
    tail = torch.logsumexp(lp.scatter(1, at, NINF), 1)
    loss = w * ((q * (v - lp.gather(1, at))).sum(1) + left * (left.log() - tail))
    loss.sum().backward()
    # 40 rows' gradients, each off by SUM of its size, and the products' own roundings, 500 + 64 terms
    torch.testing.assert_close(got.double(), W.grad.double(), rtol=1e-3, atol=600 * STEP * 40)


def test_repeats_and_streams_bit_for_bit(losses):
    for R in (40, 300):
        x, tok = rows_of(R, 20001, "bf16", 1)
        ids, v, w = teacher_of(x, 20, 1)
        gpu_case(f"losses on three streams at once R={R}")
        torch.cuda.synchronize()
        got = []
        for st in [torch.cuda.Stream() for _ in range(3)]:
            with torch.cuda.stream(st):
                got += [losses.distill_top_grad(x, ids, v, w) for _ in range(3)]
        torch.cuda.synchronize()
        for b in got[1:]:
            assert torch.equal(got[0][0], b[0]) and torch.equal(got[0][1], b[1])


@pytest.mark.parametrize("R", [24, 280])
def test_graphs_replayed_with_new_logits(losses, R):
    """Two captured graphs, replayed at once, eager calls between; autograd is refused within."""
    cases = []
    for s in range(3):
        x, tok = rows_of(R, 9003, "f16", s)
        cases.append((x, *teacher_of(x, 20, s)))
    ins = [[t.clone() for t in cases[0]] for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    gpu_case(f"losses graphs R={R}")
    torch.cuda.synchronize()
    for args, st in zip(ins, streams):
        with torch.cuda.stream(st):
            losses.distill_top_grad(*args)
        st.synchronize()
        leaf = args[0].clone().requires_grad_()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(losses.distill_top_grad(*args))
            with pytest.raises(ValueError, match="distill_top_grad"):
                losses.distill_top(leaf, *args[1:])
        graphs.append(g)
    for i in (1, 2, 0, 1):
        for j, st in enumerate(streams):
            with torch.cuda.stream(st):
                for t, s in zip(ins[j], cases[(i + j) % 3]):
                    t.copy_(s)
                graphs[j].replay()
        eager = losses.distill_top_grad(*cases[i])
        torch.cuda.synchronize()
        for j in range(2):
            want = losses.distill_top_grad(*cases[(i + j) % 3])
            torch.cuda.synchronize()
            assert torch.equal(outs[j][0], want[0]) and torch.equal(outs[j][1], want[1])
        check_distill(*eager, *cases[i])


def test_a_teachers_scores_teach_a_student(pkg, losses):
    """As used: token_logprobs' alternatives of a target's logits are what a draft learns from."""
    lp = import_module(pkg.__name__ + ".logprobs")
    x, _ = rows_of(64, 30001, "bf16", 1)
    t, tok = rows_of(64, 30001, "bf16", 2)
    gpu_case("distill from token_logprobs")
    s = lp.token_logprobs(t, tok, 20)
    w = torch.full((64,), 1 / 64, device=DEV)
    loss, grad = losses.distill_top_grad(x, s.top_ids, s.top_logprobs, w)
    again, zero = losses.distill_top_grad(t, s.top_ids, s.top_logprobs, w)
    torch.cuda.synchronize()
    check_distill(loss, grad, x, s.top_ids, s.top_logprobs, w)
    check_distill(again, zero, t, s.top_ids, s.top_logprobs, w)
    old = lp.token_logprobs(x, tok).logprob
    out = losses.policy_loss(x, tok, old, torch.ones(64, device=DEV))
    torch.cuda.synchronize()
    # the ratio of a policy to itself: both log probabilities within LP and token_logprobs' own 200 steps
    near(out.loss, torch.full((64,), -1.0, dtype=torch.float64, device=DEV), 2 * (LP + 200 * STEP) * (1 + old.abs()), "on policy")
