"""Adapters and losses as they are used together, beside the quantized head that they leave frozen: serving requests
with an adapter each, and training steps of the adapters from a teacher's scores and from rewarded samples."""
from __future__ import annotations

from importlib import import_module

import pytest

from conftest import gpu_case

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
K, V, R, N_ADAPTERS = 512, 4096, 16, 3


@pytest.fixture(scope="module")
def mods(pkg):
    return [import_module(f"{pkg.__name__}.{m}") for m in ("ops", "lora", "losses", "logprobs")]


class Head:
    """A frozen fp8 head, adapters beside it, a batch of hidden states."""

    def __init__(self, mods, M, seed):
        self.ops, self.lora, self.losses, self.scores = mods
        g = torch.Generator(DEV).manual_seed(seed)
        weight = (torch.randn(V, K, generator=g, device=DEV) * 0.08).to(torch.float8_e4m3fn)
        self.weight = self.ops.pack_fp8_dense(weight, torch.full((V // 128, K // 128), 1.0, device=DEV))
        self.a = (torch.randn(N_ADAPTERS, R, K, generator=g, device=DEV) * K ** -0.5).to(BF)
        self.b = (torch.randn(N_ADAPTERS, V, R, generator=g, device=DEV) * 0.2).to(BF)
        self.w = self.lora.LoraStack(self.a, self.b, torch.full((N_ADAPTERS,), 0.5, device=DEV))
        self.x = torch.randn(M, K, generator=g, device=DEV).to(BF)
        self.ids = (torch.arange(M, device=DEV) * (N_ADAPTERS + 1) // M - 1).int()       # the first rows without one
        self.rows = self.lora.plan_rows(self.ids, N_ADAPTERS)

    def base(self):
        return self.ops.gemm_fp8_dense(*self.ops.fp8_quant_group(self.x), self.weight)

    def teacher(self):
        """What another model's logits leave: 20 alternatives a row, and a sampled token of them."""
        g = torch.Generator(DEV).manual_seed(7)
        t = (self.base().float() + torch.randn(len(self.x), V, generator=g, device=DEV)).to(BF)
        pick = torch.randint(20, (len(self.x), 1), generator=g, device=DEV)
        s = self.scores.token_logprobs(t, t.argmax(1), 20)
        return s, s.top_ids.gather(1, pick)[:, 0].long()

    def exact(self, dlogits):
        """The adapters' gradients from the logits', in float64."""
        d, x, s = dlogits.double(), self.x.double(), 0.5
        dx, da, db = (torch.zeros(t.shape, dtype=torch.float64, device=DEV) for t in (self.x, self.a, self.b))
        size = [torch.zeros_like(t) for t in (dx, da, db)]
        for i in range(N_ADAPTERS):
            at = self.ids == i
            A, B = self.a[i].double(), self.b[i].double()
            u, h = s * d[at] @ B, s * x[at] @ A.T
            ua, ha = s * d[at].abs() @ B.abs(), s * x[at].abs() @ A.abs().T
            dx[at], da[i], db[i] = u @ A, u.T @ x[at], d[at].T @ h
            size[0][at], size[1][i], size[2][i] = ua @ A.abs(), ua.T @ x[at].abs(), d[at].abs().T @ ha
        return (dx, da, db), size


def close(got, want, size):
    """Half a step of bf16 (its eps is 2^-7), and sums of at most 4096 + 512 float32 products, of values in two parts
    of which the second is rounded by 2^-8 of 2^-8."""
    limit = (2 * 4608 * 2.0 ** -24 + 2.0 ** -16) * size + 1e-37
    limit = limit + 2.0 ** -8 * (want.abs() + limit)
    bad = ~((got.double() - want).abs() <= limit)
    assert not bad.any(), (got[bad][:4], want[bad][:4], bad.sum())


@pytest.mark.parametrize("M", [40, 1100])
def test_a_training_step_by_hand(mods, M):
    """Forward, the loss's gradient in the logits' place, and backward; all of it again in a replayed graph."""
    h = Head(mods, M, 1)
    s, tok = h.teacher()
    weight = torch.full((M,), 1 / M, device=DEV)
    weight[::7] = 0
    hidden = torch.empty(M, R, device=DEV)

    def step():
        logits = h.base()
        h.lora.add_lora(logits, h.x, h.w, h.rows, out=logits, hidden=hidden)
        keep = logits.clone()
        loss, grad = h.losses.distill_top_grad(logits, s.top_ids, s.top_logprobs, weight, out=logits)
        return keep, loss, grad, *h.lora.add_lora_grad(grad, h.x, h.w, h.rows, hidden)
    gpu_case(f"adapter step by hand M={M}")
    logits, loss, grad, dx, da, db = step()
    torch.cuda.synchronize()
    want, size = h.exact(grad)
    for got, w, z in zip((dx, da, db), want, size):
        close(got, w, z)
    # the loss's own gradient from the logits as they were, and the logits from base and adapter
    again, g2 = h.losses.distill_top_grad(logits, s.top_ids, s.top_logprobs, weight)
    assert torch.equal(again, loss) and torch.equal(g2, grad)
    assert torch.equal(logits[h.ids < 0], h.base()[h.ids < 0])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        outs = step()
    x0 = h.x.clone()
    for scale in (1.0, -0.5, 1.0):
        h.x.copy_(x0 * scale)
        eager = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert torch.equal(a, b)


@pytest.mark.parametrize("M", [40, 1100])
@pytest.mark.parametrize("kind", ["distill", "policy"])
def test_training_steps_of_autograd(mods, M, kind):
    """A few optimizer steps run, and each one's gradients are those by hand."""
    h = Head(mods, M, 2)
    s, tok = h.teacher()
    base = h.base()
    old = h.scores.token_logprobs(base, tok).logprob
    adv = torch.randn(M, device=DEV)
    params = [torch.nn.Parameter(t.clone()) for t in (h.a, h.b)]
    w = h.lora.LoraStack(*params, h.w.scale)
    mean = torch.full((M,), 1 / M, device=DEV)       # (with the rows' sum the steps lead to ratios past e^88)
    opt = torch.optim.SGD(params, lr=0.1)
    gpu_case(f"adapter steps of autograd M={M} {kind}")
    for _ in range(3):
        h.a, h.b = (p.detach().clone() for p in params)
        h.w = h.lora.LoraStack(h.a, h.b, w.scale)
        logits = h.lora.add_lora(base, h.x, w, h.rows)
        if kind == "distill":
            loss = h.losses.distill_top(logits, s.top_ids, s.top_logprobs, mean).sum()
            _, grad = h.losses.distill_top_grad(logits.detach(), s.top_ids, s.top_logprobs, mean)
        else:
            loss = h.losses.policy_loss(logits, tok, old, adv, old, mean, kl=0.1).loss.sum()
            _, grad = h.losses.policy_loss_grad(logits.detach(), tok, old, adv, old, mean, kl=0.1)
        opt.zero_grad()
        loss.backward()
        hidden = torch.empty(M, R, device=DEV)
        same = h.lora.add_lora(base, h.x, h.w, h.rows, hidden=hidden)
        _, da, db = h.lora.add_lora_grad(grad, h.x, h.w, h.rows, hidden)
        torch.cuda.synchronize()
        assert torch.equal(same, logits) and torch.isfinite(loss)
        assert torch.equal(params[0].grad, da) and torch.equal(params[1].grad, db)
        opt.step()


@pytest.mark.parametrize("M", [1, 20, 1100])
def test_serving_requests_with_an_adapter_each(mods, M):
    """The head's product, the adapters in place, scores: one plan for the batch, against the same a request at a time."""
    h = Head(mods, M, 3)
    gpu_case(f"adapters served M={M}")
    logits = h.base()
    h.lora.add_lora(logits, h.x, h.w, h.rows, out=logits)
    got = h.scores.token_logprobs(logits, logits.argmax(1), 5)
    base = h.base()
    torch.cuda.synchronize()
    assert (got.rank == 1).all()
    for i in range(-1, N_ADAPTERS):
        at = (h.ids == i).nonzero()[:, 0]
        want = base[at].double()
        size = torch.zeros_like(want)
        if i >= 0:
            hid = 0.5 * (h.x[at].double() @ h.a[i].double().T)
            want = want + hid @ h.b[i].double().T
            size = (0.5 * h.x[at].double().abs() @ h.a[i].double().abs().T) @ h.b[i].double().abs().T
        close(logits[at], want, size + base[at].double().abs())
