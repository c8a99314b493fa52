"""The operators on tokens and gradients together, as a training step of a token model uses them around the framework's dense products: lookup, a dense
layer, the head's product, token loss, back through both products, the table's gradient, clipping by the norm of all gradients, Adam."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

VOCAB, WIDTH, HIDDEN, TOKENS, MAX_NORM, SCALE = 1003, 64, 96, 250, 0.05, 8.0
SIZES = [VOCAB * WIDTH, WIDTH * HIDDEN, HIDDEN, HIDDEN * 1008]      # (the head's rows are padded to a multiple of 16 values)


class Step:
    def __init__(self, seed):
        torch.manual_seed(seed)
        n = sum(SIZES)
        self.p, self.g = torch.randn(n, device="cuda") * 0.1, torch.zeros(n, device="cuda")
        self.m, self.v, self.pows = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda"), torch.ones(2, device="cuda")
        self.params, self.grads = list(self.p.split(SIZES)), list(self.g.split(SIZES))
        self.params[3].view(HIDDEN, 1008)[:, VOCAB:] = 0.0
        self.ids, self.targets = torch.randint(0, VOCAB, (TOKENS,), device="cuda"), torch.randint(-1, VOCAB, (TOKENS,), device="cuda")
        self.ids[:40] = 7
        f = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
        self.x, self.a, self.logits, self.dl = f(TOKENS, WIDTH), f(TOKENS, HIDDEN), f(TOKENS, 1008), f(TOKENS, 1008)
        self.da, self.dx, self.logp, self.norm, self.coef = f(TOKENS, HIDDEN), f(TOKENS, WIDTH), f(TOKENS), f(1), f(1)
        self.status = torch.zeros(1, device="cuda", dtype=torch.int32)

    def run(self):
        from oxidized_neural_orchestra_b200.ops import elementwise as ew
        from oxidized_neural_orchestra_b200.ops.clip import grad_norm
        from oxidized_neural_orchestra_b200.ops.embedding import embedding, embedding_grad
        from oxidized_neural_orchestra_b200.ops.gemm import gemm
        from oxidized_neural_orchestra_b200.ops.token_loss import token_loss

        (table, w, b, head), (gt, gw, gb, gh) = self.params, self.grads
        table, gt, w, gw = table.view(VOCAB, WIDTH), gt.view(VOCAB, WIDTH), w.view(WIDTH, HIDDEN), gw.view(WIDTH, HIDDEN)
        head, gh = head.view(HIDDEN, 1008)[:, :VOCAB], gh.view(HIDDEN, 1008)[:, :VOCAB]
        logits, dl = self.logits[:, :VOCAB], self.dl[:, :VOCAB]
        embedding(table, self.ids, self.x, scale=SCALE, status=self.status)
        gemm(self.x, w, b_mn_major=True, bias=b, act="tanh", act_param=1.0, out=self.a)
        gemm(self.a, head, b_mn_major=True, out=logits)
        token_loss(logits, self.targets, out=dl, logp=self.logp, scale=1.0 / TOKENS, status=self.status)
        gemm(dl, head, out=self.da, aux=self.a, dact="tanh", dact_param=1.0)
        gemm(self.a, dl, a_mn_major=True, b_mn_major=True, out=gh)
        gemm(self.da, w, out=self.dx)
        gemm(self.x, self.da, a_mn_major=True, b_mn_major=True, out=gw)
        torch.sum(self.da, 0, out=gb)      # (elementwise.colsum's scratch is one for all streams)
        embedding_grad(self.dx, self.ids, gt, scale=SCALE, status=self.status)
        grad_norm(self.grads, self.norm, max_norm=MAX_NORM, coef=self.coef)
        ew.adam_tick(self.pows, 0.9, 0.999)
        ew.optim_step(self.p, self.g, kind="adam", lr=1e-3, m=self.m, v=self.v, adam_pows=self.pows, grad_coef=self.coef)


def test_step_against_64_bits():
    s = Step(0)
    leaves = [t.double().clone().requires_grad_() for t in s.params]
    table, w, b, head = leaves[0].view(VOCAB, WIDTH), leaves[1].view(WIDTH, HIDDEN), leaves[2], leaves[3].view(HIDDEN, 1008)[:, :VOCAB]
    lp = torch.log_softmax(torch.tanh(table[s.ids] * SCALE @ w + b) @ head, 1)
    live = s.targets >= 0
    picked = torch.where(live, lp.gather(1, s.targets.clamp_min(0).unsqueeze(1)).squeeze(1), 0.0)
    (-picked.sum() / TOKENS).backward()
    ref = torch.cat([t.grad for t in leaves])
    s.run()
    torch.cuda.synchronize()
    assert s.status.item() == 0
    # the products round their operands to tf32 (2^-11 each, or cut to 2^-10): four of them one behind the other, every rounding at random
    tol = 8 * 2.0 ** -10
    rel = lambda a, r: float((a.double() - r.detach()).norm() / r.detach().norm())  # noqa: E731
    assert rel(s.logp, picked) <= tol
    for k, (g, r) in enumerate(zip(s.grads, leaves)):
        assert rel(g, r.grad) <= tol, k
    norm = float(ref.norm())
    assert norm > MAX_NORM and abs(s.norm.item() - norm) <= tol * norm and abs(s.coef.item() - MAX_NORM / norm) <= tol * MAX_NORM / norm
    # Adam's first step: m = (1 - b1) g of the clipped gradient, 1 - b1 rounded once and three more roundings
    own = s.g.double() * s.coef.double() * 0.1
    assert ((s.m.double() - own).abs() <= 4 * 2.0 ** -24 * own.abs() + 1e-40).all()


def test_step_captured_and_replayed_beside_another():
    eager, replayed = [Step(1), Step(2)], [Step(1), Step(2)]
    for s in eager:
        for _ in range(4):
            s.run()
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s, st in zip(replayed, streams):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            s.run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            s.run()
        graphs.append((g, st))
    for _ in range(3):
        for g, st in graphs:
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(eager, replayed):
        assert a.status.item() == b.status.item() == 0 and math.isfinite(a.norm.item())
        assert torch.equal(a.p, b.p) and torch.equal(a.g, b.g) and torch.equal(a.norm, b.norm)
