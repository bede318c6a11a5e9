"""Generating with the paged cache, from prompts to the policy's gradient, on the GPU.

One layer of a decoder runs through the libraries' C ABI alone:

  prompts:  h = RMSNorm(x), qkv = h Wqkv^T, causal attention over the prompts,
            keys and values into the pages (counts: prompts of different lengths)
  a step:   h = RMSNorm(x), qkv = h Wqkv^T, append one token, attention over the
            pages (its weights add up), o Wo^T + x, RMSNorm, logits, log
            probabilities with the best alternatives; the best one is the next token
  between:  eviction to a budget into fresh pages, which then are the cache
  after:    log probabilities of the chosen tokens over all steps at once, and the
            gradient of a policy loss with an entropy term in those logits

Every operator's output is held against 64 bits from the inputs it got on the device, the
cache against rows that the test keeps beside it. Then a step is captured and replayed.
"""
import math

import pytest
import torch

import grxcp_amd as g
from helpers import say
from paged_cases import Workspace, append, attend, attention_ref, desc, evict, evict_ref, guarded, ints
from test_gpu_token_logprob import check_forward, grad_ref, near

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
D, VOCAB, PAGE, EPS, DECAY = 64, 1001, 16, 1e-5, 0.9


class Decoder:
    """Weights, buffers for `rows` tokens at once and the calls of one layer."""

    def __init__(self, blas, dnn, rows, heads, group, seed):
        self.blas, self.dnn, self.heads, self.H = blas, dnn, heads, heads * group
        self.dim, self.out = self.H * D, (self.H + 2 * heads) * D
        gen = torch.Generator().manual_seed(seed)

        def w(out, inp):
            return (torch.randn((out, inp), generator=gen) / inp ** 0.5).to(BF16).cuda()

        self.emb, self.wqkv, self.wo, self.wout = w(VOCAB, self.dim), w(self.out, self.dim), w(self.dim, self.dim), w(
            VOCAB, self.dim)
        self.emb *= 16
        self.wout *= 2
        self.norm = torch.ones(self.dim, dtype=BF16, device="cuda")
        e = lambda *s, t=BF16: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
        self.x, self.h, self.o, self.qkv = e(rows, self.dim), e(rows, self.dim), e(rows, self.dim), e(rows, self.out)
        self.logits = e(rows, VOCAB, t=torch.float32)

    def linear(self, w, x, y, beta=0.0):
        n, k = w.shape
        # (a library call that allocates nothing, so that it may be captured)
        g.check(self.blas.gemm_ex_noalloc(1, 0, n, x.shape[0], k, 1.0, w.data_ptr(), g.GRX_R_16BF, k, x.data_ptr(),
                                          g.GRX_R_16BF, k, beta, y.data_ptr(),
                                          g.GRX_R_16BF if y.dtype == BF16 else g.GRX_R_32F, n), "linear")

    def rms(self):
        xd = desc(self.x)
        g.check(self.dnn.rmsnorm(xd, self.x.data_ptr(), desc(self.norm), self.norm.data_ptr(), EPS, xd,
                                 self.h.data_ptr()), "rmsnorm")

    def project(self, tokens):
        torch.index_select(self.emb, 0, tokens, out=self.x)
        self.rms()
        self.linear(self.wqkv, self.h, self.qkv)

    def parts(self, b):
        """q, k, v of the projection of b sequences as [b, heads, tokens, D] views."""
        p = self.qkv.view(b, -1, self.H + 2 * self.heads, D).transpose(1, 2)
        return p[:, :self.H], p[:, self.H:self.H + self.heads], p[:, self.H + self.heads:]

    def answer(self):
        self.linear(self.wo, self.o, self.x, beta=1.0)
        self.rms()
        self.linear(self.wout, self.h, self.logits)


class Pages:
    """A cache that grows by append and is replaced by eviction, and its rows in order."""

    def __init__(self, b, heads, room, seed):
        self.width = -(-room // PAGE)
        self.guarded = [guarded(2 * b * self.width, PAGE, heads, D, BF16, True) for _ in range(2)]
        self.k, self.v = (p[1:-1] for p in self.guarded)
        self.order = torch.randperm(2 * b * self.width, generator=torch.Generator().manual_seed(seed)).int().cuda()
        self.tables = self.order.view(2, b, self.width)
        self.table, self.heads, self.n = self.tables[0], heads, [0] * b
        self.lengths = ints(self.n)
        self.K, self.V = ([torch.zeros(heads, 0, D, dtype=BF16) for _ in range(b)] for _ in range(2))
        self.w = torch.zeros((b, heads, self.width * PAGE), device="cuda")

    def descs(self):
        return desc(self.k), desc(self.v), desc(self.table)

    def grew(self, k, v, counts):
        """The rows appended to each sequence, kept beside the pages."""
        for i, c in enumerate(counts):
            self.K[i] = torch.cat([self.K[i], k[i, :, :c].cpu()], 1)
            self.V[i] = torch.cat([self.V[i], v[i, :, :c].cpu()], 1)
            self.n[i] += c

    def check(self):
        assert self.lengths.tolist() == self.n
        for i, n in enumerate(self.n):
            at = torch.arange(n, device="cuda")
            for pool, rows in ((self.k, self.K[i]), (self.v, self.V[i])):
                got = pool[self.table[i, at // PAGE].long(), :, at % PAGE].transpose(0, 1).cpu()
                assert torch.equal(got, rows), f"rows of sequence {i}"


@pytest.mark.parametrize("heads,group", [(4, 1), (2, 4)])
def test_prompts_steps_eviction_and_gradient(blas, dnn, heads, group):
    prompts, steps, budget, recent = [37, 1, 20], 12, 28, 9
    b, longest = len(prompts), max(prompts)
    gen = torch.Generator().manual_seed(40 + group)
    tokens = torch.randint(0, VOCAB, (b, longest), generator=gen).int().cuda()
    c = Pages(b, heads, longest + steps, seed=41)
    scale = D ** -0.5

    say(f"generation heads={heads} group={group}: prompts")
    many = Decoder(blas, dnn, b * longest, heads, group, seed=42)
    many.project(tokens.view(-1))
    q, k, v = many.parts(b)
    append(dnn, c, k, v, ints(prompts))
    c.lengths += ints(prompts)
    c.grew(k, v, prompts)
    c.check()
    if group == 1:
        # the last query of each prompt: one token's attention over the pages against
        # the causal attention's row, both within what 64 bits allow each
        full = many.o.view(b, longest, many.H, D).transpose(1, 2)
        g.check(dnn.attention(g.AttnDesc(True, scale), desc(q), q.data_ptr(), desc(k), k.data_ptr(), desc(v),
                              v.data_ptr(), desc(full), full.data_ptr()))
        last = torch.stack([q[i, :, n - 1:n] for i, n in enumerate(prompts)])
        o = torch.empty_like(last)
        attend(dnn, c, last, o, scale)
        for i, n in enumerate(prompts):
            one = last[i, :, 0].cpu()
            ref, p, bound, _ = attention_ref(one, c.K[i], c.V[i], scale)
            assert ((o[i, :, 0].cpu().double() - ref).abs() <= bound).all(), f"prompt {i}"
            # that kernel may round its scaled queries to bf16: a score is off by half a
            # step of sum |q k|, weights by twice that, relatively
            size = (c.K[i].double().abs() @ one.double().abs()[:, :, None]).amax(1) * scale
            bound = bound + 2 * 2.0 ** -8 * size * (p[:, None] @ c.V[i].double().abs())[:, 0]
            assert ((full[i, :, n - 1].cpu().double() - ref).abs() <= bound).all(), f"prompt {i}, causal"

    one = Decoder(blas, dnn, b, heads, group, seed=42)
    token = torch.stack([tokens[i, n - 1] for i, n in enumerate(prompts)]).contiguous()
    history, chosen, said = [], [], []
    for step in range(steps):
        say(f"generation step {step}")
        one.project(token)
        q, k, v = one.parts(b)
        append(dnn, c, k, v)
        c.lengths += 1
        c.grew(k, v, [1] * b)
        before = c.w.cpu()
        o = one.o.view(b, 1, one.H, D).transpose(1, 2)
        attend(dnn, c, q, o, scale, c.w, DECAY)
        for i, n in enumerate(c.n):
            ref, p, bound, pbound = attention_ref(q[i, :, 0].cpu(), c.K[i], c.V[i], scale)
            assert ((o[i, :, 0].cpu().double() - ref).abs() <= bound).all(), (step, i)
            want = DECAY * before[i, :, :n].double() + p.reshape(heads, group, n).sum(1)
            # (decay itself is rounded to fp32)
            room = pbound.reshape(heads, group, n).sum(1) + (group + 3) * 2.0 ** -23 * want
            assert ((c.w[i, :, :n].cpu().double() - want).abs() <= room).all(), (step, i)
            assert torch.equal(c.w[i, :, n:].cpu(), before[i, :, n:])
        one.answer()
        x = one.logits.clone()
        check_forward(dnn, x, token.tolist(), top=5)
        ld = desc(x)
        ws = Workspace(dnn.token_logprob_workspace(ld, 5))
        lse, best, index = torch.empty(b, device="cuda"), torch.empty((b, 5), device="cuda"), ints([[0] * 5] * b)
        g.check(dnn.token_logprob(ld, x.data_ptr(), None, None, lse.data_ptr(), None, 5, best.data_ptr(),
                                  index.data_ptr(), ws.p, ws.size))
        token = index[:, 0].contiguous()
        history.append(x)
        chosen.append(token)
        said.append(best[:, 0])
        if max(c.n) > budget and step % 4 == 3:
            say("eviction")
            other = c.tables[1] if c.table.data_ptr() == c.tables[0].data_ptr() else c.tables[0]
            new_w, lengths = torch.full_like(c.w, math.nan), torch.empty_like(c.lengths)
            kept = evict(dnn, c, c.w, budget, recent, other, new_w, lengths)
            old = c.w.cpu()
            for i, n in enumerate(c.n):
                for h in range(heads):
                    stay = evict_ref(old[i, h, :n], budget, recent)
                    assert kept[i, h].tolist() == stay + [-1] * (budget - len(stay)), (step, i, h)
                    assert torch.equal(new_w[i, h, :len(stay)].cpu(), old[i, h, stay])
                rows = [torch.stack([t[i][h][kept[i, h, :min(n, budget)].long().cpu()] for h in range(heads)])
                        for t in (c.K, c.V)]
                c.K[i], c.V[i] = rows
                c.n[i] = min(n, budget)
            assert (new_w[:, :, budget:] == 0).all()
            c.table, c.w, c.lengths = other, new_w, lengths
        c.check()
    for p in c.guarded:
        assert torch.isnan(p[0]).all() and torch.isnan(p[-1]).all()

    say("generation: the steps' policy gradient")
    x, token = torch.cat(history), torch.cat(chosen)
    rows = steps * b
    xd = desc(x)
    logp, lse, H = (torch.empty(rows, device="cuda") for _ in range(3))
    ws = Workspace(dnn.token_logprob_workspace(xd, 0))
    g.check(dnn.token_logprob(xd, x.data_ptr(), token.data_ptr(), logp.data_ptr(), lse.data_ptr(), H.data_ptr(), 0,
                              None, None, ws.p, ws.size))
    check_forward(dnn, x, token.tolist())
    # the same numbers in another number of rows: both were held to 64 bits above
    assert torch.allclose(logp, torch.cat(said), rtol=2.0 ** -16, atol=2.0 ** -16)
    da, dH = torch.randn(rows, generator=gen).cuda(), torch.full((rows,), 0.01, device="cuda")
    dx = torch.empty_like(x)
    g.check(dnn.token_logprob_backward(xd, x.data_ptr(), token.data_ptr(), lse.data_ptr(), H.data_ptr(),
                                       da.data_ptr(), dH.data_ptr(), xd, dx.data_ptr()))
    want, bound = grad_ref(x.cpu().double(), token.tolist(), lse.cpu().double(), H.cpu().double(), da.cpu().double(),
                           dH.cpu().double())
    near(dx, want, 2.0 ** -24 * (want.abs() + bound) + bound + 2.0 ** -150, "dx")


def test_a_captured_step_generates_what_eager_steps_do(gpu):
    """The whole step in one graph (token, lengths and weights updated on the device),
    replayed with eager work between: the tokens, log probabilities, weights and pages of
    eager steps, bit for bit."""
    heads, group, steps, prompts = 2, 4, 20, [30, 7]
    b, scale = len(prompts), D ** -0.5
    blas, dnn = g.Blas(), g.Dnn()
    gen = torch.Generator().manual_seed(44)
    start = torch.randn((b, 2 * heads, max(prompts), D), generator=gen).to(BF16).cuda()
    ad = g.AttnDesc(False, scale)

    def session():
        c, m = Pages(b, heads, max(prompts) + steps, seed=45), Decoder(blas, dnn, b, heads, group, seed=46)
        append(dnn, c, start[:, :heads], start[:, heads:], ints(prompts))
        c.lengths += ints(prompts)
        token, best = ints([[3], [900]]), torch.zeros((b, 1), device="cuda")
        lse = torch.zeros(b, device="cuda")
        q, k, v = m.parts(b)
        o = m.o.view(b, 1, m.H, D).transpose(1, 2)
        kd, vd, td = c.descs()
        d = [desc(t) for t in (q, k, v, o, c.w, m.logits)]
        sizes = (dnn.paged_attention_workspace(d[0], kd, td, d[4]), dnn.token_logprob_workspace(d[5], 1))
        ws = [Workspace(s) for s in sizes]

        def step():
            m.project(token[:, 0])
            g.check(dnn.paged_append(d[1], k.data_ptr(), d[2], v.data_ptr(), kd, c.k.data_ptr(), vd, c.v.data_ptr(),
                                     td, c.table.data_ptr(), c.lengths.data_ptr()))
            c.lengths.add_(1)
            g.check(dnn.paged_attention(ad, d[0], q.data_ptr(), kd, c.k.data_ptr(), vd, c.v.data_ptr(), td,
                                        c.table.data_ptr(), c.lengths.data_ptr(), DECAY, d[4], c.w.data_ptr(), d[3],
                                        o.data_ptr(), ws[0].p, ws[0].size))
            m.answer()
            g.check(dnn.token_logprob(d[5], m.logits.data_ptr(), None, None, lse.data_ptr(), None, 1,
                                      best.data_ptr(), token.data_ptr(), ws[1].p, ws[1].size))

        return c, m, token, best, step, (d, kd, vd, td, ws, lse)

    eager, captured = session(), session()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    say("capturing a step")
    with torch.cuda.graph(graph, stream=side):
        stream = torch.cuda.current_stream().cuda_stream
        dnn.set_stream(stream)
        blas.set_stream(stream)
        captured[4]()
    dnn.set_stream(None)
    blas.set_stream(None)
    for i in range(steps):
        say(f"captured step {i}")
        eager[4]()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager[2], captured[2]), f"token of step {i}"
        assert torch.equal(eager[3], captured[3]), f"log probability of step {i}"
        for a, c in ((eager[0].w, captured[0].w), (eager[1].o, captured[1].o), (eager[1].logits, captured[1].logits)):
            assert torch.equal(a, c), f"step {i}"
    # (as bits: rows that no token reached hold NaN)
    for a, c in ((eager[0].k, captured[0].k), (eager[0].v, captured[0].v)):
        assert torch.equal(a.view(torch.int16), c.view(torch.int16))
    assert captured[0].lengths.tolist() == [n + steps for n in prompts]
    del graph
    blas.close()
    dnn.close()
