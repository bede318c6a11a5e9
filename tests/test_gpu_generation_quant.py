"""Generating with norm and rotation per head and the paged cache in 8 bits, on the GPU.

One layer of a decoder runs through the libraries' C ABI alone, as test_gpu_generation.py's
does over 16 bits:

  prompts:  qkv = RMSNorm(x) Wqkv^T, queries and keys normalised and turned inside it, keys and
            values into the pages in 8 bits (prompts of different lengths)
  a step:   the same for one token, whose position is its sequence's length, then attention
            over the pages, and logits, whose best token is the next one
  after:    the cache read back, into a cache of 16 bits that answers the same; the gradient of
            norm and rotation from the attention's outputs' side

Every operator's output is held against 64 bits from the inputs it got on the device. Then a
step is captured and replayed."""
import math

import pytest
import torch

import grxcp_amd as g
import paged_cases
import quant_cases as qc
from helpers import say
from paged_cases import Workspace, desc, ints
from test_gpu_generation import D, EPS, PAGE, VOCAB, Decoder
from test_gpu_qk_norm_rope import LEAST, STEP, TURN, angles, backward_ref, forward_ref, norm_error, reach

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
ROTARY = 48


class Layer(Decoder):
    """Decoder with gains for the heads of queries and keys, and a rotation of 48 of 64 values."""

    def __init__(self, blas, dnn, rows, heads, group, seed):
        super().__init__(blas, dnn, rows, heads, group, seed)
        gen = torch.Generator().manual_seed(seed + 1)
        self.qg, self.kg = ((1 + 0.2 * torch.randn(D, generator=gen)).to(BF16).cuda() for _ in range(2))
        self.freq = (1e4 ** (-torch.arange(0, ROTARY, 2).double() / ROTARY)).float().cuda()

    def turn(self, q, k, positions):
        """In place, inside the projection."""
        g.check(self.dnn.qk_norm_rope(desc(q), q.data_ptr(), desc(k), k.data_ptr(), desc(self.qg), self.qg.data_ptr(),
                                      self.kg.data_ptr(), EPS, g.ROPE_HALVES, ROTARY, positions.data_ptr(),
                                      self.freq.data_ptr(), desc(q), q.data_ptr(), desc(k), k.data_ptr()), "turn")

    def check_turn(self, before, after, positions):
        for x, y, gain in zip(before, after, (self.qg, self.kg)):
            want, plain = forward_ref(x.cpu(), gain.cpu(), EPS, angles(positions.cpu(), self.freq.cpu()), False)
            u = STEP[BF16]
            bound = u * want.abs() + (1 + u) * reach(plain, ROTARY, False) * (norm_error(D) + TURN) + LEAST[BF16]
            assert ((y.cpu().double() - want).abs() <= bound).all()


def turned(m, b, positions):
    q, k, v = m.parts(b)
    before = [x.clone() for x in (q, k, v)]
    m.turn(q, k, positions)
    m.check_turn(before[:2], (q, k), positions)
    assert torch.equal(v, before[2])
    return q, k, v, before


@pytest.mark.parametrize("heads,group,block", [(4, 1, 16), (2, 4, 4), (1, 8, 1)])
def test_prompts_steps_and_the_way_back(blas, dnn, heads, group, block):
    prompts, steps = [37, 1, 20], 10
    b, longest = len(prompts), max(prompts)
    gen = torch.Generator().manual_seed(50 + group)
    tokens = torch.randint(0, VOCAB, (b, longest), generator=gen).int().cuda()
    c = qc.QuantCache(gen, [0] * b, heads, PAGE, block, D, True, room=longest + steps)
    scale = D ** -0.5

    say(f"generation in 8 bits, heads={heads} group={group}: prompts")
    many = Layer(blas, dnn, b * longest, heads, group, seed=52)
    many.project(tokens.view(-1))
    positions = torch.arange(longest).int().repeat(b, 1).cuda()
    q, k, v, before = turned(many, b, positions)
    want = c.append_ref(k, v, prompts)
    qc.append(dnn, c, k, v, ints(prompts))
    c.check(want)
    c.lengths += ints(prompts)
    c.n = list(prompts)

    say("the prompts' gradient")
    dq, dk = (torch.randn(x.shape, generator=gen).to(BF16).cuda() for x in (q, k))
    dqg, dkg = (torch.empty(D, device="cuda") for _ in range(2))
    out = [torch.empty_like(x) for x in (dq, dk)]
    xq, xk = before[:2]
    wd = desc(many.qg)
    ws = Workspace(dnn.qk_norm_rope_workspace(desc(xq), desc(xk), wd))
    g.check(dnn.qk_norm_rope_backward(
        desc(xq), xq.data_ptr(), desc(xk), xk.data_ptr(), wd, many.qg.data_ptr(), many.kg.data_ptr(), EPS,
        g.ROPE_HALVES, ROTARY, positions.data_ptr(), many.freq.data_ptr(), desc(dq), dq.data_ptr(), desc(dk),
        dk.data_ptr(), desc(out[0]), out[0].data_ptr(), desc(out[1]), out[1].data_ptr(), dqg.data_ptr(),
        dkg.data_ptr(), ws.p, ws.size))
    for x, gain, dy, dx, dgain in ((xq, many.qg, dq, out[0], dqg), (xk, many.kg, dk, out[1], dkg)):
        ref, off, gref, mass = backward_ref(x.cpu(), gain.cpu(), dy.cpu(), EPS,
                                            angles(positions.cpu(), many.freq.cpu()), False, ROTARY)
        u = STEP[BF16]
        assert ((dx.cpu().double() - ref).abs() <= u * ref.abs() + (1 + u) * off + LEAST[BF16]).all()
        count = x.shape[0] * x.shape[1] * x.shape[2]
        assert ((dgain.cpu().double() - gref).abs() <= mass[0] * (mass[1] + (count + 2) * 2.0 ** -24)).all()

    one = Layer(blas, dnn, b, heads, group, seed=52)
    token = torch.stack([tokens[i, n - 1] for i, n in enumerate(prompts)]).contiguous()
    for step in range(steps):
        say(f"step {step}")
        one.project(token)
        q, k, v, _ = turned(one, b, c.lengths[:, None])      # the token's position: what came before it
        want = c.append_ref(k, v, [1] * b)
        qc.append(dnn, c, k, v)
        c.check(want)
        c.lengths += 1
        c.n = [n + 1 for n in c.n]
        o = one.o.view(b, 1, one.H, D).transpose(1, 2)
        qc.attend(dnn, c, q, o, scale)
        for i in range(b):
            K, V, there = c.rows(i)
            ref, bound = qc.attention_ref(q[i, :, 0].cpu(), K, V, scale, there)
            assert ((o[i, :, 0].cpu().double() - ref).abs() <= bound).all(), (step, i)
        one.answer()
        token = one.logits.argmax(1).int()

    say("the cache back in 16 bits")
    longest = max(c.n)
    K, V = (torch.full((b, heads, longest, D), math.nan, dtype=BF16, device="cuda") for _ in range(2))
    qc.read(dnn, c, K, V)
    full = paged_cases.Cache(gen, BF16, [0] * b, heads, PAGE, D, True, room=longest)
    paged_cases.append(dnn, full, K, V, c.lengths)
    full.lengths = c.lengths.clone()
    for i, n in enumerate(c.n):
        k64, v64, _ = c.rows(i)
        assert torch.equal(K[i, :, :n].cpu(), k64.to(BF16)) and torch.equal(V[i, :, :n].cpu(), v64.to(BF16))
        assert (K[i, :, n:] == 0).all() and (V[i, :, n:] == 0).all()
    o, other = one.o.view(b, 1, one.H, D).transpose(1, 2).clone(), torch.empty((b, one.H, 1, D), dtype=BF16, device="cuda")
    qc.attend(dnn, c, q, o, scale)
    paged_cases.attend(dnn, full, q, other, scale)
    for i, n in enumerate(c.n):
        k64, v64, _ = c.rows(i)
        one_q = q[i, :, 0].cpu()
        ref, _, theirs, _ = paged_cases.attention_ref(one_q, K[i, :, :n].cpu(), V[i, :, :n].cpu(), scale)
        mine, bound = qc.attention_ref(one_q, k64, v64, scale)
        assert ((o[i, :, 0].cpu().double() - mine).abs() <= bound).all()
        assert ((other[i, :, 0].cpu().double() - ref).abs() <= theirs).all()


def test_a_captured_step_generates_what_eager_steps_do(gpu):
    """The step in one graph, positions and lengths on the device, replayed with eager work
    between: the tokens, outputs, codes and scales of eager steps, bit for bit."""
    heads, group, steps, prompts = 2, 4, 20, [30, 7]
    b, scale = len(prompts), D ** -0.5
    blas, dnn = g.Blas(), g.Dnn()
    start = torch.randn((b, 2 * heads, max(prompts), D), generator=torch.Generator().manual_seed(54)).to(BF16).cuda()
    ad = g.AttnDesc(True, scale)

    def session():
        gen = torch.Generator().manual_seed(55)
        c = qc.QuantCache(gen, [0] * b, heads, PAGE, 8, D, True, room=max(prompts) + steps)
        m = Layer(blas, dnn, b, heads, group, seed=56)
        qc.append(dnn, c, start[:, :heads], start[:, heads:], ints(prompts))
        c.lengths += ints(prompts)
        token, best = ints([[3], [900]]), torch.zeros((b, 1), device="cuda")
        lse = torch.zeros(b, device="cuda")
        q, k, v = m.parts(b)
        o = m.o.view(b, 1, m.H, D).transpose(1, 2)
        args = c.args()
        d = [desc(t) for t in (q, k, v, o, m.logits)]
        ws = [Workspace(dnn.paged_attention_quantized_workspace(d[0], args[0], args[7])),
              Workspace(dnn.token_logprob_workspace(d[4], 1))]

        def step():
            m.project(token[:, 0])
            m.turn(q, k, c.lengths)
            g.check(dnn.paged_append_quantized(d[1], k.data_ptr(), d[2], v.data_ptr(), *args))
            c.lengths.add_(1)
            g.check(dnn.paged_attention_quantized(ad, d[0], q.data_ptr(), *args, d[3], o.data_ptr(), ws[0].p, ws[0].size))
            m.answer()
            g.check(dnn.token_logprob(d[4], m.logits.data_ptr(), None, None, lse.data_ptr(), None, 1, best.data_ptr(),
                                      token.data_ptr(), ws[1].p, ws[1].size))

        return c, m, token, best, step, (d, args, ws, lse)

    eager, captured = session(), session()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    say("capturing a step in 8 bits")
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
        for x, y in ((eager[1].o, captured[1].o), (eager[1].logits, captured[1].logits), (eager[1].qkv, captured[1].qkv)):
            assert torch.equal(x, y), f"step {i}"
    captured[0].check(eager[0].state())
    assert captured[0].lengths.tolist() == [n + steps for n in prompts]
    del graph
    blas.close()
    dnn.close()
