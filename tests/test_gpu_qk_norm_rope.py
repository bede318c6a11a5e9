"""grxdnnQkNormRopeForward / Backward against the formulas in 64 bits, on the GPU."""
import math

import pytest
import torch

import grxcp_amd as g
from helpers import say
from paged_cases import F32, Workspace, desc

pytestmark = pytest.mark.gpu
BF16, F16, FP32 = torch.bfloat16, torch.float16, torch.float32
STEP = {BF16: 2.0 ** -8, F16: 2.0 ** -11, FP32: F32}       # half a step, relative
LEAST = {BF16: 2.0 ** -134, F16: 2.0 ** -25, FP32: 2.0 ** -150}


# ---- in 64 bits -----------------------------------------------------------------

def turn(x, angle, pairs, way=1.0):
    """Rows of x [b, h, s, d] with their first 2 * angle.shape[-1] values turned."""
    n = 2 * angle.shape[-1]
    c, s = angle.cos()[:, None], way * angle.sin()[:, None]
    y = x.clone()
    i, j = (slice(0, n, 2), slice(1, n, 2)) if pairs else (slice(0, n // 2), slice(n // 2, n))
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    return y


def reach(x, rotary, pairs):
    """|x| plus the |value| that each is turned with: what relative errors act on."""
    a = x.abs()
    y = a.clone()
    i, j = ((slice(0, rotary, 2), slice(1, rotary, 2)) if pairs
            else (slice(0, rotary // 2), slice(rotary // 2, rotary)))
    y[..., i] = y[..., j] = a[..., i] + a[..., j]
    return y


def angles(positions, freq):
    return positions.double()[..., None] * freq.double()


def forward_ref(x, gain, eps, angle, pairs):
    x = x.double()
    if gain is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gain.double()
    return turn(x, angle, pairs), x


def norm_error(d):
    """Relative error of n * gamma in fp32: a sum of d positive products (d half steps, half of
    that after the root), the root's and the division's two steps, two products."""
    return (d / 2 + 8) * F32


TURN = 2.0 ** -21        # of a cosine or a sine (polynomial and the angle's rounding below 2^-22), its product and sum


# ---- calls ---------------------------------------------------------------------

class Case:
    def __init__(self, seed, dtype, b, s, hq, hk, d, rotary, pairs, norm, first=0, packed=True, scale=1.0, eps=1e-6):
        gen = torch.Generator().manual_seed(seed)
        self.dtype, self.b, self.s, self.hq, self.hk, self.d = dtype, b, s, hq, hk, d
        self.rotary, self.pairs, self.norm, self.eps = rotary, pairs, norm, eps

        def rows(heads, extra=0):
            t = torch.randn((b, s, heads + extra, d), generator=gen).mul(scale).to(dtype).cuda()
            return t.transpose(1, 2)

        if packed:
            p = rows(hq + 2 * hk)
            self.q, self.k = p[:, :hq], p[:, hq:hq + hk]
            self.packed = p
        else:
            self.q, self.k = rows(hq).contiguous(), rows(hk).contiguous()
        self.dyq, self.dyk = rows(hq), rows(hk)
        self.qg, self.kg = ((1 + 0.3 * torch.randn(d, generator=gen)).to(dtype).cuda() for _ in range(2))
        self.positions = (torch.randint(0, first + 1, (b, 1), generator=gen) + torch.arange(s)).int().cuda()
        self.freq = (1e4 ** (-torch.arange(0, rotary, 2).double() / max(rotary, 1))).float().cuda()

    def gains(self):
        if not self.norm:
            return None, None, None
        return desc(self.qg), self.qg.data_ptr(), self.kg.data_ptr()

    def how(self):
        return (self.eps, g.ROPE_PAIRS if self.pairs else g.ROPE_HALVES, self.rotary,
                self.positions.data_ptr() if self.rotary else None, self.freq.data_ptr() if self.rotary else None)

    def keys(self, *pairs):
        """The key arguments, or as many None where there are no keys."""
        out = []
        for t in pairs:
            out += [desc(t), t.data_ptr()] if self.hk else [None, None]
        return out

    def forward(self, dnn, yq, yk):
        w, qg, kg = self.gains()
        kg = kg if self.hk else None
        g.check(dnn.qk_norm_rope(desc(self.q), self.q.data_ptr(), *self.keys(self.k), w, qg, kg, *self.how(),
                                 desc(yq), yq.data_ptr(), *self.keys(yk)), "qk_norm_rope")
        torch.cuda.synchronize()

    def backward(self, dnn, dq, dk, dqg, dkg, ws=None):
        w, qg, kg = self.gains()
        kg = kg if self.hk else None
        size = dnn.qk_norm_rope_workspace(desc(self.q), desc(self.k) if self.hk else None, w)
        ws = ws or Workspace(size)
        g.check(dnn.qk_norm_rope_backward(
            desc(self.q), self.q.data_ptr(), *self.keys(self.k), w, qg, kg, *self.how(), desc(self.dyq),
            self.dyq.data_ptr(), *self.keys(self.dyk), desc(dq), dq.data_ptr(), *self.keys(dk),
            dqg.data_ptr() if dqg is not None else None, dkg.data_ptr() if dkg is not None else None, ws.p, ws.size),
            "qk_norm_rope_backward")
        torch.cuda.synchronize()

    def sides(self):
        return [(self.q, self.qg, self.dyq)] + ([(self.k, self.kg, self.dyk)] if self.hk else [])


def within(got, want, bound, what):
    got, want = got.cpu().double(), want.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    off = (got - want).abs() - bound.cpu()
    assert not (off > 0).any(), f"{what}: {off.max().item():.3g} past the bound"


def check_forward(dnn, c, what, inplace=False):
    want = [forward_ref(x.cpu(), gain.cpu() if c.norm else None, c.eps, angles(c.positions.cpu(), c.freq.cpu()), c.pairs)
            for x, gain, _ in c.sides()]
    outs = (c.q, c.k) if inplace else (torch.full_like(c.q, math.nan), torch.full_like(c.k, math.nan))
    c.forward(dnn, *outs)
    u = STEP[c.dtype]
    for got, (y, before) in zip(outs, want):
        bound = u * y.abs() + (1 + u) * reach(before, c.rotary, c.pairs) * (norm_error(c.d) + TURN) + LEAST[c.dtype]
        within(got, y, bound, what)
    return outs


def backward_ref(x, gain, dy, eps, angle, pairs, rotary):
    """dx, its bound without its own rounding, and dgamma with sum |g n|."""
    u = turn(dy.double(), angle, pairs, -1.0)
    size = reach(dy.double(), rotary, pairs)
    if gain is None:
        return u, size * TURN, None, None
    x, gain, d = x.double(), gain.double(), x.shape[-1]
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    n, w = x * r, u * gain
    m = (w * n).mean(-1, keepdim=True)
    dx = r * (w - n * m)
    mass = size * gain.abs()
    rel = 2 * norm_error(d) + TURN
    # the mean is a sum of d products, each off by rel of what it is made of, and rounded d times
    off = r * (rel * mass + n.abs() * (2 * rel + d * F32) * (mass * n.abs()).mean(-1, keepdim=True)) + rel * dx.abs()
    return dx, off, (u * n).sum((0, 1, 2)), ((size * n.abs()).sum((0, 1, 2)), rel)


def check_backward(dnn, c, what, inplace=None):
    angle = angles(c.positions.cpu(), c.freq.cpu())
    want = [backward_ref(x.cpu(), gain.cpu() if c.norm else None, dy.cpu(), c.eps, angle, c.pairs, c.rotary)
            for x, gain, dy in c.sides()]
    outs = {None: (torch.full_like(c.q, math.nan), torch.full_like(c.k, math.nan)), "x": (c.q, c.k),
            "dy": (c.dyq, c.dyk)}[inplace]
    gains = [torch.full((c.d,), math.nan, device="cuda") if c.norm else None for _ in range(2)]
    if not c.hk:
        gains[1] = None
    c.backward(dnn, *outs, *gains)
    u = STEP[c.dtype]
    rows = [c.b * c.s * c.hq, c.b * c.s * c.hk]
    for got, gg, (dx, off, dgain, mass), count in zip(outs, gains, want, rows):
        within(got, dx, u * dx.abs() + (1 + u) * off + LEAST[c.dtype], what)
        if c.norm:
            # a sum of `count` terms in any order rounds each at most count times
            within(gg, dgain, mass[0] * (mass[1] + (count + 2) * F32), what + ", gains")
    return outs, gains


CASES = [
    # dtype, b, s, hq, hk, d, rotary, pairs, norm, first position, packed
    (BF16, 3, 1, 32, 8, 128, 128, False, True, 100000, True),
    (BF16, 2, 77, 6, 2, 128, 128, False, True, 0, True),
    (F16, 1, 1, 1, 1, 64, 64, True, True, 5, False),
    (F16, 2, 33, 5, 1, 256, 256, False, True, 0, True),
    (FP32, 2, 19, 3, 3, 64, 32, True, False, 9, False),
    (FP32, 1, 130, 4, 2, 128, 96, False, True, 70000, True),
    (FP32, 1, 65, 2, 1, 256, 16, False, True, 3, False),
    (BF16, 1, 45, 7, 0, 64, 48, False, True, 0, True),         # queries alone
    (BF16, 2, 9, 4, 4, 128, 0, False, True, 0, False),         # norm alone
    (F16, 2, 9, 4, 4, 256, 240, True, False, 11, True),        # rotation alone
    (BF16, 5, 600, 3, 2, 64, 64, False, True, 0, False),
    (BF16, 4, 700, 20, 5, 128, 64, True, True, 0, True),       # rows enough for tiles of many tokens
    (F16, 2, 1500, 40, 8, 128, 128, False, True, 0, True),
    (FP32, 1, 9001, 9, 1, 64, 64, True, True, 0, False),
    (F16, 1, 3001, 7, 1, 256, 256, False, True, 0, False),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_forward_against_64_bits(dnn, case):
    say(f"qk_norm_rope {CASES[case]}")
    c = Case(300 + case, *CASES[case])
    check_forward(dnn, c, str(CASES[case]))


@pytest.mark.parametrize("case", range(len(CASES)))
def test_backward_against_64_bits(dnn, case):
    say(f"qk_norm_rope backward {CASES[case]}")
    c = Case(400 + case, *CASES[case])
    check_backward(dnn, c, str(CASES[case]))


LARGE = [
    # calls past the caches: 48 MB and more, rows that end inside a pass
    (BF16, 2, 2003, 40, 10, 128, 128, False, True, 0, True),
    (BF16, 2, 4099, 40, 9, 64, 64, False, True, 0, True),
    (F16, 1, 5003, 33, 7, 128, 48, False, True, 0, False),
    (BF16, 3, 1111, 23, 7, 256, 96, False, True, 7, True),
    (FP32, 1, 4999, 17, 3, 128, 128, False, True, 0, False),
    (FP32, 2, 3001, 33, 0, 64, 32, True, True, 0, True),
    (BF16, 1, 8193, 44, 5, 64, 48, True, False, 0, True),
    (FP32, 5, 501, 15, 5, 256, 240, False, False, 0, False),
]


@pytest.mark.parametrize("case", range(len(LARGE)))
def test_large_calls(dnn, case):
    say(f"qk_norm_rope {LARGE[case]}")
    c = Case(500 + case, *LARGE[case])
    check_forward(dnn, c, str(LARGE[case]))
    say(f"qk_norm_rope backward {LARGE[case]}")
    check_backward(dnn, c, str(LARGE[case]))


def test_large_calls_in_place(dnn):
    args = (F16, 1, 8195, 41, 8, 64, 64, False, True, 0, True)
    for where in (None, "x", "dy"):
        say(f"qk_norm_rope in place, large: {where}")
        c = Case(510, *args)
        if where:
            check_backward(dnn, c, "in place", inplace=where)
        else:
            v = c.packed[:, 49:].clone()
            check_forward(dnn, c, "in place", inplace=True)
            assert torch.equal(c.packed[:, 49:], v)


def test_the_gradient_is_that_of_differences():
    """backward_ref against central differences of forward_ref (host, 64 bits)."""
    gen = torch.Generator().manual_seed(1)
    for pairs, norm, rotary in ((False, True, 64), (True, True, 32), (True, False, 64)):
        x, dy = (torch.randn((2, 3, 5, 64), generator=gen, dtype=torch.float64) for _ in range(2))
        gain = 1 + 0.3 * torch.randn(64, generator=gen, dtype=torch.float64)
        angle = angles(torch.tensor([[3, 4, 5, 6, 7], [100, 2, 1, 0, -9]]), 0.7 ** torch.arange(rotary // 2).double())
        eps, h = 1e-3, 1e-5
        dx, _, dgain, _ = backward_ref(x, gain if norm else None, dy, eps, angle, pairs, rotary)

        def loss(x, gain):
            return (forward_ref(x, gain if norm else None, eps, angle, pairs)[0] * dy).sum().item()  # noqa: B023

        for _ in range(4):
            v = torch.randn(x.shape, generator=gen, dtype=torch.float64)
            num = (loss(x + h * v, gain) - loss(x - h * v, gain)) / (2 * h)
            assert abs(num - (dx * v).sum().item()) < 1e-6 * (1 + abs(num))
            if norm:
                w = torch.randn(64, generator=gen, dtype=torch.float64)
                num = (loss(x, gain + h * w) - loss(x, gain - h * w)) / (2 * h)
                assert abs(num - (dgain * w).sum().item()) < 1e-6 * (1 + abs(num))


def test_in_place(dnn):
    """yq over q and yk over k inside one packed projection, whose values stay as they were;
    gradients over the inputs and over the outputs' gradients."""
    args = (BF16, 2, 50, 4, 2, 128, 128, False, True, 10)
    c = Case(20, *args)
    v = c.packed[:, 6:].clone()
    check_forward(dnn, c, "in place", inplace=True)
    assert torch.equal(c.packed[:, 6:], v)
    for where in ("x", "dy"):
        say(f"qk_norm_rope backward in place over {where}")
        check_backward(dnn, Case(21, *args), where, inplace=where)


def test_the_same_bits_every_time(dnn):
    c = Case(22, BF16, 2, 1100, 20, 4, 128, 128, False, True)
    runs = []
    for fill in (0, 0xFF):
        dq, dk = torch.empty_like(c.q), torch.empty_like(c.k)
        dqg, dkg = torch.empty(128, device="cuda"), torch.empty(128, device="cuda")
        ws = Workspace(dnn.qk_norm_rope_workspace(desc(c.q), desc(c.k), desc(c.qg)))
        ws.t.fill_(fill)
        c.backward(dnn, dq, dk, dqg, dkg, ws)
        runs.append((dq, dk, dqg, dkg))
    for a, b in zip(*runs):
        assert torch.equal(a, b)
    # one gain's gradient alone, and none: the others are not touched
    for one in ((runs[0][2].clone().zero_(), None), (None, runs[0][3].clone().zero_()), (None, None)):
        dq, dk = torch.empty_like(c.q), torch.empty_like(c.k)
        c.backward(dnn, dq, dk, *one)
        assert torch.equal(dq, runs[0][0]) and torch.equal(dk, runs[0][1])
        for x, y in zip(one, runs[0][2:]):
            assert x is None or torch.equal(x, y)


def test_strides_and_bounds(dnn):
    """Rows with pitches of their own, NaN around every one of them; nothing but them is
    read or written."""
    gen = torch.Generator().manual_seed(23)
    c = Case(23, F16, 2, 13, 3, 2, 64, 64, False, True, packed=False)

    def spread(t):
        b, h, s, d = t.shape
        big = torch.full((b, h + 1, s + 2, d + 8), math.nan, dtype=t.dtype, device="cuda")
        view = big[:, :h, 1:s + 1, :d]
        view.copy_(t)
        return big, view

    (_, c.q), (_, c.k) = spread(c.q), spread(c.k)
    (_, c.dyq), (_, c.dyk) = spread(c.dyq), spread(c.dyk)
    (bq, yq), (bk, yk) = spread(torch.randn(c.q.shape, generator=gen)), spread(torch.randn(c.k.shape, generator=gen))
    bq.fill_(7.0)
    bk.fill_(7.0)
    yq, yk = (x.half() for x in (yq, yk))
    (bq, yq), (bk, yk) = spread(yq), spread(yk)
    c.forward(dnn, yq, yk)
    for y, x, gain in ((yq, c.q, c.qg), (yk, c.k, c.kg)):
        want, before = forward_ref(x.cpu(), gain.cpu(), c.eps, angles(c.positions.cpu(), c.freq.cpu()), False)
        u = STEP[F16]
        within(y, want, u * want.abs() + (1 + u) * reach(before, 64, False) * (norm_error(64) + TURN) + LEAST[F16], "spread")
    for big, y in ((bq, yq), (bk, yk)):
        assert int(torch.isnan(big).sum()) == big.numel() - y.numel()
    (bq, dq), (bk, dk) = spread(yq), spread(yk)
    gains = [torch.empty(64, device="cuda") for _ in range(2)]
    c.backward(dnn, dq, dk, *gains)
    assert torch.isfinite(gains[0]).all() and torch.isfinite(gains[1]).all()
    for big, y in ((bq, dq), (bk, dk)):
        assert torch.isfinite(y).all() and int(torch.isnan(big).sum()) == big.numel() - y.numel()


def test_a_broadcast_input(dnn):
    """Keys that all heads share: one row read by each head (stride 0)."""
    c = Case(24, FP32, 2, 6, 4, 1, 64, 64, True, True, packed=False)
    c.k = c.k.expand(2, 4, 6, 64)
    c.hk = 4
    c.dyk = torch.randn((2, 4, 6, 64), generator=torch.Generator().manual_seed(1)).cuda()
    check_forward(dnn, c, "broadcast")[1]
    outs = torch.full((2, 4, 6, 64), math.nan, device="cuda")
    gains = [torch.empty(64, device="cuda") for _ in range(2)]
    c.backward(dnn, torch.empty_like(c.q), outs, *gains)
    dx, off, dgain, mass = backward_ref(c.k.cpu(), c.kg.cpu(), c.dyk.cpu(), c.eps, angles(c.positions.cpu(), c.freq.cpu()),
                                        True, 64)
    within(outs, dx, F32 * dx.abs() + (1 + F32) * off + LEAST[FP32], "broadcast, backward")
    within(gains[1], dgain, mass[0] * (mass[1] + 50 * F32), "broadcast, gains")


def test_far_positions_and_signs(dnn):
    """Angles of positions up to 2^31 - 1 and back below 0, frequencies from 1 to 10^-7."""
    c = Case(25, FP32, 1, 8, 2, 1, 128, 128, False, False)
    c.positions = torch.tensor([[2 ** 31 - 1, -2 ** 31, 2 ** 24 + 1, 10 ** 9 + 7, -3, 0, 1, 123456789]],
                               dtype=torch.int32, device="cuda")
    c.freq = (10.0 ** -torch.linspace(0, 7, 64)).float().cuda()
    check_forward(dnn, c, "far")
    # (64 bits lose 2^31 * 2^-53 of an angle: nothing here)
    check_backward(dnn, c, "far")


def test_specials(dnn):
    """Rows of zeros, of NaN and infinities, of values whose squares overflow, and eps 0;
    their neighbours are as without them."""
    c = Case(26, BF16, 1, 10, 2, 1, 64, 64, False, True, packed=False, eps=1e-6)
    c.q[0, 0, 0] = 0.0
    c.q[0, 0, 1, 5] = math.nan
    c.q[0, 1, 2, 7] = math.inf
    c.q[0, 1, 3] = 2.0 ** 100
    c.k[0, 0, 4] = 2.0 ** -100
    yq, yk = torch.empty_like(c.q), torch.empty_like(c.k)
    c.forward(dnn, yq, yk)
    assert (yq[0, 0, 0] == 0).all() and torch.isnan(yq[0, 0, 1]).all()
    assert torch.isnan(yq[0, 1, 2, 7]) and torch.isnan(yq[0, 1, 2, 39])        # inf * 0, and its partner
    assert (yq[0, 1, 3] == 0).all()                                            # scaled by 0
    assert torch.isfinite(yk).all()
    fine = torch.ones(1, 2, 10, dtype=torch.bool)
    fine[0, 0, 0] = fine[0, 0, 1] = fine[0, 1, 2] = fine[0, 1, 3] = False
    want, before = forward_ref(c.q.cpu(), c.qg.cpu(), c.eps, angles(c.positions.cpu(), c.freq.cpu()), False)
    u = STEP[BF16]
    bound = u * want.abs() + (1 + u) * reach(before, 64, False) * (norm_error(64) + TURN) + LEAST[BF16]
    assert ((yq.cpu().double() - want).abs() <= bound)[fine].all()


def test_no_rows(dnn):
    """No tokens or no heads: nothing is written, and the gains' gradients are sums over nothing."""
    for b, s, hq in ((0, 5, 2), (2, 0, 2), (2, 5, 0)):
        c = Case(27, BF16, b, s, hq, 0, 64, 64, False, True, packed=False)
        dqg = torch.full((64,), math.nan, device="cuda")
        c.forward(dnn, torch.empty_like(c.q), None)
        c.backward(dnn, torch.empty_like(c.q), None, dqg, None)
        assert (dqg == 0).all()


def test_captured(gpu):
    """Forward and backward in one graph; replays follow the inputs and positions of their time."""
    dnn = g.Dnn()
    c = Case(28, BF16, 2, 300, 8, 2, 128, 128, False, True)
    yq, yk, dq, dk = (torch.empty_like(t) for t in (c.q, c.k, c.q, c.k))
    dqg, dkg = (torch.empty(128, device="cuda") for _ in range(2))
    qd, kd, wd = desc(c.q), desc(c.k), desc(c.qg)
    yqd, ykd, dyqd, dykd = (desc(t) for t in (yq, yk, c.dyq, c.dyk))
    dqd, dkd = desc(dq), desc(dk)
    ws = Workspace(dnn.qk_norm_rope_workspace(qd, kd, wd))
    outs = (yq, yk, dq, dk, dqg, dkg)

    def calls():
        g.check(dnn.qk_norm_rope(qd, c.q.data_ptr(), kd, c.k.data_ptr(), wd, c.qg.data_ptr(), c.kg.data_ptr(),
                                 *c.how(), yqd, yq.data_ptr(), ykd, yk.data_ptr()))
        g.check(dnn.qk_norm_rope_backward(qd, c.q.data_ptr(), kd, c.k.data_ptr(), wd, c.qg.data_ptr(),
                                          c.kg.data_ptr(), *c.how(), dyqd, c.dyq.data_ptr(), dykd, c.dyk.data_ptr(),
                                          dqd, dq.data_ptr(), dkd, dk.data_ptr(), dqg.data_ptr(), dkg.data_ptr(),
                                          ws.p, ws.size))

    calls()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    say("capturing qk_norm_rope")
    with torch.cuda.graph(graph, stream=side):
        dnn.set_stream(torch.cuda.current_stream().cuda_stream)
        calls()
    dnn.set_stream(None)
    for step in range(4):
        c.positions += 17
        c.packed.mul_(-1.25)
        calls()
        torch.cuda.synchronize()
        want = [t.clone() for t in outs]
        for t in outs:
            t.fill_(math.nan)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, outs):
            assert torch.equal(a, b), f"replay {step}"
    del graph
    dnn.close()


def test_a_row_does_not_depend_on_its_neighbours(dnn):
    """NaN, infinities and tiny rows beside it (eps 0): the other rows' bits stay."""
    c = Case(29, BF16, 1, 40, 8, 2, 64, 64, False, True, packed=False, eps=0.0)
    runs = []
    for odd in (False, True):
        if odd:
            c.q[0, 3, 5], c.q[0, 4, 5, 7], c.dyq[0, 2, 5, 1] = 2.0 ** -40, math.nan, math.inf
        yq, yk, dq, dk = (torch.empty_like(t) for t in (c.q, c.k, c.q, c.k))
        c.forward(dnn, yq, yk)
        c.backward(dnn, dq, dk, None, None)
        runs.append((yq, yk, dq, dk))
    same = torch.ones(8, 40, dtype=torch.bool)
    same[3, 5] = same[4, 5] = same[2, 5] = False
    for i, (a, b) in enumerate(zip(*runs)):
        if i % 2 == 0:
            a, b = a[0, same], b[0, same]
        assert torch.equal(a, b), i
    # a row of 2^-40 alone is normalised like any other: dx is 2^40 times a row's of ones
    assert torch.isfinite(runs[1][0][0, 3, 5]).all() and torch.isfinite(runs[1][2][0, 3, 5]).all()


def test_rows_far_apart(dnn):
    """A batch that lies 2^31 bytes behind the other."""
    c = Case(30, BF16, 2, 3, 2, 1, 128, 128, False, True, packed=False)
    far = torch.empty((1 << 31) + 4096, dtype=BF16, device="cuda")
    wide = [(1 << 30) + 2048, 128, 512, 1]

    def spread(t, at):
        v = far.as_strided(t.shape, wide, at)
        v.copy_(t)
        return v

    q, k = c.q, c.k
    yq, yk = torch.empty_like(q), torch.empty_like(k)
    c.forward(dnn, yq, yk)
    c.q, c.k = spread(q, 0), spread(k, 256)
    outs = (far.as_strided(q.shape, wide, 1024 * 1024), far.as_strided(k.shape, wide, 1024 * 1024 + 256))
    c.forward(dnn, *outs)
    assert torch.equal(outs[0], yq) and torch.equal(outs[1], yk)


@pytest.mark.parametrize("args", [CASES[i] for i in (1, 5, 11, 12, 13, 14)] + [c for c in LARGE if c[8]])
def test_the_gains_gradients_hold_every_row(dnn, args):
    """The sums over rows by their real depth: a lane adds 15 rows at most in these calls, then its
    row's lanes (4 steps), the waves (3), and of up to 768 workgroups' parts 12 to a lane, two
    steps over lanes, 15 over waves: 51 roundings of what is summed, where 64 are allowed. A
    wave's rows, a 3072nd of them, make six times that or more of a difference."""
    say(f"qk_norm_rope, gains {args}")
    c = Case(600, *args)
    angle = angles(c.positions.cpu(), c.freq.cpu())
    gains = [torch.full((c.d,), math.nan, device="cuda") for _ in range(1 + (c.hk > 0))]
    c.backward(dnn, torch.empty_like(c.q), torch.empty_like(c.k), gains[0], gains[1] if c.hk else None)
    for got, (x, gain, dy) in zip(gains, c.sides()):
        _, _, want, mass = backward_ref(x.cpu(), gain.cpu(), dy.cpu(), c.eps, angle, c.pairs, c.rotary)
        bound = mass[0] * (mass[1] + 64 * F32)
        within(got, want, bound, str(args))
        assert bound.max() < 0.05 * want.abs().median()


def test_small_rows_with_large_gains(dnn):
    """Gains whose product with 1 / root lies past fp32's range, either way, where y does not."""
    for scale, gain in ((2.0 ** -60, 2.0 ** 75), (2.0 ** 55, 2.0 ** -85)):
        c = Case(31, FP32, 1, 9, 3, 2, 128, 64, False, True, packed=False, scale=scale, eps=0.0)
        for t in (c.qg, c.kg):
            t.mul_(gain)
        check_forward(dnn, c, f"rows of {scale}, gains of {gain}")
