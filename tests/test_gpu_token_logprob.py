"""grxdnnTokenLogProbForward / Backward against the formulas in 64 bits, on the GPU."""
import math

import pytest
import torch

import grxcp_amd as g
from helpers import say
from paged_cases import Workspace, desc, ints

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}
TINY = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -150}


def forward(dnn, x, tokens, top=0, entropy=True, expect=g.SUCCESS):
    rows = x.numel() // x.shape[-1]
    xd = desc(x)
    out = [torch.full((rows,), 7.5, device="cuda") for _ in range(3)]
    best = torch.full((rows, top), 7.5, device="cuda")
    index = torch.full((rows, top), -7, dtype=torch.int32, device="cuda")
    ws = Workspace(dnn.token_logprob_workspace(xd, top))
    st = dnn.token_logprob(xd, x.data_ptr(), None if tokens is None else tokens.data_ptr(),
                           None if tokens is None else out[0].data_ptr(), out[1].data_ptr(),
                           out[2].data_ptr() if entropy else None, top, best.data_ptr() if top else None,
                           index.data_ptr() if top else None, ws.p, ws.size)
    assert st == expect, g.STATUS[st]
    torch.cuda.synchronize()
    return out + [best, index]


def order(x, top):
    """The first `top` places of every row by (NaN, value) downwards, then place upwards."""
    key = x.masked_fill(torch.isnan(x), math.inf) + 0.0
    nan = torch.isnan(x)
    places = []
    for r in range(x.shape[0]):
        idx = torch.argsort(-key[r], stable=True)
        if nan[r].any():
            idx = torch.cat([idx[nan[r][idx]], idx[~nan[r][idx]]])
        places.append(idx[:top])
    return torch.stack(places)


def check_forward(dnn, x, tokens=None, top=0, entropy=True, logits=None):
    """x: a device tensor whose last dimension is the vocabulary."""
    got = forward(dnn, x, None if tokens is None else ints(tokens), top, entropy)
    h = x.cpu().double().reshape(-1, x.shape[-1])
    V = h.shape[1]
    m = h.amax(1, keepdim=True)
    # (not below the lowest value, so that a row of only -inf has sum 0)
    d = h - m.clamp(min=-1.7e308)
    total = d.exp().sum(1, keepdim=True)     # +inf in the row: inf - inf
    logp, lse = d - total.log(), (m + total.log())[:, 0]
    lse[torch.isnan(total[:, 0])] = math.nan
    p = d.exp() / total
    H = -torch.where(p == 0, 0.0, p * logp).sum(1)
    # d = x - m is one rounding, e^d follows |d| half steps and a few of its own; the
    # sum of positive terms keeps the largest of those that weigh. 32 half steps stand
    # for exp, the sum's tree and the log.
    span = (d.abs().nan_to_num(posinf=0.0) * p.nan_to_num()).sum(1)
    rel = span * 2.0 ** -23 + 32 * HALF[F32]
    ls = total.log().abs()[:, 0].nan_to_num(posinf=0.0)
    near(got[1], lse, rel + 2 * HALF[F32] * (lse.abs() + ls), "logSumExp")
    if entropy:
        # log s - t / s: both off by rel, t / s = sum p d
        near(got[2], H, 2 * rel * (1 + span) + 4 * HALF[F32] * (H.abs() + ls), "entropy")
    if tokens is not None:
        want = torch.tensor([logp[r, t].item() if 0 <= t < V else 0.0 for r, t in enumerate(tokens)], dtype=torch.float64)
        near(got[0], want, rel + 4 * HALF[F32] * (want.abs().nan_to_num(posinf=0.0) + ls), "logProb")
    if top:
        index = order(h, top)
        assert torch.equal(got[4].cpu().long(), index), "topIndex"
        want = logp.gather(1, index)
        near(got[3], want, rel[:, None] + 4 * HALF[F32] * (want.abs().nan_to_num(posinf=0.0, neginf=0.0) + ls[:, None]),
             "topLogProb")
    return lse, H


def near(got, want, bound, what):
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN"
    far = torch.isinf(want)
    assert torch.equal(got[far], want[far]), f"{what}: infinities"
    fine = ~far & ~torch.isnan(want)
    off = ((got - want).abs() - bound.expand_as(want))[fine]
    assert not (off > 0).any(), f"{what}: {off.max().item():.3g} past the bound"


def logits(gen, shape, dtype, scale=3.0):
    return torch.randn(shape, generator=gen).mul(scale).to(dtype).cuda()


CASES = [
    # dtype, rows, vocabulary, alternatives
    (F32, 5, 1, 1), (BF16, 3, 2, 2), (F16, 4, 7, 7), (F32, 3, 63, 5), (BF16, 2, 64, 64), (F16, 2, 65, 64),
    (BF16, 70, 1000, 20), (F32, 33, 2049, 1), (F16, 9, 4096, 64), (BF16, 300, 8191, 3), (F32, 17, 16385, 40),
    (F16, 8, 32000, 5), (BF16, 5, 32001, 64), (F32, 3, 50257, 20), (BF16, 1, 131072, 8), (F16, 2, 131071, 64),
    (F32, 1, 262145, 10), (BF16, 1, 1 << 20, 33), (F32, 1100, 300, 0), (BF16, 600, 5000, 4), (F16, 2, 9000, 0),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_forward(dnn, case):
    dtype, rows, vocab, top = CASES[case]
    gen = torch.Generator().manual_seed(case)
    x = logits(gen, (rows, vocab), dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=gen).tolist()
    tokens[0] = vocab - 1
    say(f"logprob {CASES[case]}")
    check_forward(dnn, x, tokens, top)


def test_rows_without_a_token_and_optional_outputs(dnn):
    gen = torch.Generator().manual_seed(30)
    x = logits(gen, (6, 999), BF16)
    check_forward(dnn, x, [-1, 999, 998, 0, -2 ** 31, 2 ** 31 - 1], 3)
    check_forward(dnn, x, None, 0, entropy=False)
    check_forward(dnn, x, None, 64, entropy=False)
    check_forward(dnn, x, [1] * 6, 0, entropy=False)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shift,pitch", [(0, 1003), (1, 1007), (3, 1008), (8, 1100)])
def test_padded_rows_off_16_bytes(dnn, dtype, shift, pitch):
    """Rows of a wider array that starts anywhere; what lies between is NaN."""
    gen = torch.Generator().manual_seed(31)
    flat = torch.full((shift + 2 * 3 * pitch + 8,), math.nan, dtype=dtype, device="cuda")
    x = torch.as_strided(flat, (2, 3, 1003), (3 * pitch, pitch, 1), shift)
    x.copy_(logits(gen, (2, 3, 1003), dtype))
    check_forward(dnn, x, [5, 1002, 0, 1, 2, -1], 9)


@pytest.mark.parametrize("vocab", [500, 20000, 140000])
@pytest.mark.parametrize("kind", ["equal", "two_values", "rising", "falling", "one_lane", "end", "minus_zero"])
def test_alternatives_in_awkward_orders(dnn, vocab, kind):
    """Rows where many elements tie, come in order, or lie where one thread reads."""
    at = torch.arange(vocab)
    x = {"equal": torch.zeros(vocab), "two_values": (at % 3 == 1).float(), "rising": at / 64.0,
         "falling": -at / 64.0, "one_lane": torch.where(at % 2048 < 8, 4.0 + (at % 7), 0.0),
         "end": torch.where(at >= vocab - 70, 3.0, -1.0),
         "minus_zero": torch.where(at % 2 == 0, -0.0, 0.0)}[kind]
    for dtype in (F32, BF16):
        check_forward(dnn, x.to(dtype).expand(2, vocab).contiguous().cuda(), [0, vocab - 1], 64)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("vocab", [40, 5000, 70000])
def test_special_values(dnn, dtype, vocab):
    gen = torch.Generator().manual_seed(32)
    x = logits(gen, (8, vocab), dtype)
    low = torch.finfo(dtype).min
    x[0, : vocab - 2] = -math.inf            # a vocabulary mask
    x[1, :] = -math.inf
    x[2, vocab // 2] = math.nan
    x[3, 7] = math.inf
    x[4, :] = low                            # every logit the lowest value
    x[5, 3:] = low
    x[6, 11] = 300.0                         # all of the mass on one
    x[7, :] = torch.finfo(dtype).max
    check_forward(dnn, x, [0, 1, 2, 7, 4, 5, 11, vocab - 1], 6)


def grad_ref(x, tokens, lse, H, dlogp, dH):
    """The gradient and the bound on its error, from the fp32 lse and H that the call gets."""
    lp = x - lse[:, None]
    p = lp.exp()
    V = x.shape[1]
    one = torch.zeros_like(x)
    given = torch.tensor([0 <= t < V for t in tokens]) if tokens is not None else torch.zeros(len(x), dtype=torch.bool)
    for r, t in enumerate(tokens or []):
        if 0 <= t < V:
            one[r, t] = 1.0
    gl = torch.where(given, dlogp, 0.0)[:, None] if tokens is not None else torch.zeros(len(x), 1, dtype=torch.float64)
    dx = gl * (one - p)
    size = gl.abs() * (one + p)
    if dH is not None:
        term = torch.where(p > 0, p * (lp + H[:, None]), 0.0)
        dx = dx - dH[:, None] * term
        size = size + dH.abs()[:, None] * p * (lp.abs().nan_to_num(posinf=0.0) + H.abs()[:, None])
    # x - lse one rounding, e to it |lp| more, exp's and the products' own: 16 half steps
    return dx, size * (lp.abs().nan_to_num(posinf=0.0) * 2 + 16) * HALF[F32]


def backward(dnn, x, tokens, lse, H, dlogp, dH, dx, expect=g.SUCCESS):
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    st = dnn.token_logprob_backward(desc(x), x.data_ptr(), ptr(tokens), lse.data_ptr(), ptr(H), ptr(dlogp), ptr(dH),
                                    desc(dx), dx.data_ptr())
    assert st == expect, g.STATUS[st]
    torch.cuda.synchronize()


def check_backward(dnn, x, tokens, entropy, gen, inplace=False, dx=None):
    h = x.cpu().double().reshape(-1, x.shape[-1])
    rows = h.shape[0]
    lse = torch.logsumexp(h, 1).float()
    p = (h - lse.double()[:, None]).exp()
    H = -torch.where(p > 0, p * (h - lse.double()[:, None]), 0.0).sum(1).float() if entropy else None
    dlogp = torch.randn(rows, generator=gen) if tokens is not None else None
    dH = torch.randn(rows, generator=gen) if entropy else None
    up = lambda t: None if t is None else t.double()  # noqa: E731
    want, bound = grad_ref(h, tokens, lse.double(), up(H), up(dlogp), up(dH))
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    dtype = x.dtype
    dx = x if inplace else dx if dx is not None else torch.full_like(x, math.nan)
    backward(dnn, x, None if tokens is None else ints(tokens), dev(lse), dev(H), dev(dlogp), dev(dH), dx)
    got = dx.cpu().double().reshape(rows, -1)
    near(got, want, HALF[dtype] * (want.abs() + bound) + bound + TINY[dtype], "dx")


GRADS = [(F32, 5, 1), (BF16, 3, 8), (F16, 4, 7), (F32, 3, 63), (BF16, 2, 65), (BF16, 70, 1000), (F32, 33, 2049),
         (F16, 9, 4096), (BF16, 300, 8191), (F16, 8, 32000), (BF16, 5, 32001), (F32, 3, 50257), (F16, 2, 131071),
         (F32, 1100, 300), (BF16, 1, 1 << 20)]


@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("case", range(len(GRADS)))
def test_backward(dnn, case, entropy):
    dtype, rows, vocab = GRADS[case]
    gen = torch.Generator().manual_seed(200 + case)
    x = logits(gen, (rows, vocab), dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=gen).tolist()
    tokens[-1] = -1 if rows > 2 else vocab - 1
    say(f"logprob gradient {GRADS[case]} entropy={entropy}")
    check_backward(dnn, x, tokens, entropy, gen)


def test_backward_entropy_alone_and_in_place(dnn):
    gen = torch.Generator().manual_seed(33)
    check_backward(dnn, logits(gen, (7, 3001), BF16), None, True, gen)
    for dtype, vocab in ((BF16, 4096), (F32, 777), (F16, 50001)):
        check_backward(dnn, logits(gen, (5, vocab), dtype), [0, 1, 2, vocab - 1, -1], True, gen, inplace=True)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shift,pitch,dshift,dpitch", [(0, 1003, 1, 1003), (1, 1007, 0, 1008), (3, 1008, 3, 1100)])
def test_backward_padded_rows(dnn, dtype, shift, pitch, dshift, dpitch):
    gen = torch.Generator().manual_seed(34)
    flat = torch.full((shift + 6 * pitch + 8,), math.nan, dtype=dtype, device="cuda")
    x = torch.as_strided(flat, (2, 3, 1003), (3 * pitch, pitch, 1), shift)
    x.copy_(logits(gen, (2, 3, 1003), dtype))
    out = torch.full((dshift + 6 * dpitch + 8,), 7.0, dtype=dtype, device="cuda")
    dx = torch.as_strided(out, (2, 3, 1003), (3 * dpitch, dpitch, 1), dshift)
    check_backward(dnn, x, [5, 1002, 0, 1, 2, -1], True, gen, dx=dx)
    dx.fill_(7.0)
    assert (out == 7.0).all()                # nothing else was written


def test_backward_of_masked_and_padded_rows(dnn):
    """-inf logits get gradient 0; a row without a token and without the entropy term
    gets 0 whatever its logits are."""
    gen = torch.Generator().manual_seed(35)
    x = logits(gen, (4, 600), F32)
    x[0, 5:300] = -math.inf
    x[1, :599] = -math.inf
    check_backward(dnn, x, [0, 599, 3, 4], True, gen)
    x[2, 7], x[3] = math.nan, math.inf
    dx = torch.full_like(x, math.nan)
    lse, dl = torch.zeros(4, device="cuda"), torch.ones(4, device="cuda")
    lse[2:] = math.nan
    backward(dnn, x, ints([0, 599, -1, 600]), lse, None, dl, None, dx)
    assert (dx[2:] == 0).all() and torch.isfinite(dx).all()
    # with an entropy term for the first rows only
    dx.fill_(math.nan)
    H = torch.full_like(lse, math.nan)
    H[:2] = 1.0
    backward(dnn, x, ints([0, 599, -1, 600]), lse, H, dl, torch.tensor([0.5, 0.5, 0.0, -0.0], device="cuda"), dx)
    assert (dx[2:] == 0).all() and torch.isfinite(dx).all()


def test_gradient_against_differences(dnn):
    """f = sum_r a_r logProb_r + c_r entropy_r through the forward call itself, in fp32:
    central differences with h = 2^-6 on logits of size 1 are off by the third
    derivative (below 8 here) times h^2 / 6 and by the outputs' roundings, about
    2^-21 (|a| + |c| H), over h."""
    gen = torch.Generator().manual_seed(36)
    rows, vocab, h = 3, 40, 2.0 ** -6
    x = torch.randn((rows, vocab), generator=gen).mul(64).round().div(64)
    a, c = torch.randn(rows, generator=gen).double(), torch.randn(rows, generator=gen).double()
    tokens = [3, 39, 0]
    both = x.repeat(2 * vocab, 1, 1)
    for j in range(vocab):
        both[j, :, j] += h
        both[vocab + j, :, j] -= h
    out = forward(dnn, both.cuda(), ints(tokens * 2 * vocab))
    f = (a * out[0].cpu().double().reshape(-1, rows) + c * out[2].cpu().double().reshape(-1, rows))
    diff = ((f[:vocab] - f[vocab:]) / (2 * h)).T
    base = forward(dnn, x.cuda(), ints(tokens))
    dx = torch.empty_like(x, device="cuda")
    backward(dnn, x.cuda(), ints(tokens), base[1], base[2], a.float().cuda(), c.float().cuda(), dx)
    bound = (8 * h * h / 6 + 2.0 ** -21 * 5 / h) * (a.abs() + c.abs())[:, None]
    assert ((dx.cpu().double() - diff).abs() <= bound).all()


def test_more_rows_than_one_launch_wave(dnn):
    gen = torch.Generator().manual_seed(37)
    x = logits(gen, (70001, 9), BF16)
    tokens = torch.randint(-1, 9, (70001,), generator=gen).tolist()
    check_forward(dnn, x, tokens, 2)
    check_backward(dnn, x, tokens, True, gen)


def test_rows_beyond_32_bits(dnn):
    """Rows whose place in their array passes 2^31 elements."""
    gen = torch.Generator().manual_seed(38)
    flat = torch.empty(2 * (2 ** 30 + 8) + 2048, dtype=BF16, device="cuda")
    x = torch.as_strided(flat, (3, 2003), (2 ** 30 + 8, 1), 5)
    x.copy_(logits(gen, (3, 2003), BF16))
    check_forward(dnn, x, [1, 2, 2002], 5)
    check_backward(dnn, x, [1, 2, 2002], True, gen, inplace=True)
    del x, flat
    torch.cuda.empty_cache()


def test_captured_forward_and_backward(gpu):
    """Both calls in one graph, replayed on new logits with eager work between."""
    gen = torch.Generator().manual_seed(39)
    dnn = g.Dnn()
    x = logits(gen, (4, 40000), BF16)
    xd = desc(x)
    tokens = ints([1, 2, 39999, -1])
    logp, lse, H = (torch.zeros(4, device="cuda") for _ in range(3))
    best, index = torch.zeros((4, 5), device="cuda"), torch.zeros((4, 5), dtype=torch.int32, device="cuda")
    dl, dH, dx = torch.ones(4, device="cuda"), torch.full((4,), 0.5, device="cuda"), torch.empty_like(x)
    ws = Workspace(dnn.token_logprob_workspace(xd, 5))
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        dnn.set_stream(torch.cuda.current_stream().cuda_stream)
        g.check(dnn.token_logprob(xd, x.data_ptr(), tokens.data_ptr(), logp.data_ptr(), lse.data_ptr(), H.data_ptr(),
                                  5, best.data_ptr(), index.data_ptr(), ws.p, ws.size))
        g.check(dnn.token_logprob_backward(xd, x.data_ptr(), tokens.data_ptr(), lse.data_ptr(), H.data_ptr(),
                                           dl.data_ptr(), dH.data_ptr(), xd, dx.data_ptr()))
    dnn.set_stream(None)
    for rep in range(4):
        x.copy_(logits(gen, (4, 40000), BF16))
        torch.cuda.synchronize()
        say(f"replay {rep}")
        graph.replay()
        torch.cuda.synchronize()
        again = forward(dnn, x, tokens, 5)
        for a, b in zip((logp, lse, H, best, index), again):
            assert torch.equal(a, b), rep
        eager = torch.empty_like(x)
        backward(dnn, x, tokens, lse, H, dl, dH, eager)
        assert torch.equal(eager, dx), rep
    dnn.close()


@pytest.mark.parametrize("dtype,vocab", [(BF16, 1 << 24), (F32, (1 << 24) - 3)])
def test_the_largest_vocabulary(dnn, dtype, vocab):
    gen = torch.Generator().manual_seed(50)
    x = logits(gen, (2, vocab), dtype)
    x[1, -1] = 25.0
    check_forward(dnn, x, [vocab - 1, vocab], 64)
    check_backward(dnn, x, [vocab - 1, vocab], True, gen)


@pytest.mark.parametrize("vocab", [700, 33000, 200001])
@pytest.mark.parametrize("kind", ["few", "lowest_first", "steps", "minus_one", "rising_negative", "late_half", "blocks"])
@pytest.mark.parametrize("top", [5, 33, 64])
def test_alternatives_behind_masks_and_in_runs(dnn, vocab, kind, top):
    """Vocabulary masks that leave few tokens, runs of one value, values that rise or jump
    far into a row, so that more elements pass a threshold at once than a list holds."""
    gen = torch.Generator().manual_seed(vocab + top)
    at = torch.arange(vocab)
    n = torch.randn(vocab, generator=gen).mul(3)
    few = torch.full((vocab,), -math.inf)
    few[torch.randperm(vocab, generator=gen)[:7]] = n[:7]
    x = {"few": few, "lowest_first": torch.where(at < vocab // 3, -3.3e38, n), "steps": (at // 900).float() / 8 - 20,
         "minus_one": torch.where(at % 1000 == 999, -0.5, -1.0), "rising_negative": (at - vocab) / 128.0,
         "late_half": torch.where((at > vocab // 2) & (at // 8 % 2 == 0), 5.0, n.clamp(max=4.0)),
         "blocks": torch.where(at // 512 % 3 == 2, (at // 512).float() / 50, -7.0)}[kind]
    for dtype in (F32, BF16, F16):
        y = x.clamp(min=-65504.0) if dtype == F16 and kind == "lowest_first" else x
        check_forward(dnn, y.to(dtype).expand(2, vocab).contiguous().cuda(), [0, vocab - 1], top)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("vocab", [700, 40000])       # a row in one piece, in several
def test_rows_far_below_zero(dnn, dtype, vocab):
    """Finite rows whose logits all lie around -1126 log 2 = -780.5, where powers of two
    relative to 2^-1000 leave fp32: equal ones, spread ones, and one among -inf."""
    gen = torch.Generator().manual_seed(51)
    at = torch.arange(-800.0, -680.0, 0.5)[:, None]
    one = torch.full((len(at), vocab), -math.inf)
    one[torch.arange(len(at)), torch.randint(0, vocab, (len(at),), generator=gen)] = at[:, 0]
    spread = at + torch.randn((len(at), vocab), generator=gen)
    for x in (at.expand(-1, vocab), spread, one):
        check_forward(dnn, x.to(dtype).contiguous().cuda(), [r % vocab for r in range(len(at))], 3)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("vocab", [2, 700, 40000])
@pytest.mark.parametrize("rest", [100, 30])
def test_no_probability_above_one(dnn, dtype, vocab, rest):
    """One logit m with all of the mass, m = -64 .. 64 and the others `rest` below it: its log
    probability is never above 0 and the entropy never below, and both are right to 8 half
    steps of 1. (Two powers of two, each within a unit in the last place, 4 half steps, and
    their product, 1, make the sum; a log next to 1 moves by what the sum does. What the
    others add is in the reference: 40000 e^-30 is 2^-28.)"""
    m = torch.arange(-64.0, 65.0)
    x = (m[:, None] - rest).expand(-1, vocab).clone()
    at = torch.arange(len(m)) * 17 % vocab
    x[torch.arange(len(m)), at] = m
    x = x.to(dtype)
    say(f"one logit, {dtype}, {vocab}, the others {rest} below")
    logp, lse, H, best, index = (t.cpu() for t in forward(dnn, x.cuda(), ints(at.tolist()), 1))
    ref = x.double().log_softmax(1)
    want = ref.amax(1)
    entropy = -(ref.exp() * ref).sum(1)
    assert torch.equal(index[:, 0].long(), at)
    assert (logp <= 0).all() and (best <= 0).all() and (H >= 0).all()
    eight = 8 * HALF[F32]
    assert ((logp.double() - want).abs() <= eight).all() and torch.equal(best[:, 0], logp)
    assert ((H.double() - entropy).abs() <= eight + 2.0 ** -18 * entropy).all()
    assert ((lse.double() - (m.double() - want)).abs() <= eight + HALF[F32] * m.abs()).all()


def last_tokens(gen, dtype, rows, vocab, how):
    """[rows, 1, vocab] views of a wider array whose other elements are NaN."""
    shape = {"slice": (rows, 3, vocab), "transposed": (1, rows, vocab), "padded": (rows, 3, vocab + 5)}[how]
    wide = torch.full(shape, math.nan, dtype=dtype, device="cuda")
    x = {"slice": wide[:, -1:], "transposed": wide.transpose(0, 1), "padded": wide[:, 1:2, 5:]}[how]
    assert x.shape == (rows, 1, vocab)
    x.copy_(logits(gen, (rows, 1, vocab), dtype))
    return wide, x


@pytest.mark.parametrize("how", ["slice", "transposed", "padded"])
@pytest.mark.parametrize("dtype,vocab", [(BF16, 1000), (F32, 777), (F16, 33000)])
def test_a_dimension_of_one_before_the_vocabulary(dnn, dtype, vocab, how):
    """The last tokens' logits of a batch, where the rows' pitch is not the stride next to
    the vocabulary's."""
    gen = torch.Generator().manual_seed(52)
    wide, x = last_tokens(gen, dtype, 5, vocab, how)
    tokens = [0, vocab - 1, -1, 3, 4]
    check_forward(dnn, x, tokens, 4)
    out, dx = last_tokens(gen, dtype, 5, vocab, how)
    check_backward(dnn, x, tokens, True, gen, dx=dx)
    dx.fill_(math.nan)
    assert torch.isnan(out).all()                # nothing else was written


@pytest.mark.parametrize("how", ["slice", "transposed", "padded"])
def test_softmax_gelu_and_norms_of_a_dimension_of_one(dnn, how):
    """The same views in the other calls that take rows, against 64 bits: a few half steps
    of a sum of 1000 terms."""
    gen = torch.Generator().manual_seed(53)
    _, x = last_tokens(gen, F32, 6, 1000, how)
    gamma, beta = (torch.randn(1000, generator=gen).cuda() for _ in range(2))
    h, G, B = x.cpu().double()[:, 0], gamma.cpu().double(), beta.cpu().double()
    rms = h * (h.square().mean(1, keepdim=True) + 1e-5).rsqrt() * G
    layer = (h - h.mean(1, keepdim=True)) * (h.var(1, unbiased=False, keepdim=True) + 1e-5).rsqrt() * G + B
    xd, wd = desc(x), desc(gamma)
    for name, call, want in (
            ("softmax", lambda yd, y: dnn.softmax(xd, x.data_ptr(), yd, y), h.softmax(1)),
            ("gelu", lambda yd, y: dnn.gelu(0, xd, x.data_ptr(), yd, y), torch.nn.functional.gelu(h)),
            ("rmsnorm", lambda yd, y: dnn.rmsnorm(xd, x.data_ptr(), wd, gamma.data_ptr(), 1e-5, yd, y), rms),
            ("layernorm", lambda yd, y: dnn.layernorm(xd, x.data_ptr(), wd, gamma.data_ptr(), beta.data_ptr(), 1e-5,
                                                      yd, y), layer)):
        out, y = last_tokens(gen, F32, 6, 1000, how)
        say(f"{name}, {how}")
        g.check(call(desc(y), y.data_ptr()), name)
        torch.cuda.synchronize()
        assert torch.allclose(y.cpu().double()[:, 0], want, rtol=2.0 ** -16, atol=2.0 ** -18), name
        y.fill_(math.nan)
        assert torch.isnan(out).all(), name


@pytest.mark.parametrize("dtype,rows,vocab,top", [(F32, 32, 131072, 8), (F16, 300, 9000, 64), (BF16, 2500, 3000, 64)])
def test_same_bits_every_time(dnn, dtype, rows, vocab, top):
    """The alternatives are ranked in lists that fill in any order; whichever lane writes
    one, its log probability is the same number, and the token's."""
    gen = torch.Generator().manual_seed(55)
    x = logits(gen, (rows, vocab), dtype)
    tokens = x.float().argmax(1).int()
    first = forward(dnn, x, tokens, top)
    assert torch.equal(first[3][:, 0], first[0])
    shift = x.float().gather(1, first[4].long()).double() - first[3].double()
    assert (shift - shift[:, :1]).abs().max() <= 2.0 ** -19       # roundings of values below 16
    for i in range(20):
        for a, b in zip(first, forward(dnn, x, tokens, top)):
            assert torch.equal(a, b), i


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("vocab,top", [(1, 1), (3, 3), (700, 4), (40000, 64)])
def test_nan_in_the_first_place(dnn, dtype, vocab, top):
    """NaN is the largest alternative at place 0 as elsewhere, alone and among others."""
    gen = torch.Generator().manual_seed(54)
    x = logits(gen, (4, vocab), dtype)
    x[0, 0] = math.nan
    x[1, [0, -1]] = math.nan
    x[2, :] = math.nan
    x[3, 1:] = math.inf
    x[3, 0] = math.nan
    check_forward(dnn, x, [0, vocab - 1, 0, 0], top)
