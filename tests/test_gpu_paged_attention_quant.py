"""grxdnnPagedAttentionQuantizedForward against attention in 64 bits, on the GPU."""
import math

import pytest
import torch

import grxcp_amd as g
from helpers import say
from paged_cases import Workspace, ints
from quant_cases import QuantCache, append, attend, attention_ref, desc

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def query(gen, b, H, d, dtype, scale=1.0):
    return torch.randn((b, H, 1, d), generator=gen).mul(scale).to(dtype).cuda()


def check(dnn, c, q, scale, inplace=False):
    qh = q.cpu()
    o = q if inplace else torch.full_like(q, math.nan)
    attend(dnn, c, q, o, scale)
    got = o.cpu().double()[:, :, 0]
    for i, n in enumerate(c.n):
        K, V, there = c.rows(i, min(max(n, 0), c.width * c.page))
        ref, bound = attention_ref(qh[i, :, 0], K, V, scale, there)
        assert torch.equal(torch.isnan(got[i]), torch.isnan(ref)), f"sequence {i}: NaN where 64 bits have none"
        off = (got[i] - ref).abs() - bound
        assert not (off > 0).any(), f"sequence {i} of {n} slots: {off.max().item():.3g} past the bound"
    return o


CASES = [
    # dtype, d, query heads, key heads, page, block, tokmajor, lengths
    (BF16, 128, 8, 2, 16, 16, True, [1, 0, 15, 16, 17, 200]),
    (F16, 64, 4, 4, 16, 1, False, [31, 32, 33, 63, 64, 65, 127, 128, 129]),
    (BF16, 64, 6, 2, 7, 7, True, [5, 700, 0, 6]),
    (F16, 128, 16, 1, 1, 1, False, [3, 257, 1]),
    (BF16, 128, 17, 1, 64, 4, True, [500, 20]),
    (F16, 64, 32, 1, 256, 64, False, [1000]),
    (BF16, 64, 33, 1, 32, 8, False, [100, 4]),
    (BF16, 128, 40, 8, 16, 16, True, [4097, 1, 2048]),
    (F16, 128, 130, 2, 24, 3, False, [333, 0, 90]),
    (BF16, 64, 5, 5, 5, 1, True, [0]),
    (BF16, 128, 3, 3, 48, 16, True, [0, 0, 0, 1]),
    (F16, 64, 2, 1, 16, 2, True, [9001]),
    (BF16, 128, 1, 1, 100, 50, False, [20000, 3, 12001]),
    (F16, 128, 64, 2, 32, 32, True, [3000, 63, 64, 65]),
    (BF16, 128, 16, 2, 16, 16, True, [1100, 2, 64, 130]),
    (F16, 64, 24, 3, 16, 1, False, [513, 200, 0]),
    (BF16, 64, 16, 4, 64, 32, False, [4000, 33]),
    (F16, 128, 8, 8, 16, 16, True, [1000 - 30 * i for i in range(32)]),      # a workgroup to each
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_against_64_bits(dnn, case):
    dtype, d, H, heads, page, block, tokmajor, lengths = CASES[case]
    gen = torch.Generator().manual_seed(500 + case)
    c = QuantCache(gen, lengths, heads, page, block, d, tokmajor, quick=True)
    say(f"paged attention i8 {CASES[case]}")
    check(dnn, c, query(gen, len(lengths), H, d, dtype, 2.0), d ** -0.5)


@pytest.mark.parametrize("b", [65, 300, 1100])
def test_many_ragged_sequences(dnn, b):
    gen = torch.Generator().manual_seed(b)
    lengths = [0 if x % 3 == 0 else x % 211 for x in torch.randint(0, 10000, (b,), generator=gen).tolist()]
    c = QuantCache(gen, lengths, 2, 16, 4, 64, True, quick=True)
    say(f"paged attention i8, {b} ragged sequences")
    state = c.state()
    c.state = lambda: state                     # (rows() reads it once per sequence)
    check(dnn, c, query(gen, b, 4, 64, BF16), 0.125)


def test_room_far_beyond_the_lengths(dnn):
    gen = torch.Generator().manual_seed(5)
    c = QuantCache(gen, [40, 3, 0], 2, 16, 16, 128, True, room=6000, quick=True)
    c.table[:, 3:] = -1
    check(dnn, c, query(gen, 3, 4, 128, F16), 128 ** -0.5)


def test_pages_that_do_not_exist_and_lengths_outside_the_table(dnn):
    gen = torch.Generator().manual_seed(7)
    c = QuantCache(gen, [100, 300, 32, 40, 40], 2, 16, 8, 64, False, quick=True)
    c.table[0, 2], c.table[1, 0], c.table[1, 18], c.table[2, :] = -1, c.k.shape[0], 2 ** 31 - 1, -3
    c.lengths = ints([100, 300, 32, -5, 40])
    c.n[3] = 0
    check(dnn, c, query(gen, 5, 4, 64, F16), 0.125)
    c = QuantCache(gen, [64, 64], 2, 16, 8, 64, True, quick=True)
    c.lengths = ints([10 ** 9, 64])
    check(dnn, c, query(gen, 2, 2, 64, BF16), 0.125)


def test_shared_pages_strides_and_in_place(dnn):
    """A table row that all sequences share, pools and scales with pitches, q and o as rows of a
    packed projection, o over q."""
    gen = torch.Generator().manual_seed(9)
    c = QuantCache(gen, [500, 0], 4, 16, 4, 64, False, quick=True)
    k = torch.full((c.k.shape[0], 5, 18, 80), 99, dtype=torch.int8, device="cuda")
    v = torch.full((c.k.shape[0], 4, 17, 96), 99, dtype=torch.int8, device="cuda")
    s = torch.full((2, c.k.shape[0], 4, 7), math.nan, device="cuda")
    views = (k[:, 1:, 1:17, 16:], v[:, :, :16, :64], s[0, :, :, 1:5], s[1, :, :, 1:5])
    for to, x in zip(views, (c.k, c.v, c.ks, c.vs)):
        to.copy_(x)
    c.k, c.v, c.ks, c.vs = views
    c.table = c.table[:1].expand(2, -1)
    c.n, c.lengths = [500, 150], ints([500, 150])
    packed = torch.randn((2, 1, 24, 64), generator=gen).to(F16).cuda()
    rest = packed[:, :, 8:].clone()
    q = packed[:, :, :8].transpose(1, 2)
    apart = check(dnn, c, q, 0.125)
    over = check(dnn, c, q, 0.125, inplace=True)
    assert torch.equal(apart, over) and torch.equal(packed[:, :, 8:], rest)


def test_scales_of_every_size(dnn):
    """Values' scales that grow and shrink by powers of ten along a sequence, zeros among them,
    and keys' scales that make scores of every size."""
    gen = torch.Generator().manual_seed(10)
    for dtype, kind in ((BF16, "up"), (F16, "down"), (BF16, "zeros")):
        c = QuantCache(gen, [900, 333], 2, 16, 16, 128, True, quick=True)
        for i, n in enumerate(c.n):
            pages = c.table[i, : -(-n // 16)].long()
            ramp = torch.linspace(-9, 2, len(pages), device="cuda")
            if kind == "zeros":
                c.vs[pages[::2]] = 0.0
                c.ks[pages[1::3]] = 0.0
            else:
                c.vs[pages] = (10.0 ** (ramp if kind == "up" else ramp.flip(0)))[:, None, None].expand(-1, 2, 1)
                c.ks[pages] = (10.0 ** (ramp.flip(0) / 3 - 2))[:, None, None].expand(-1, 2, 1)
        say(f"paged attention i8, scales {kind}")
        check(dnn, c, query(gen, 2, 8, 128, dtype), 128 ** -0.5)


def test_large_scores(dnn):
    """A slot that outweighs the others by far, wherever it lies, and scores of +-1000."""
    gen = torch.Generator().manual_seed(11)
    c = QuantCache(gen, [700, 64, 1], 1, 16, 1, 64, False, quick=True)
    c.ks.mul_(20.0)
    check(dnn, c, query(gen, 3, 4, 64, F16, 4.0), 1.0)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_queries_of_every_size(dnn, dtype):
    """Rows of zeros, of one value, of values from the type's least to its largest; NaN and
    infinities make their rows NaN and no other."""
    gen = torch.Generator().manual_seed(12)
    c = QuantCache(gen, [150], 1, 16, 8, 128, True, quick=True)
    top = torch.finfo(dtype).max
    q = query(gen, 1, 8, 128, dtype)
    q[0, 0] = 0.0
    q[0, 1] = 0.0
    q[0, 1, 0, 77] = 1.0
    q[0, 2] *= 2.0 ** -12
    q[0, 3, 0, 5] = 100.0
    scale = 0.01
    q[0, 4, 0, 3], q[0, 5, 0, 9], q[0, 6, 0, 127] = math.nan, math.inf, -math.inf
    o = torch.full_like(q, 7.0)
    attend(dnn, c, q, o, scale)
    K, V, _ = c.rows(0)
    for h in range(8):
        if h in (4, 5, 6):
            assert torch.isnan(o[0, h]).all()
            continue
        ref, bound = attention_ref(q[0, h].cpu(), K, V, scale)
        assert ((o[0, h].cpu().double() - ref).abs() <= bound).all(), h
    q[0, :] = 0.0
    q[0, 1], q[0, 2] = torch.finfo(dtype).tiny, top / 1024
    c.ks.fill_(2.0 ** -20 if dtype == F16 else 2.0 ** -125)
    check(dnn, c, q, scale)


def test_nan_scales(dnn):
    """A block of NaN makes its head of its sequence NaN and no other; one behind the end does
    not, nor one on a page that does not exist."""
    gen = torch.Generator().manual_seed(13)
    for which in ("ks", "vs"):
        c = QuantCache(gen, [100, 90, 33], 2, 16, 4, 64, True, quick=True)
        getattr(c, which)[int(c.table[0, 3]), 1, 2] = math.nan
        getattr(c, which)[int(c.table[2, 2]), :, 1:] = math.nan         # from slot 36 on
        o = torch.empty((3, 6, 1, 64), dtype=F16, device="cuda")
        attend(dnn, c, query(gen, 3, 6, 64, F16), o, 0.125)
        nan = torch.isnan(o[:, :, 0]).cpu()
        assert nan[0, 3:].all() and not nan[0, :3].any() and not nan[1:].any()


def test_the_same_bits_every_time(dnn):
    """Whatever the workspace held, and next to other sequences or alone."""
    gen = torch.Generator().manual_seed(14)
    c = QuantCache(gen, [3000, 10, 700], 2, 16, 16, 128, True, quick=True)
    q = query(gen, 3, 8, 128, BF16)
    first = torch.empty_like(q)
    attend(dnn, c, q, first, 0.1)
    for _ in range(3):
        o = torch.full_like(q, math.nan)
        attend(dnn, c, q, o, 0.1)
        assert torch.equal(o, first)


def test_two_streams_and_two_calls_at_once(gpu):
    gen = torch.Generator().manual_seed(15)
    handles, sides = [g.Dnn(), g.Dnn()], [torch.cuda.Stream(), torch.cuda.Stream()]
    caches = [QuantCache(gen, [2000, 5, 900], 4, 16, 16, 64, True, quick=True) for _ in range(2)]
    qs = [query(gen, 3, 16, 64, F16) for _ in range(2)]
    want = []
    for dnn, c, q in zip(handles, caches, qs):
        want.append(check(dnn, c, q, 0.125).clone())
    outs, keep = [torch.full_like(q, math.nan) for q in qs], []
    torch.cuda.synchronize()
    for dnn, side, c, q, o in zip(handles, sides, caches, qs, outs):
        dnn.set_stream(side.cuda_stream)
        args = c.args()
        qd = desc(q)
        ws = Workspace(dnn.paged_attention_quantized_workspace(qd, args[0], args[7]))
        keep.append((args, qd, ws))
    torch.cuda.synchronize()
    ad = g.AttnDesc(False, 0.125)
    for _ in range(10):
        for dnn, (args, qd, ws), q, o in zip(handles, keep, qs, outs):
            g.check(dnn.paged_attention_quantized(ad, qd, q.data_ptr(), *args, qd, o.data_ptr(), ws.p, ws.size))
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)
    for dnn in handles:
        dnn.close()


def test_captured_steps(gpu):
    """Append, the new lengths and attention in one graph: replays generate what eager calls do."""
    dnn = g.Dnn()
    caches = []
    for _ in range(2):
        gen = torch.Generator().manual_seed(16)
        caches.append(QuantCache(gen, [30, 0, 17], 2, 16, 16, 64, True, room=120))
    gen = torch.Generator().manual_seed(17)
    k, v, q = (torch.randn((3, h, 1, 64), generator=gen).to(BF16).cuda() for h in (2, 2, 8))
    kd, qd = desc(k), desc(q)
    outs = [torch.zeros_like(q) for _ in range(2)]
    args = [c.args() for c in caches]
    ws = Workspace(dnn.paged_attention_quantized_workspace(qd, args[0][0], args[0][7]))
    ad = g.AttnDesc(True, 0.125)

    def calls(i):
        g.check(dnn.paged_append_quantized(kd, k.data_ptr(), kd, v.data_ptr(), *args[i]))
        caches[i].lengths.add_(1)
        g.check(dnn.paged_attention_quantized(ad, qd, q.data_ptr(), *args[i], qd, outs[i].data_ptr(), ws.p, ws.size))

    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    say("capturing append8 and attention")
    with torch.cuda.graph(graph, stream=side):
        dnn.set_stream(torch.cuda.current_stream().cuda_stream)
        calls(1)
    dnn.set_stream(None)
    for step in range(20):
        k.mul_(1.05)
        v.roll(1, 3)
        calls(0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(*outs), f"replay {step}"
    caches[1].check(caches[0].state())
    del graph
    dnn.close()


def test_against_the_cache_of_16_bits(dnn):
    """Rows that 8 bits hold exactly (codes times a scale that is a power of two): the same
    attention as over a cache of 16 bits, within both bounds."""
    import paged_cases
    gen = torch.Generator().manual_seed(18)
    n, heads, d = [400, 65], 2, 128
    c = QuantCache(gen, n, heads, 16, 16, d, True, quick=True)
    c.ks.fill_(2.0 ** -5)
    c.vs.fill_(2.0 ** -6)
    q = query(gen, 2, 8, d, BF16)
    o = check(dnn, c, q, d ** -0.5)
    full = paged_cases.Cache(gen, BF16, n, heads, 16, d, True)
    for i in range(2):
        K, V, _ = c.rows(i)
        full.K[i], full.V[i] = K.to(BF16), V.to(BF16)
        assert torch.equal(full.K[i].double(), K)
    full.store()
    other = torch.empty_like(o)
    paged_cases.attend(dnn, full, q, other, d ** -0.5)
    for i in range(2):
        K, V, _ = c.rows(i)
        _, bound = attention_ref(q[i, :, 0].cpu(), K, V, d ** -0.5)
        _, _, theirs, _ = paged_cases.attention_ref(q[i, :, 0].cpu(), full.K[i], full.V[i], d ** -0.5)
        assert ((o[i, :, 0] - other[i, :, 0]).cpu().double().abs() <= bound + theirs).all()


def test_appended_rows_are_attended(dnn):
    gen = torch.Generator().manual_seed(19)
    c = QuantCache(gen, [0, 0], 2, 16, 8, 64, True, room=200)
    k, v = (torch.randn((2, 2, 190, 64), generator=gen).to(F16).cuda() for _ in range(2))
    append(dnn, c, k, v, ints([190, 77]))
    c.n, c.lengths = [190, 77], ints([190, 77])
    check(dnn, c, query(gen, 2, 4, 64, F16), 0.125)


def weighed_ref(q, K, V, vs, scale):
    """attention_ref with the weights held to what they are said to keep: a weight times its slot's
    scale of a value, 21 bits, or half of fp16's least, 2^-25, where the largest such product of
    the query has 2^11 or more: 2^-36 of that. vs [heads, n]: the slots' scales of values."""
    H, d = q.shape
    group = H // K.shape[0]
    k, v, vs = (x.repeat_interleave(group, 0) for x in (K, V, vs.double()))
    q64 = q.double()
    p = torch.softmax(torch.matmul(k, q64[:, :, None])[..., 0] * scale, 1)
    o = torch.matmul(p[:, None], v)[:, 0]
    size = torch.matmul(k.abs(), q64.abs()[:, :, None])[..., 0]
    off = 2.0 ** -22 * q64.abs().amax(1, keepdim=True) * k.abs().sum(2)
    delta = (off + 8 * 2.0 ** -24 * size).amax(1, keepdim=True) * scale
    rel = 2 * delta + 2.0 ** -18 + 2.0 ** -21
    u = {BF16: 2.0 ** -8, F16: 2.0 ** -11}[q.dtype]
    mass = torch.matmul(p[:, None], v.abs())[:, 0]
    floor = k.shape[1] * 2.0 ** -36 * 127 * (p * vs).amax(1, keepdim=True)
    return o, u * o.abs() + (1 + u) * (rel * mass + floor) + {BF16: 2.0 ** -134, F16: 2.0 ** -25}[q.dtype]


def check_weighed(dnn, gen, dtype, d, H, heads, n, special, log_scale, ratios, block, what):
    """The slots of `special` (multiples of block) have scores 26 below the others' (weights of
    about 2^-37) and values 2^ratio times as large; a sequence to each ratio."""
    b = len(ratios)
    c = QuantCache(gen, [n] * b, heads, block, block, d, True, quick=True)
    q = query(gen, b, H, d, dtype, 0.25)
    q[..., 0] = 4.0
    scales = torch.full((b, heads, n), 2.0 ** log_scale)
    for i, ratio in enumerate(ratios):
        at = torch.arange(n, device="cuda")
        page, row = c.table[i, at // block].long(), at % block
        c.ks[page] = 1.0 / 39
        c.vs[page] = 2.0 ** log_scale
        c.k[page, :, row, 0] = 127
        odd = at[special[0]:special[1]]
        c.k[c.table[i, odd // block].long(), :, odd % block, 0] = -127
        c.vs[c.table[i, odd // block].long()] = 2.0 ** (log_scale + ratio)
        scales[i, :, special[0]:special[1]] = 2.0 ** (log_scale + ratio)
    o = torch.full_like(q, math.nan)
    say(what)
    attend(dnn, c, q, o, 1.0)
    for i, ratio in enumerate(ratios):
        K, V, _ = c.rows(i)
        ref, bound = weighed_ref(q[i, :, 0].cpu(), K, V, scales[i], 1.0)
        assert (bound < 0.02 * ref.abs().amax(1, keepdim=True)).all(), "a bound that holds nothing"
        off = (o[i, :, 0].cpu().double() - ref).abs() - bound
        assert not (off > 0).any(), f"{what}, 2^{ratio}: {off.max().item():.3g} past the bound"


@pytest.mark.parametrize("H,heads,n", [(4, 1, 320), (8, 1, 320), (16, 1, 320), (33, 1, 320), (4, 1, 1600), (16, 2, 1600),
                                       (13, 1, 1600), (64, 2, 1600)])
@pytest.mark.parametrize("special", [(0, 16), (144, 160), (304, 320)])
def test_values_of_little_weight_and_large_scale(dnn, H, heads, n, special):
    """Whatever a slot's scale, o is made of what its slots weigh: from nothing to all of it."""
    gen = torch.Generator().manual_seed(20)
    for dtype, log_scale, ratios in ((BF16, -8, (10, 20, 25, 30, 34, 37, 40, 50, 70)), (F16, -6, (15, 25, 30, 34, 37, 40)),
                                     (BF16, -100, (-20, 30, 60))):
        check_weighed(dnn, gen, dtype, 128 if n > 1000 else 64, H, heads, n, special, log_scale, ratios, 16,
                      f"values of little weight {dtype} {H} on {heads} heads, {n} slots, {special}, 2^{log_scale}")


@pytest.mark.parametrize("dtype,b,H,heads,d,room,tokmajor,kernel", [
    (BF16, 3, 8, 2, 64, 256, True, "whole1"),          # groups of 4, and so on
    (F16, 20, 39, 3, 128, 500, False, "whole1"),       # 13
    (BF16, 5, 42, 2, 128, 500, True, "whole1"),        # 21
    (F16, 3, 70, 2, 64, 500, True, "whole1"),          # 35
    (BF16, 3, 8, 2, 128, 1040, True, "split1"),        # 4
    (F16, 20, 28, 4, 128, 1040, False, "split1"),      # 7
    (BF16, 20, 36, 4, 64, 1040, False, "split1"),      # 9
    (F16, 3, 32, 2, 128, 1200, True, "split1"),        # 16
    (BF16, 2, 66, 2, 128, 1040, True, "split1"),       # 33
    (F16, 40, 6, 6, 128, 1040, True, "split2"),        # 1
    (BF16, 40, 30, 6, 64, 1040, True, "split2"),       # 5
    (F16, 40, 72, 6, 128, 1040, True, "split2"),       # 12
    (BF16, 40, 80, 2, 64, 1040, True, "split2"),       # 40
    (BF16, 64, 16, 4, 128, 1040, True, "split4"),      # 4
    (F16, 64, 32, 4, 64, 1040, True, "split4"),        # 8
    (BF16, 64, 52, 4, 128, 1040, True, "split4"),      # 13
    (F16, 64, 80, 4, 128, 1040, True, "split4"),       # 20
    (F16, 40, 132, 4, 64, 1040, True, "split4"),       # 33
])
def test_every_kernel_choice(dnn, capfd, monkeypatch, dtype, b, H, heads, d, room, tokmajor, kernel):
    """The choice that GRXDNN_LOG names, on ragged lengths from none to the room's."""
    gen = torch.Generator().manual_seed(21)
    lengths = [0, 1, room] + torch.randint(0, room + 1, (max(0, b - 3),), generator=gen).tolist()
    c = QuantCache(gen, lengths[:b], heads, 20 if room % 20 == 0 else 16, 4, d, tokmajor, room=room, quick=True)
    state = c.state()
    c.state = lambda: state
    capfd.readouterr()
    monkeypatch.setenv("GRXDNN_LOG", "1")
    check(dnn, c, query(gen, b, H, d, dtype, 2.0), d ** -0.5)
    monkeypatch.delenv("GRXDNN_LOG")
    log = [x for x in capfd.readouterr().err.splitlines() if x.startswith("grxdnn: paged attention i8 ")]
    assert len(log) == 1 and log[0].endswith(f"kernel={kernel}"), log


def test_the_same_bits_whatever_the_workspace_held(dnn):
    """And, within the bound, the same next to other sequences as alone (where the work is
    shared otherwise)."""
    gen = torch.Generator().manual_seed(22)
    c = QuantCache(gen, [3000, 10, 700], 2, 16, 16, 128, True, quick=True)
    q = query(gen, 3, 8, 128, BF16)
    args, qd, ad = c.args(), desc(q), g.AttnDesc(True, 0.1)
    runs = []
    for fill in (0, 0xFF, 0x7F):
        o = torch.full_like(q, math.nan)
        ws = Workspace(dnn.paged_attention_quantized_workspace(qd, args[0], args[7]))
        ws.t.fill_(fill)
        torch.cuda.synchronize()
        g.check(dnn.paged_attention_quantized(ad, qd, q.data_ptr(), *args, qd, o.data_ptr(), ws.p, ws.size))
        torch.cuda.synchronize()
        runs.append(o)
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])
    table, n = c.table, c.n
    for i in range(3):
        c.table, c.lengths, c.n = table[i:i + 1], ints(n[i:i + 1]), n[i:i + 1]
        alone = check(dnn, c, q[i:i + 1].clone(), 0.1)
        K, V, _ = c.rows(0)
        ref, bound = attention_ref(q[i, :, 0].cpu(), K, V, 0.1)
        assert ((runs[0][i, :, 0].cpu().double() - ref).abs() <= bound).all(), i
        assert ((runs[0][i, :, 0] - alone[0, :, 0]).cpu().double().abs() <= 2 * bound).all(), i


def test_captured_steps_with_new_rows(gpu):
    """As test_captured_steps, with other keys, values and queries at every replay."""
    dnn = g.Dnn()
    caches = []
    for _ in range(2):
        gen = torch.Generator().manual_seed(23)
        caches.append(QuantCache(gen, [30, 0, 700], 2, 16, 16, 128, True, room=1100))
    gen = torch.Generator().manual_seed(24)
    k, v, q = (torch.empty((3, h, 1, 128), dtype=F16, device="cuda") for h in (2, 2, 8))
    kd, qd = desc(k), desc(q)
    outs = [torch.zeros_like(q) for _ in range(2)]
    args = [c.args() for c in caches]
    ws = Workspace(dnn.paged_attention_quantized_workspace(qd, args[0][0], args[0][7]))
    ad = g.AttnDesc(True, 128 ** -0.5)

    def calls(i):
        g.check(dnn.paged_append_quantized(kd, k.data_ptr(), kd, v.data_ptr(), *args[i]))
        caches[i].lengths.add_(1)
        g.check(dnn.paged_attention_quantized(ad, qd, q.data_ptr(), *args[i], qd, outs[i].data_ptr(), ws.p, ws.size))

    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    say("capturing append8 and attention, new rows")
    with torch.cuda.graph(graph, stream=side):
        dnn.set_stream(torch.cuda.current_stream().cuda_stream)
        calls(1)
    dnn.set_stream(None)
    seen = []
    for step in range(20):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=gen).mul(1.0 + 0.2 * step))
        calls(0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(*outs), f"replay {step}"
        seen.append(outs[0].clone())
        assert all(not torch.equal(outs[0], x) for x in seen[:-1])
    caches[1].check(caches[0].state())
    c = caches[0]
    c.n = [n + 20 for n in c.n]
    for i in range(3):
        K, V, _ = c.rows(i)
        ref, bound = attention_ref(q[i, :, 0].cpu(), K, V, 128 ** -0.5)
        assert ((outs[1][i, :, 0].cpu().double() - ref).abs() <= bound).all(), i
    del graph
    dnn.close()
