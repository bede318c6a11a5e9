"""grxdnnPagedCacheAppendQuantized and grxdnnPagedCacheReadQuantized against 64 bits: every
code, every scale and every byte around them."""
import math

import pytest
import torch

import grxcp_amd as g
from helpers import say
from paged_cases import ints
from quant_cases import QuantCache, append, desc, least8, over, read

pytestmark = pytest.mark.gpu
BF16, F16, FP32 = torch.bfloat16, torch.float16, torch.float32


def rows(gen, b, heads, T, d, dtype, spread=0.0):
    """New rows [b, heads, T, d]; spread: the standard deviation of their size's logarithm."""
    x = torch.randn((2, b, heads, T, d), generator=gen)
    if spread:
        x *= (spread * torch.randn((2, b, heads, T, 1), generator=gen)).exp()
    return (t.to(dtype).cuda() for t in x)


def check_append(dnn, c, k, v, counts=None):
    want = c.append_ref(k, v, [k.shape[2]] * len(c.n) if counts is None else counts)
    say(f"append8 {tuple(k.shape)} {k.dtype} blocks of {c.block}/{c.page} to {c.n[:8]}")
    append(dnn, c, k, v, None if counts is None else ints(counts))
    c.check(want)


# ---- append ------------------------------------------------------------------

APPENDS = [
    # dtype, d, heads, page, block, tokmajor, lengths before, T, counts
    (BF16, 128, 8, 16, 16, True, [0, 15, 16, 17, 5], 1, None),
    (F16, 64, 1, 1, 1, False, [3, 0], 5, [5, 2]),
    (BF16, 64, 3, 7, 7, True, [6, 7, 8, 0, 20], 23, [0, 23, -4, 100, 1]),
    (F16, 128, 2, 64, 32, False, [63, 100], 300, None),
    (BF16, 64, 5, 256, 256, True, [0, 250], 700, [699, 8]),
    (F16, 128, 2, 256, 256, False, [40, 255], 300, None),
    (BF16, 128, 3, 256, 128, True, [200], 77, None),
    (F16, 64, 2, 16, 4, False, [40, 1, 2], 70, [0, 0, 1]),
    (BF16, 128, 2, 48, 3, True, [1, 47, 50], 9, None),
    (F16, 64, 4, 100, 50, False, [49, 50], 2, None),
    (BF16, 64, 2, 128, 128, False, [100], 40, None),
    (F16, 128, 4, 32, 1, True, [5, 31, 64], 90, [90, 0, 33]),
    (BF16, 128, 1, 8, 2, False, [1, 2, 3], 3, None),
    (BF16, 64, 1, 64, 64, True, [10, 63], 65, None),
]


@pytest.mark.parametrize("spread", [0.0, 1.5])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(dnn, case, spread):
    dtype, d, heads, page, block, tokmajor, lengths, T, counts = APPENDS[case]
    gen = torch.Generator().manual_seed(case)
    c = QuantCache(gen, lengths, heads, page, block, d, tokmajor, room=max(lengths) + T, dtype=dtype)
    check_append(dnn, c, *rows(gen, len(lengths), heads, T, d, dtype, spread), counts)


@pytest.mark.parametrize("stream", [False, True])
@pytest.mark.parametrize("d, page, block", [(64, 16, 1), (128, 7, 1), (64, 6, 2), (128, 9, 3), (64, 14, 7), (128, 5, 5),
                                            (64, 24, 12), (128, 16, 16), (128, 40, 20)])
def test_append_of_many_rows(dnn, d, page, block, stream):
    """As many blocks as give a thread more than one chunk, or task, at a time; blocks that hold
    rows before, odd ones, pages that do not exist, and sequences that take fewer."""
    T = 32 * 2 ** 20 // (2 * 40 * d * 2) + 19 if stream else 1300
    gen = torch.Generator().manual_seed(17 * d + block)
    c = QuantCache(gen, [3 * block + block // 2, block - 1], 40, page, block, d, block % 2 == 0, room=4 * block + T)
    c.table[0, 5], c.table[1, 2] = -1, c.k.shape[0]
    check_append(dnn, c, *rows(gen, 2, 40, T, d, (BF16, F16)[block % 2], 1.0), [T, T - 3 * block - 1])


def test_tokens_one_at_a_time(dnn):
    """Blocks that fill row by row, their scales growing as they do; every step against 64 bits
    from the step before."""
    gen = torch.Generator().manual_seed(40)
    c = QuantCache(gen, [0, 7, 13], 2, 16, 8, 64, True, room=60)
    for _ in range(20):
        check_append(dnn, c, *rows(gen, 3, 2, 1, 64, F16, 1.0))
        c.n = [n + 1 for n in c.n]
        c.lengths += 1


def test_ties_go_to_the_even_code(dnn):
    """Rows of (k + 1/2) * scale for every k that has one, with scales of few bits."""
    gen = torch.Generator().manual_seed(41)
    c = QuantCache(gen, [0] * 6, 2, 4, 1, 128, room=4)
    x = torch.zeros(6, 2, 1, 128)
    for i, s in enumerate((1.0, 2.0 ** -9, 0.5, 4.0, 2.0 ** -14, 1.5)):
        x[i] = (torch.arange(128) - 64 + 0.5) * s
        x[i, :, :, 0] = 127 * s                      # the largest one: the scale is s
    x = x.to(F16)
    assert (x[5, 0, 0, 1] == -62.5 * 1.5)
    want = over(x.double(), torch.tensor([1.0, 2.0 ** -9, 0.5, 4.0, 2.0 ** -14, 1.5]).double()[:, None, None, None])
    check_append(dnn, c, x.cuda(), x.cuda())
    for i in range(6):
        assert torch.equal(c.k[int(c.table[i, 0]), :, 0].cpu(), want[i, :, 0])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_ties_of_every_scale(dnn, dtype):
    """Scales of every odd significand of 8 bits: all halves of codes that the type holds, and their
    neighbours; then a row that doubles the scale, so that the odd codes before lie half way."""
    odd = torch.arange(1, 256, 2, dtype=torch.float64)
    c = QuantCache(torch.Generator().manual_seed(44), [0] * len(odd), 2, 2, 2, 128, room=2)
    for power, step in ((-9, 1), (-9, 2)):
        s = (odd * 2.0 ** power * step)[:, None, None, None]
        k = torch.stack([torch.arange(128.0) - 64, torch.arange(128.0)])[None, :, None].double()
        x = ((k + 0.5) * s).to(dtype)
        most = (127 * s).to(dtype)
        bits = most.view(torch.int16)
        most = torch.where(most.double() > 127 * s, (bits - 1).view(dtype), most)     # not above 127 scales
        x[..., :1] = most
        x = torch.minimum(x, most)
        scale = least8(most.double() / 127)
        assert torch.equal(scale, s)
        assert ((x.double() / scale % 1).abs() == 0.5).sum() > 1000      # ties
        check_append(dnn, c, x.cuda(), -x.cuda())
        c.n = [n + 1 for n in c.n]
        c.lengths += 1


@pytest.mark.parametrize("dtype, d, block, heads, T", [
    (BF16, 64, 1, 2, 5), (F16, 128, 2, 2, 7), (BF16, 128, 16, 2, 35), (F16, 64, 32, 2, 67), (F16, 128, 64, 2, 131),
    (BF16, 64, 7, 2, 17), (F16, 64, 2, 40, 150)])     # the last: two tasks to a thread
def test_scales_that_the_caller_set(dnn, dtype, d, block, heads, T):
    """Blocks with scales of 24 bits: larger than the new rows need, smaller (the rows before are
    rounded again), and quotients so close to a half that fp32 would miss it."""
    gen = torch.Generator().manual_seed(45)
    n = 3 * block + block // 2
    c = QuantCache(gen, [n] * 12, heads, 2 * block, block, d, block == 16, room=n + T, dtype=dtype, quick=True)
    k, v = rows(gen, 12, heads, T, d, dtype, 1.0)
    new = block - block // 2                 # rows that the block of each head still takes
    page, at = c.table[:, 3 * block // c.page].long(), 3 * block % c.page // block
    for t, scale in ((k, c.ks), (v, c.vs)):
        nudge = torch.randint(-9, 9, (12, heads, 1, 1), generator=gen).cuda()
        by = scale[page, :, at][:, :, None, None] * (1 + 2.0 ** -20 * nudge)
        scale[page, :, at] = by[:, :, 0, 0]
        half = (torch.arange(new * d, device="cuda").reshape(new, d) % 100 + 0.5) * by
        t[:6, :, :new] = half[:6].to(dtype)
    check_append(dnn, c, k, v)


def test_every_value_of_the_types(dnn):
    """All finite bf16 and fp16 values as rows of blocks whose largest magnitude is of every
    size: the codes and scales of 64 bits."""
    for dtype, count in ((BF16, 0x7f80), (F16, 0x7c00)):
        x = torch.arange(count, dtype=torch.int32).to(torch.int16).view(dtype)
        gen = torch.Generator().manual_seed(42)
        x = x[: count // 128 * 128].reshape(1, 1, -1, 128)
        x = x * (1 - 2 * torch.randint(0, 2, x.shape, generator=gen)).to(dtype)
        # ordered rows (all of one size), and mixed ones
        mixed = x.reshape(-1)[torch.randperm(x.numel(), generator=gen)].reshape(x.shape)
        c = QuantCache(gen, [0], 1, 64, 4, 128, room=x.shape[2])
        check_append(dnn, c, x.cuda(), mixed.cuda())


def test_specials(dnn):
    """Blocks of zeros, of infinities and NaN, before and after others; the others are as they
    would be without."""
    gen = torch.Generator().manual_seed(43)
    c = QuantCache(gen, [2, 2, 2, 2, 2, 0], 1, 8, 4, 64, room=16)
    k, v = rows(gen, 6, 1, 6, 64, BF16)
    k[0, :, 0, 3] = math.inf                    # into a block that holds rows
    k[1, :, 3, 7] = math.nan                    # the next block alone
    v[2, :, 1, 0] = -math.inf
    k[3] = 0.0
    v[5, :, :4] = 0.0
    c.ks[int(c.table[4, 0]), 0, 0] = math.nan   # a block that was NaN before stays so
    check_append(dnn, c, k, v)
    assert torch.isnan(c.ks[int(c.table[0, 0]), 0, 0]) and torch.isfinite(c.ks[int(c.table[0, 0]), 0, 1])
    assert torch.isfinite(c.ks[int(c.table[1, 0]), 0, 0]) and torch.isnan(c.ks[int(c.table[1, 0]), 0, 1])
    assert torch.isnan(c.ks[int(c.table[4, 0]), 0, 0])
    assert c.vs[int(c.table[5, 0]), 0, 0] == 0
    # a page that held NaN is taken by another sequence: its scales are not looked at
    c.n[0], c.lengths[0] = 0, 0
    k, v = rows(gen, 6, 1, 5, 64, BF16)
    check_append(dnn, c, k, v, [5, 0, 0, 0, 0, 0])
    assert torch.isfinite(c.ks[int(c.table[0, 0]), 0]).all()


def test_pages_that_do_not_exist_and_full_tables(dnn):
    gen = torch.Generator().manual_seed(44)
    c = QuantCache(gen, [10, 0, 30], 2, 8, 4, 64, True, room=40)
    c.table[0, 2], c.table[1, 0], c.table[1, 3] = -1, c.k.shape[0], 2 ** 31 - 1
    k, v = rows(gen, 3, 2, 50, 64, F16)
    check_append(dnn, c, k, v)
    # lengths outside the table
    c.lengths = ints([10 ** 9, -7, 40])
    c.n = [10 ** 9, -7, 40]
    check_append(dnn, c, *rows(gen, 3, 2, 9, 64, F16))


def test_strides(dnn):
    """Rows as views of a packed projection, pools and scales with pitches."""
    gen = torch.Generator().manual_seed(45)
    c = QuantCache(gen, [5, 20], 3, 16, 8, 64, room=64)
    k = torch.full((c.k.shape[0], 4, 17, 80), 77, dtype=torch.int8, device="cuda")
    v = torch.full((c.k.shape[0], 3, 18, 96), 77, dtype=torch.int8, device="cuda")
    s = torch.full((2, c.k.shape[0], 3, 5), math.nan, device="cuda")
    views = (k[:, 1:, 1:, 16:], v[:, :, :16, :64], s[0, :, :, 1:3], s[1, :, :, 1:3])
    for to, x in zip(views, (c.k, c.v, c.ks, c.vs)):
        to.copy_(x)
    c.k, c.v, c.ks, c.vs = views
    packed = torch.randn((2, 30, 9, 64), generator=gen).to(BF16).cuda()
    check_append(dnn, c, packed[:, :, 3:6].transpose(1, 2), packed[:, :, 6:].transpose(1, 2))
    assert (k[:, 0] == 77).all() and (k[..., :16] == 77).all() and (k[:, :, 0] == 77).all()
    assert (v[..., 64:] == 77).all() and (v[:, :, 16:] == 77).all() and torch.isnan(s[..., [0, 3, 4]]).all()


@pytest.mark.parametrize("b", [70, 70000])
def test_many_sequences(dnn, b):
    """More sequences than a launch has workgroups along y; a few distinct pages, so that most
    have entries that name none."""
    gen = torch.Generator().manual_seed(b)
    c = QuantCache(gen, [0] * 5, 1, 4, 2, 64, room=4)
    table = torch.full((b, 1), -1, dtype=torch.int32)
    own = torch.randperm(b, generator=gen)[:5]
    table[own, 0] = c.table[:, 0].cpu()
    c.table, c.n = table.cuda(), [0] * b
    c.lengths = ints(c.n)
    k, v = rows(gen, b, 1, 2, 64, BF16)
    check_append(dnn, c, k, v)


def test_the_same_bits_every_time(dnn):
    gen = torch.Generator().manual_seed(46)
    c = QuantCache(gen, [100, 3, 64], 4, 32, 32, 128, True, room=200)
    before = c.state()
    k, v = rows(gen, 3, 4, 70, 128, BF16, 1.0)
    append(dnn, c, k, v)
    want = c.state()
    append(dnn, c, k, v)             # again, over its own rows: the scales are there already
    c.check(want)
    c.store(*before)
    append(dnn, c, k, v)
    c.check(want)


# ---- read --------------------------------------------------------------------

READS = [
    # dtype, d, heads, page, block, tokmajor, lengths, T, first
    (BF16, 128, 8, 16, 16, True, [0, 1, 16, 200], 200, None),
    (F16, 64, 3, 7, 7, False, [5, 30], 41, [0, 3]),
    (FP32, 64, 2, 1, 1, True, [9, 2, 0], 7, [2, 0, 0]),
    (F16, 128, 1, 256, 64, False, [700], 333, [390]),
    (BF16, 64, 5, 64, 1, True, [100, 65], 100, None),
    (FP32, 128, 2, 32, 4, False, [33, 500], 1, [32, 499]),
]


def read_ref(c, dtype, T, first):
    out = []
    for i, n in enumerate(c.n):
        n = min(max(n, 0), c.width * c.page)
        f = max(0, first[i]) if first else 0
        k, v, there = c.rows(i, n)
        both = torch.zeros(2, c.heads, T, c.d, dtype=torch.float64)
        at = torch.arange(min(f, n), min(n, f + T))
        at = at[there[at]] if len(at) else at
        both[0, :, at - f], both[1, :, at - f] = k[:, at], v[:, at]
        out.append(both)
    x = torch.stack(out, 1)
    most = torch.finfo(dtype).max
    return torch.where(torch.isnan(x), x, x.clamp(-most, most)).to(dtype)


def check_read(dnn, c, dtype, T, first=None):
    b = len(c.n)
    k, v = (torch.full((b, c.heads, T, c.d), math.nan, dtype=dtype, device="cuda") for _ in range(2))
    say(f"read8 {dtype} {T} rows from {first} of {c.n[:8]}")
    read(dnn, c, k, v, None if first is None else ints(first))
    want = read_ref(c, dtype, T, first)
    for got, ref in ((k, want[0]), (v, want[1])):
        got = got.cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        # 8 and 7 bits multiplied, rounded once: the same as from 64 bits
        assert torch.equal(got.nan_to_num(), ref.nan_to_num())
    return k, v


@pytest.mark.parametrize("case", range(len(READS)))
def test_read(dnn, case):
    dtype, d, heads, page, block, tokmajor, lengths, T, first = READS[case]
    gen = torch.Generator().manual_seed(60 + case)
    c = QuantCache(gen, lengths, heads, page, block, d, tokmajor)
    check_read(dnn, c, dtype, T, first)


@pytest.mark.parametrize("dtype", [BF16, F16, FP32])
@pytest.mark.parametrize("d, page, block", [(64, 32, 32), (128, 21, 21)])
def test_large_reads(dnn, d, page, block, dtype):
    """Calls past the caches, from the middle of the sequences to behind their ends."""
    T = 32 * 2 ** 20 // (3 * 40 * d * 2) + 5
    c = QuantCache(torch.Generator().manual_seed(59), [T + 7, 300, T + 40], 40, page, block, d, d == 64)
    c.table[2, 3] = -1
    check_read(dnn, c, dtype, T, [11, 0, 40])


def test_read_outside_the_sequences(dnn):
    """First slots past the end and below 0, lengths outside the table, pages that do not exist."""
    gen = torch.Generator().manual_seed(70)
    c = QuantCache(gen, [40, 40, 40, 40], 2, 8, 8, 64, True)
    c.table[1, 2], c.table[1, 0] = c.k.shape[0], -1
    c.lengths = ints([40, 40, -3, 10 ** 9])
    c.n = [40, 40, -3, 10 ** 9]
    for first in ([2 ** 31 - 1, 0, 0, 39], [-2 ** 31, 15, 5, -1], [40, 24, 0, 41]):
        check_read(dnn, c, BF16, 50, first)


def test_read_values_past_the_range_and_nan(dnn):
    gen = torch.Generator().manual_seed(71)
    c = QuantCache(gen, [8], 1, 8, 2, 64)
    at = int(c.table[0, 0])
    c.ks[at, 0] = torch.tensor([600.0, math.nan, 3e36, 2.0 ** -130], device="cuda")
    c.vs[at, 0] = torch.tensor([0.0, 1.0, math.nan, 515.0], device="cuda")
    for dtype in (F16, BF16, FP32):
        check_read(dnn, c, dtype, 8)


def test_read_into_strided_rows(dnn):
    """Outputs as [b, T, heads, d] memory with pitches, NaN around them."""
    gen = torch.Generator().manual_seed(72)
    c = QuantCache(gen, [20, 9], 3, 4, 4, 64, True)
    big = torch.full((2, 2, 22, 4, 72), math.nan, dtype=F16, device="cuda")
    k, v = (x[:, 1:21, 1:, :64].transpose(1, 2) for x in big)
    read(dnn, c, k, v)
    want = read_ref(c, F16, 20, None)
    assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1])
    assert int(torch.isnan(big).sum()) == big.numel() - k.numel() - v.numel()


def test_written_and_read_back(dnn):
    """A row comes back within half a step of its block's scale: what 8 bits keep."""
    gen = torch.Generator().manual_seed(73)
    c = QuantCache(gen, [0, 0], 4, 16, 8, 128, True, room=100)
    k, v = rows(gen, 2, 4, 100, 128, BF16)
    check_append(dnn, c, k, v)
    c.n, c.lengths = [100, 100], ints([100, 100])
    for got, x in zip(check_read(dnn, c, FP32, 100), (k, v)):
        x = x.cpu().double()
        pad = torch.nn.functional.pad(x, (0, 0, 0, 4)).reshape(2, 4, 13, 8, 128)
        s = least8(pad.abs().amax((3, 4)) / 127).repeat_interleave(8, 2)[:, :, :100, None]
        assert ((got.cpu().double() - x).abs() <= s / 2).all()


def test_captured(gpu):
    """Append, the new lengths and a read in one graph: replays follow lengths, counts and
    tables of their time, as eager calls do."""
    dnn = g.Dnn()
    gen = torch.Generator().manual_seed(74)
    caches = []
    for _ in range(2):
        gen.manual_seed(74)
        caches.append(QuantCache(gen, [3, 0, 17], 2, 16, 8, 64, True, room=120))
    k, v = rows(gen, 3, 2, 7, 64, F16, 1.0)
    counts, first = ints([7, 3, 1]), ints([0, 0, 10])
    kd, vd = desc(k), desc(v)
    outs = [[torch.zeros((3, 2, 40, 64), dtype=F16, device="cuda") for _ in range(2)] for _ in range(2)]
    od = desc(outs[0][0])
    args = [c.args() for c in caches]

    def calls(i):
        g.check(dnn.paged_append_quantized(kd, k.data_ptr(), vd, v.data_ptr(), *args[i], counts.data_ptr()))
        caches[i].lengths.add_(counts)
        g.check(dnn.paged_read_quantized(*args[i], first.data_ptr(), od, outs[i][0].data_ptr(), od,
                                         outs[i][1].data_ptr()))

    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    say("capturing append8 and read8")
    with torch.cuda.graph(graph, stream=side):
        dnn.set_stream(torch.cuda.current_stream().cuda_stream)
        calls(1)
    dnn.set_stream(None)
    for step in range(6):
        k.mul_(1.3)
        counts.copy_(counts.roll(1))
        first.add_(1)
        calls(0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        caches[1].check(caches[0].state())
        for a, b in zip(*outs):
            assert torch.equal(a, b), f"replay {step}"
    del graph
    dnn.close()


def test_pages_past_32_bits(dnn):
    """Pools of more than 2^32 bytes, scales of more than 2^31 / 4: rows on the last pages."""
    from quant_cases import attend, attention_ref
    gen = torch.Generator().manual_seed(75)
    c = QuantCache(gen, [0, 0], 8, 16, 4, 128, True, room=64)
    pages = 270000
    c.k, c.v = (torch.empty((pages, 16, 8, 128), dtype=torch.int8, device="cuda").transpose(1, 2) for _ in range(2))
    c.ks, c.vs = (torch.empty((pages, 8, 4), device="cuda") for _ in range(2))
    last = torch.arange(pages - 8, pages).flip(0).reshape(2, 4).int()
    c.table = last.cuda()
    for t in (c.k, c.v, c.ks, c.vs):
        t[pages - 8:] = 1
    small = QuantCache(gen, [0, 0], 8, 16, 4, 128, True, room=64)
    k, v = rows(gen, 2, 8, 60, 128, BF16)
    for x in (c, small):
        append(dnn, x, k, v)
        x.n, x.lengths = [60, 60], ints([60, 60])
    out = [[torch.empty((2, 8, 60, 128), dtype=BF16, device="cuda") for _ in range(2)] for _ in range(2)]
    q = torch.randn((2, 16, 1, 128), generator=gen).to(BF16).cuda()
    o = [torch.empty_like(q) for _ in range(2)]
    for x, (a, b), y in zip((c, small), out, o):
        read(dnn, x, a, b)
        attend(dnn, x, q, y, 0.1)
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1]) and torch.equal(*o)
    K, V, _ = small.rows(0)
    ref, bound = attention_ref(q[0, :, 0].cpu(), K, V, 0.1)
    assert ((o[0][0, :, 0].cpu().double() - ref).abs() <= bound).all()
