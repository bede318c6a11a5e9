"""grxdnnPagedCacheAppend and grxdnnPagedCacheEvict, every pool byte checked."""
import math

import pytest
import torch

import grxcp_amd as g
from helpers import say
from paged_cases import Cache, append, desc, evict, evict_ref, guarded, ints

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def bits(t):
    return t.cpu().contiguous().view(torch.int16)


def guards_intact(pools):
    return all(torch.isnan(p[[0, -1]].float()).all() for p in pools)


# ---- append ------------------------------------------------------------------

APPENDS = [
    # dtype, d, heads, page, tokmajor, lengths before, T, counts
    (BF16, 128, 8, 16, True, [0, 15, 16, 17], 1, None),
    (F16, 64, 1, 1, False, [3, 0], 5, [5, 2]),
    (BF16, 64, 3, 7, True, [6, 7, 8, 0, 20], 23, [0, 23, -4, 100, 1]),
    (F16, 128, 2, 64, False, [63, 100], 300, None),
    (BF16, 64, 5, 256, True, [0], 1000, [999]),
    (F16, 64, 2, 16, False, [40, 1], 70, [0, 0]),
]


def check_append(dnn, c, k, v, counts):
    """c.n: lengths before. The pools before the call, with every row where it
    belongs, are the pools after it."""
    T = k.shape[2]
    want = [c.k.clone(), c.v.clone()]
    room, pages = c.width * c.page, c.k.shape[0]
    for i, n in enumerate(c.n):
        n = min(max(n, 0), room)
        m = T if counts is None else min(max(counts[i], 0), T)
        for t in range(min(m, room - n)):
            at = int(c.table[i, (n + t) // c.page])
            if 0 <= at < pages:
                for pool, rows in zip(want, (k, v)):
                    pool[at, :, (n + t) % c.page] = rows[i, :, t]
    say(f"append {tuple(k.shape)} to {c.n}")
    append(dnn, c, k, v, None if counts is None else ints(counts))
    assert torch.equal(bits(c.k), bits(want[0])) and torch.equal(bits(c.v), bits(want[1]))
    assert guards_intact(c.guarded)


@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(dnn, case):
    dtype, d, heads, page, tokmajor, lengths, T, counts = APPENDS[case]
    gen = torch.Generator().manual_seed(case)
    c = Cache(gen, dtype, lengths, heads, page, d, tokmajor, room=max(lengths) + T)
    shape = (len(lengths), T, heads, d)
    k, v = (torch.randn(shape, generator=gen).to(dtype).cuda().transpose(1, 2) for _ in range(2))
    if case % 2:
        k = k.contiguous()
    check_append(dnn, c, k, v, counts)


def test_append_beyond_the_room_and_to_missing_pages(dnn):
    """Rows without a place are dropped; the others and the rest of the pools stand."""
    gen = torch.Generator().manual_seed(20)
    c = Cache(gen, BF16, [30, 60, 5, 0], 2, 16, 64, True, room=64)
    c.table[2, 1] = -1
    c.table[3, 0], c.table[3, 2] = c.k.shape[0], 2 ** 31 - 1
    k, v = (torch.randn((4, 2, 40, 64), generator=gen).to(BF16).cuda() for _ in range(2))
    c.n = [30, 64, 5, 0]
    c.lengths = ints([30, 10 ** 9, 5, -3])
    check_append(dnn, c, k, v, None)


def test_append_interleaved_pools_and_a_packed_projection(dnn):
    """K and V pools as the halves of one [pages, page, 2, heads, d] array, the new
    rows as slices of one [B, T, q + k + v heads, d] projection, a repeated prompt as
    a broadcast batch."""
    gen = torch.Generator().manual_seed(21)
    c = Cache(gen, F16, [0, 37], 4, 16, 64, False, room=90)
    both = torch.zeros((c.k.shape[0], 16, 2, 4, 64), dtype=F16, device="cuda")
    c.k, c.v = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    c.store()
    qkv = torch.randn((1, 50, 16, 64), generator=gen).to(F16).cuda().expand(2, -1, -1, -1)
    check_append(dnn, c, qkv[:, :, 8:12].transpose(1, 2), qkv[:, :, 12:].transpose(1, 2), [50, 49])


def test_append_beyond_32_bits(dnn):
    gen = torch.Generator().manual_seed(22)
    c = Cache(gen, BF16, [0], 2, 16, 64, False, room=48, spare=0)
    stride = 2 ** 30 + 8
    flat = torch.empty(2 * stride + 2 * 2 * 16 * 64, dtype=BF16, device="cuda")
    far = torch.as_strided(flat, (3, 2, 2, 16, 64), (stride, 2048, 1024, 64, 1))
    far[:, 0], far[:, 1] = c.k, c.v
    c.k, c.v = far[:, 0], far[:, 1]
    k, v = (torch.randn((1, 2, 45, 64), generator=gen).to(BF16).cuda() for _ in range(2))
    append(dnn, c, k, v)
    page, row = c.places(0, torch.arange(45, device="cuda"))
    assert torch.equal(c.k[page, :, row], k[0].transpose(0, 1)) and torch.equal(c.v[page, :, row], v[0].transpose(0, 1))
    del flat, far
    c.k = c.v = None
    torch.cuda.empty_cache()


# ---- evict -------------------------------------------------------------------

def check_evict(dnn, c, w, budget, recent, bad=(), width=None, slots=None, inplace=False, spare=None):
    """w: host weights [B, heads, S]. bad: (sequence, entry) of the new table that name
    no page."""
    b, pages = len(c.n), c.k.shape[0]
    width = width or -(-budget // c.page)
    grown = b * width
    pools = [guarded(pages + grown, c.page, c.heads, c.d, c.dtype) for _ in range(2)]
    k, v = (p[1:-1] for p in pools)
    k[:pages], v[:pages] = c.k, c.v
    c.k, c.v = k, v
    new_table = ints(torch.randperm(grown).add(pages).reshape(b, width).tolist())
    for i, e in bad:
        new_table[i, e] = -1
    slots = slots or budget
    new_w = torch.full((b, c.heads, slots), math.nan, device="cuda")
    new_lengths = c.lengths if inplace else torch.full((b,), -9, dtype=torch.int32, device="cuda")
    want = [k.clone(), v.clone()]
    keep = torch.full((b, c.heads, budget), -1, dtype=torch.int32)
    want_w = torch.zeros((b, c.heads, slots))
    for i, n in enumerate(c.n):
        for h in range(c.heads):
            stay = evict_ref(w[i, h, :n], budget, recent)
            m = len(stay)
            keep[i, h, :m] = torch.tensor(stay, dtype=torch.int32)
            want_w[i, h, :m] = w[i, h, stay]
            to = torch.arange(m, device="cuda")
            dst, src = new_table[i, to // c.page].long(), c.places(i, torch.tensor(stay, device="cuda").long())
            ok = (dst >= 0) & (src[0] >= 0) & (src[0] < pages)
            for pool, old in zip(want, (k, v)):
                pool[dst[ok], h, (to % c.page)[ok]] = old[src[0][ok], h, src[1][ok]]
    say(f"evict {c.n} to {budget}, newest {recent}")
    got = evict(dnn, c, w.cuda(), budget, recent, new_table, new_w, new_lengths)
    assert torch.equal(got.cpu(), keep)
    assert new_lengths.tolist() == [min(n, budget) for n in c.n]
    assert torch.equal(new_w.cpu().view(torch.int32), want_w.view(torch.int32))
    assert torch.equal(bits(c.k), bits(want[0])) and torch.equal(bits(c.v), bits(want[1]))
    assert guards_intact(pools)
    return new_table, new_w, new_lengths


def weights(gen, c, ties=False):
    w = torch.rand((len(c.n), c.heads, c.width * c.page), generator=gen).pow(4)
    return (w * 6).floor() if ties else w


EVICTS = [
    # dtype, d, heads, page, tokmajor, lengths, budget, recent, ties
    (BF16, 128, 2, 16, True, [100, 50, 51, 0, 1], 50, 10, False),
    (F16, 64, 3, 7, False, [300, 299, 12], 33, 0, True),
    (BF16, 64, 1, 1, False, [40, 39, 38], 39, 39, False),
    (F16, 128, 2, 64, True, [5000, 1023, 1025], 1024, 1, True),
    (BF16, 64, 4, 256, False, [257, 2000], 1, 0, True),
    (F16, 64, 2, 16, True, [2000, 9], 1, 1, False),
    (BF16, 64, 2, 32, True, [40000, 100], 3000, 1500, False),
    (F16, 64, 1, 100, False, [70000], 65000, 11, True),
]


@pytest.mark.parametrize("case", range(len(EVICTS)))
def test_evict(dnn, case):
    dtype, d, heads, page, tokmajor, lengths, budget, recent, ties = EVICTS[case]
    gen = torch.Generator().manual_seed(50 + case)
    c = Cache(gen, dtype, lengths, heads, page, d, tokmajor)
    check_evict(dnn, c, weights(gen, c, ties), budget, recent, slots=budget + 3 * (case % 2), inplace=case % 3 == 0)


@pytest.mark.parametrize("kind", ["equal", "zero", "last_bit", "rising", "falling"])
def test_evict_weights_that_hardly_differ(dnn, kind):
    gen = torch.Generator().manual_seed(70)
    c = Cache(gen, BF16, [3001, 500], 2, 16, 64, True)
    S = c.width * c.page
    step = torch.arange(S, dtype=torch.float32)
    w = {"equal": torch.ones(S), "zero": torch.zeros(S), "last_bit": 1 + (step % 2) * 2.0 ** -23,
         "rising": step, "falling": -step}[kind].expand(2, 2, S).contiguous()
    check_evict(dnn, c, w, 400, 100)


def test_evict_special_weights(dnn):
    """NaN stays first, then +inf; -0 equals 0; -inf goes first."""
    gen = torch.Generator().manual_seed(71)
    c = Cache(gen, F16, [64, 64], 1, 16, 64, True)
    w = torch.zeros((2, 1, 64))
    w[0, 0, ::2] = -0.0
    w[0, 0, [40, 50]] = math.nan
    w[0, 0, 45] = math.inf
    w[0, 0, :5] = -math.inf
    w[1] = -1.0
    w[1, 0, 3] = -math.nan
    w[1, 0, 60:] = 100.0
    check_evict(dnn, c, w, 12, 2)


def test_evict_shared_prompt_and_missing_pages(dnn):
    """Two sequences that read one prompt's pages; source and target pages that do
    not exist are left out and nothing else is touched."""
    gen = torch.Generator().manual_seed(72)
    c = Cache(gen, BF16, [90, 90, 90], 2, 16, 64, False)
    c.table[1] = c.table[0]
    c.table[2, 1] = -1
    check_evict(dnn, c, weights(gen, c), 40, 8, bad=[(0, 1), (2, 2)], width=5)


def test_evict_lengths_outside_the_table(dnn):
    gen = torch.Generator().manual_seed(73)
    c = Cache(gen, BF16, [64, 0], 2, 16, 64, True, room=64)
    c.lengths = ints([10 ** 9, -1])
    check_evict(dnn, c, weights(gen, c), 20, 4)


def test_evict_after_append_and_capture(gpu):
    """append, then evict, in one captured graph: every replay against the eager
    result, with other work between."""
    gen = torch.Generator().manual_seed(74)
    dnn = g.Dnn()
    c = Cache(gen, F16, [100, 33], 2, 16, 64, True, room=200, spare=8)
    k, v = (torch.randn((2, 2, 3, 64), generator=gen).to(F16).cuda() for _ in range(2))
    w = weights(gen, c).cuda()
    new_table = c.spare[:8].reshape(2, 4).int().cuda()
    longer = ints([103, 36])
    kept = torch.empty((2, 2, 60), dtype=torch.int32, device="cuda")
    new_w, new_lengths = torch.empty((2, 2, 60), device="cuda"), torch.empty(2, dtype=torch.int32, device="cuda")
    kd, vd, td = c.descs()
    nd, wd, nwd, kn = desc(new_table), desc(w), desc(new_w), desc(k)

    def both():
        g.check(dnn.paged_append(kn, k.data_ptr(), kn, v.data_ptr(), kd, c.k.data_ptr(), vd, c.v.data_ptr(), td,
                                 c.table.data_ptr(), c.lengths.data_ptr(), None))
        g.check(dnn.paged_evict(kd, c.k.data_ptr(), vd, c.v.data_ptr(), td, c.table.data_ptr(), longer.data_ptr(),
                                wd, w.data_ptr(), 60, 5, kept.data_ptr(), nd, new_table.data_ptr(),
                                new_lengths.data_ptr(), nwd, new_w.data_ptr()))

    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        dnn.set_stream(torch.cuda.current_stream().cuda_stream)
        both()
    dnn.set_stream(None)
    for rep in range(4):
        k.copy_(torch.randn((2, 2, 3, 64), generator=gen).to(F16))
        w.copy_(weights(gen, c))
        start = [c.k.clone(), c.v.clone()]
        both()
        torch.cuda.synchronize()
        eager = [t.clone() for t in (c.k, c.v, kept, new_w, new_lengths)]
        for t, s in zip((c.k, c.v), start):
            t.copy_(s)
        for t in (kept, new_w, new_lengths):
            t.fill_(-5)
        torch.cuda.synchronize()
        say(f"replay {rep}")
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, (c.k, c.v, kept, new_w, new_lengths)):
            same = bits(a) if a.dtype == F16 else a.cpu(), bits(b) if b.dtype == F16 else b.cpu()
            assert torch.equal(*same), rep
    dnn.close()


def test_more_sequences_than_a_grid_has_rows(dnn):
    """70000 sequences of up to 6 slots: a token appended to each, then 3 slots kept."""
    gen = torch.Generator().manual_seed(60)
    b, heads, page, d, budget = 70000, 1, 2, 64, 3
    old = torch.randint(0, 6, (b,), generator=gen).int().cuda()
    order = torch.randperm(b * 5, generator=gen).int().cuda()
    table, new_table = order[: 3 * b].view(b, 3), order[3 * b:].view(b, 2)
    shape = (b * 5, heads, page, d)
    k, v = (torch.zeros(shape, dtype=BF16, device="cuda") for _ in range(2))
    # a row's values say whose and which it is: sequence and slot, exact in bf16
    who, slots = torch.arange(b, device="cuda"), torch.arange(6, device="cuda")
    rows = torch.stack([(who % 256)[:, None] + 0 * slots, (who // 256)[:, None] + 0 * slots, 0 * who[:, None] + slots], 2)
    for j in range(6):
        at = table[:, j // page].long()
        live = j < old
        k[at[live], 0, j % page, :3] = rows[live, j].to(BF16)
        v[at[live], 0, j % page, 1:4] = rows[live, j].to(BF16)
    kn, vn = (torch.zeros((b, heads, 1, d), dtype=BF16, device="cuda") for _ in range(2))
    kn[:, 0, 0, :3] = rows[who, old.long()].to(BF16)
    vn[:, 0, 0, 1:4] = rows[who, old.long()].to(BF16)
    kd, td = desc(k), desc(table)
    say("append to and eviction of 70000 sequences")
    nd = desc(kn)
    g.check(dnn.paged_append(nd, kn.data_ptr(), nd, vn.data_ptr(), kd, k.data_ptr(), kd, v.data_ptr(), td,
                             table.data_ptr(), old.data_ptr()))
    n = old + 1
    w = torch.randint(0, 4, (b, heads, 6), generator=gen).float().cuda()
    kept = torch.full((b, heads, budget), -7, dtype=torch.int32, device="cuda")
    new_n, new_w = torch.empty_like(n), torch.full((b, heads, 4), math.nan, device="cuda")
    g.check(dnn.paged_evict(kd, k.data_ptr(), kd, v.data_ptr(), td, table.data_ptr(), n.data_ptr(), desc(w),
                            w.data_ptr(), budget, 1, kept.data_ptr(), desc(new_table), new_table.data_ptr(),
                            new_n.data_ptr(), desc(new_w), new_w.data_ptr()))
    torch.cuda.synchronize()
    assert torch.equal(new_n, n.clamp(max=budget))
    # order of the old ones by (weight, lower slot), the newest before all
    rank = w[:, 0] * 8 - slots
    rank[slots == (n - 1)[:, None]] = 100
    rank[slots >= n[:, None]] = -100
    want = rank.argsort(1, descending=True)[:, :budget]
    want[torch.arange(budget, device="cuda") >= n[:, None]] = 99
    want = want.sort(1).values
    there = want < 99
    assert torch.equal(kept[:, 0], want.masked_fill(~there, -1).int())
    assert torch.equal(new_w[:, 0, :3], torch.where(there, w[:, 0].gather(1, want.clamp(max=5)), 0.0))
    assert (new_w[:, 0, 3] == 0).all()
    for i in range(budget):
        here = there[:, i]
        for pool, c in ((k, 0), (v, 1)):
            got = pool[new_table[here, i // page].long(), 0, i % page, c:c + 3]
            assert torch.equal(got, rows[who[here], want[here, i]].to(BF16)), (i, c)


def test_evict_of_more_heads_than_one_launch_takes(dnn):
    """2^22 + 24 (sequence, head) pairs of up to 2 slots, 1 of which stays: the heavier one,
    the lower of equal ones."""
    gen = torch.Generator(device="cuda").manual_seed(61)
    b, heads, d, shared = 2 ** 19 + 3, 8, 64, 1000
    def rand(hi, shape):
        return torch.randint(0, hi, shape, generator=gen, device="cuda", dtype=torch.int32)
    n, table = rand(3, (b,)), rand(shared, (b, 2))
    k, v = (torch.zeros((shared + b, heads, 1, d), dtype=BF16, device="cuda") for _ in range(2))
    k[:shared] = torch.randn((shared, heads, 1, d), generator=gen, device="cuda").to(BF16)
    v[:shared] = torch.randn((shared, heads, 1, d), generator=gen, device="cuda").to(BF16)
    w = rand(3, (b, heads, 2)).float()
    new_table = torch.arange(shared, shared + b, device="cuda", dtype=torch.int32)[:, None]
    kept = torch.full((b, heads, 1), -7, dtype=torch.int32, device="cuda")
    new_n, new_w = torch.full_like(n, -9), torch.full((b, heads, 1), math.nan, device="cuda")
    kd = desc(k)
    say("eviction of 2^22 + 24 heads")
    g.check(dnn.paged_evict(kd, k.data_ptr(), kd, v.data_ptr(), desc(table), table.data_ptr(), n.data_ptr(), desc(w),
                            w.data_ptr(), 1, 0, kept.data_ptr(), desc(new_table), new_table.data_ptr(),
                            new_n.data_ptr(), desc(new_w), new_w.data_ptr()), "evict")
    torch.cuda.synchronize()
    want = torch.where((n == 2)[:, None] & (w[..., 1] > w[..., 0]), 1, 0)
    want = want.masked_fill((n == 0)[:, None], -1)
    assert torch.equal(kept[..., 0].long(), want) and torch.equal(new_n, n.clamp(max=1))
    slot = want.clamp(min=0)
    assert torch.equal(new_w[..., 0], w.gather(2, slot[..., None])[..., 0].masked_fill(want < 0, 0.0))
    page = table.long().gather(1, slot)
    head = torch.arange(heads, device="cuda")
    for pool in (k, v):
        rows = pool[page, head, 0].masked_fill((want < 0)[..., None], 0.0)
        assert torch.equal(pool[shared:, :, 0], rows)
    del k, v, rows, w
    torch.cuda.empty_cache()
