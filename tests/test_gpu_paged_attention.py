"""grxdnnPagedAttentionForward against attention in 64 bits, on the GPU."""
import math

import pytest
import torch

import grxcp_amd as g
from helpers import say
from paged_cases import HALF_STEP, Cache, Workspace, attend, attention_ref, desc, ints

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def check(dnn, c, q, scale, weights=False, decay=1.0, skip=None, inplace=False):
    """One call on cache c with queries q [B, H, 1, d], every output against 64 bits."""
    H = q.shape[1]
    old = None
    if weights:
        old = torch.rand((len(c.n), c.heads, c.width * c.page + 5), generator=torch.Generator().manual_seed(3))
        if decay == 0.0:
            old.fill_(math.nan)          # not read
        for i, n in enumerate(c.n):
            old[i, :, n:] = math.nan     # neither read nor written
    w = None if old is None else old.cuda()
    qh = q.cpu()
    o = q if inplace else torch.full_like(q, math.nan)
    attend(dnn, c, q, o, scale, w, decay)
    got = o.cpu().double()[:, :, 0]
    for i, n in enumerate(c.n):
        ref, p, bound, pbound = attention_ref(qh[i, :, 0], c.K[i], c.V[i], scale, skip=skip[i] if skip else ())
        assert torch.equal(torch.isnan(got[i]), torch.isnan(ref)), f"sequence {i}: NaN where 64 bits have none"
        far = torch.isinf(ref)
        assert torch.equal(got[i][far], ref[far])
        off = (got[i] - ref).abs() - bound
        assert not (off > 0).any(), f"sequence {i} of {n} slots: {off.max().item():.3g} past the bound"
        if w is None:
            continue
        wi, oi = w[i].cpu().double(), old[i].double()
        base = decay * oi[:, :n] if decay else torch.zeros(c.heads, n, dtype=torch.float64)
        there = torch.ones(n, dtype=torch.bool)
        want = base + p.reshape(c.heads, H // c.heads, n).sum(1)
        room = pbound.reshape(c.heads, H // c.heads, n).sum(1) + (H // c.heads + 2) * 2.0 ** -23 * want
        off = (wi[:, :n] - want).abs() - room
        assert not (off[:, there] > 0).any(), f"weights of {i}: {off.max().item():.3g} past the bound"
        assert torch.isnan(wi[:, n:]).all(), f"weights of {i}: entries behind the sequence were written"


def query(gen, b, H, d, dtype, scale=1.0):
    return torch.randn((b, H, 1, d), generator=gen).mul(scale).to(dtype).cuda()


def within(o, ref, bound):
    return bool(((o.cpu().double() - ref).abs() <= bound).all())


CASES = [
    # dtype, d, query heads, key heads, page, tokmajor, lengths, weights
    (BF16, 128, 8, 2, 16, True, [1, 0, 15, 16, 17, 200], False),
    (F16, 64, 4, 4, 16, False, [31, 32, 33, 63, 64, 65, 127, 128, 129], True),
    (BF16, 64, 6, 2, 7, True, [5, 700, 0, 6], True),
    (F16, 128, 16, 1, 1, False, [3, 257, 1], False),
    (BF16, 128, 17, 1, 64, True, [500, 20], True),
    (F16, 64, 32, 1, 256, False, [1000], True),
    (BF16, 64, 33, 1, 32, False, [100, 4], False),
    (BF16, 128, 40, 8, 16, True, [4097, 1, 2048], False),
    (F16, 128, 130, 2, 24, False, [333, 0, 90], True),
    (BF16, 64, 5, 5, 5, True, [0], True),
    (BF16, 128, 3, 3, 48, True, [0, 0, 0, 1], False),
    (F16, 64, 2, 1, 16, True, [9001], True),
    (BF16, 128, 1, 1, 100, False, [20000, 3, 12001], True),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_against_64_bits(dnn, case):
    dtype, d, H, heads, page, tokmajor, lengths, weights = CASES[case]
    gen = torch.Generator().manual_seed(100 + case)
    c = Cache(gen, dtype, lengths, heads, page, d, tokmajor)
    q = query(gen, len(lengths), H, d, dtype, 2.0)
    say(f"paged attention {CASES[case]}")
    check(dnn, c, q, d ** -0.5, weights, decay=0.9)


@pytest.mark.parametrize("b", [65, 300, 1100])
def test_many_ragged_sequences(dnn, b):
    """More sequences than a wave or a workgroup has lanes, many of them empty."""
    gen = torch.Generator().manual_seed(b)
    lengths = [0 if x % 3 == 0 else x % 211 for x in torch.randint(0, 10000, (b,), generator=gen).tolist()]
    c = Cache(gen, BF16, lengths, 2, 16, 64, True)
    say(f"paged attention, {b} ragged sequences")
    check(dnn, c, query(gen, b, 4, 64, BF16), 0.125, weights=True, decay=0.0)


def test_room_far_beyond_the_lengths(dnn):
    """A table wide enough for long sequences, of which none is long yet."""
    gen = torch.Generator().manual_seed(5)
    c = Cache(gen, F16, [40, 3, 0], 2, 16, 128, True, room=6000)
    c.table[:, 3:] = -1
    check(dnn, c, query(gen, 3, 4, 128, F16), 128 ** -0.5, weights=True, decay=0.5)


def test_lengths_outside_the_table_are_clamped(dnn):
    gen = torch.Generator().manual_seed(6)
    c = Cache(gen, BF16, [64, 64, 10], 2, 16, 64, True)
    c.lengths = ints([10 ** 9, -5, 10])
    c.n[1] = 0
    c.K[1], c.V[1] = c.K[1][:, :0], c.V[1][:, :0]
    check(dnn, c, query(gen, 3, 2, 64, BF16), 0.125, weights=True)


def test_slots_on_pages_that_do_not_exist_are_absent(dnn):
    """Entries outside the pool weigh nothing, wherever they stand; a sequence of
    only such pages is as empty as one of length 0."""
    gen = torch.Generator().manual_seed(7)
    c = Cache(gen, F16, [100, 300, 32], 2, 16, 64, False)
    c.table[0, 2] = -1
    c.table[1, 0] = c.k.shape[0]
    c.table[1, 18] = 2 ** 31 - 1
    c.table[2, :] = -3
    skip = [range(32, 48), [*range(16), *range(288, 300)], range(32)]
    check(dnn, c, query(gen, 3, 4, 64, F16), 0.125, weights=True, skip=skip)


def test_shared_pages_and_a_shared_table_row(dnn):
    """Sequences that share a prompt's pages; a table row broadcast to all."""
    gen = torch.Generator().manual_seed(8)
    c = Cache(gen, BF16, [200, 150], 2, 16, 128, True)
    c.table = c.table[:1].expand(2, -1)
    c.K[1], c.V[1] = c.K[0][:, :150], c.V[0][:, :150]
    check(dnn, c, query(gen, 2, 8, 128, BF16), 128 ** -0.5, weights=True)


def test_strides_and_in_place(dnn):
    """q and o as views of [B, 1, H, d] and of a packed QKV row, o over q, pools with
    padded pages, heads and slots, a table and weights with a pitch."""
    gen = torch.Generator().manual_seed(9)
    c = Cache(gen, F16, [77, 0, 500], 4, 16, 64, False)
    k = torch.full((c.k.shape[0], 5, 18, 72), math.nan, dtype=F16, device="cuda")
    v = torch.full((c.k.shape[0], 4, 17, 80), math.nan, dtype=F16, device="cuda")
    k[:, :4, :16, :64], v[:, :4, :16, :64] = c.k, c.v
    c.k, c.v = k[:, :4, :16, :64], v[:, :4, :16, :64]
    wide = torch.full((3, c.width + 3), -1, dtype=torch.int32, device="cuda")
    wide[:, :c.width] = c.table
    c.table = wide[:, :c.width]
    qkv = torch.randn((3, 1, 24, 64), generator=gen).to(F16).cuda()
    check(dnn, c, qkv[:, :, :16].transpose(1, 2), 0.125, weights=True)
    rest = qkv[:, :, 16:].clone()
    check(dnn, c, qkv[:, :, :16].transpose(1, 2), 0.125, inplace=True)
    assert torch.equal(qkv[:, :, 16:], rest)


def test_rows_behind_the_batch_stay(dnn):
    """Output and weights of sequences that the call does not have."""
    gen = torch.Generator().manual_seed(10)
    c = Cache(gen, BF16, [130, 7], 2, 16, 64, True)
    q = query(gen, 4, 4, 64, BF16)
    o = torch.full((4, 4, 1, 64), 7.0, dtype=BF16, device="cuda")
    w = torch.full((4, 2, c.width * 16), 3.0, device="cuda")
    attend(dnn, c, q[:2], o[:2], 0.125, w[:2])
    assert (o[2:] == 7.0).all() and (w[2:] == 3.0).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scores_of_minus_infinity(dnn, dtype):
    """-inf scores weigh nothing wherever they lie; a row of only such is NaN."""
    gen = torch.Generator().manual_seed(11)
    c = Cache(gen, dtype, [300, 300, 40], 1, 16, 64, True)
    c.K[0][:, :140, 0] = -math.inf
    c.K[1][:, 5:, 0] = -math.inf
    c.K[2][:, :, 0] = -math.inf
    c.store()
    q = query(gen, 3, 2, 64, dtype)
    q[..., 0] = 1.0
    check(dnn, c, q, 0.125)


def test_nan_and_infinity_stay_in_their_head(dnn):
    """A NaN key makes its own head's rows NaN, an infinite value shows as it is, and
    other heads and sequences do not see them."""
    gen = torch.Generator().manual_seed(12)
    c = Cache(gen, BF16, [70, 70], 3, 16, 64, True)
    c.K[0][1, 33, 7] = math.nan
    c.V[1][2, 69, 5] = math.inf
    c.store()
    check(dnn, c, query(gen, 2, 6, 64, BF16), 0.125)


@pytest.mark.parametrize("dtype,factor", [(BF16, 1.0), (F16, 1.0), (BF16, 300.0), (F16, 40.0)])
def test_growing_and_peaked_scores(dnn, dtype, factor):
    """Scores that grow along the cache (the maximum moves in every tile), and one
    slot that outweighs thousands of small ones whose sum still counts."""
    gen = torch.Generator().manual_seed(13)
    c = Cache(gen, dtype, [2000, 4000], 1, 16, 64, False)
    c.K[0][0, :, :] = torch.linspace(-1, 1, 2000)[:, None].expand(2000, 64).to(dtype)
    c.K[1][0, :, :] = 0.0
    c.K[1][0, 1234, :] = 1.3
    c.V[1][0].abs_()
    c.store()
    q = torch.full((2, 2, 1, 64), factor, dtype=dtype, device="cuda")
    check(dnn, c, q, 0.125)


def test_scale_and_decay_reach_the_kernel(dnn):
    gen = torch.Generator().manual_seed(14)
    c = Cache(gen, BF16, [90], 2, 16, 64, True)
    q = query(gen, 1, 4, 64, BF16)
    for scale, decay in ((0.01, 0.0), (1.0, 0.25), (3.0, 2.0)):
        check(dnn, c, q, scale, weights=True, decay=decay)


def test_weights_add_up_over_steps(dnn):
    """Two calls on the same weights: the sum of both, 64 queries' mass in all."""
    gen = torch.Generator().manual_seed(15)
    c = Cache(gen, F16, [257], 2, 16, 64, True)
    w = torch.zeros((1, 2, c.width * 16), device="cuda")
    for _ in range(4):
        q = query(gen, 1, 16, 64, F16)
        attend(dnn, c, q, torch.empty_like(q), 0.125, w)
    # every query's weights sum to 1 within its fp32 roundings
    assert torch.allclose(w.sum(2).cpu(), torch.full((1, 2), 32.0), rtol=2.0 ** -16, atol=0)
    assert (w[:, :, 257:] == 0).all()


def test_pools_beyond_32_bits(dnn):
    """A page more than 2^31 elements from its pool's base."""
    gen = torch.Generator().manual_seed(16)
    c = Cache(gen, BF16, [50], 2, 16, 64, False, spare=0)
    stride = 2 ** 30 + 8
    pages = c.k.shape[0]
    flat = torch.empty((pages - 1) * stride + 2 * 2 * 16 * 64, dtype=BF16, device="cuda")
    far = torch.as_strided(flat, (pages, 2, 2, 16, 64), (stride, 2048, 1024, 64, 1))
    far[:, 0], far[:, 1] = c.k, c.v
    c.k, c.v = far[:, 0], far[:, 1]
    assert (pages - 1) * stride > 2 ** 31
    check(dnn, c, query(gen, 1, 4, 64, BF16), 0.125, weights=True)
    del flat, far
    c.k = c.v = None
    torch.cuda.empty_cache()


def test_two_streams_at_once(gpu):
    """Two handles on two streams, a workspace each, calls that overlap."""
    gen = torch.Generator().manual_seed(17)
    dnns, streams, sets = [g.Dnn() for _ in range(2)], [torch.cuda.Stream() for _ in range(2)], []
    for i in range(2):
        c = Cache(gen, BF16, [3000, 17], 2, 16, 128, True)
        q = query(gen, 2, 8, 128, BF16)
        o = torch.empty_like(q)
        kd, vd, td = c.descs()
        qd = desc(q)
        size = dnns[i].paged_attention_workspace(qd, kd, td)
        sets.append((c, q, o, kd, vd, td, qd, Workspace(size)))
        dnns[i].set_stream(streams[i].cuda_stream)
    torch.cuda.synchronize()
    ad = g.AttnDesc(False, 128 ** -0.5)
    for _ in range(20):
        for dnn, (c, q, o, kd, vd, td, qd, ws) in zip(dnns, sets):
            g.check(dnn.paged_attention(ad, qd, q.data_ptr(), kd, c.k.data_ptr(), vd, c.v.data_ptr(), td,
                                        c.table.data_ptr(), c.lengths.data_ptr(), 0.0, None, None, qd, o.data_ptr(),
                                        ws.p, ws.size))
    torch.cuda.synchronize()
    for c, q, o, *_ in sets:
        for i in range(2):
            ref, _, bound, _ = attention_ref(q[i, :, 0].cpu(), c.K[i], c.V[i], 128 ** -0.5)
            assert within(o[i, :, 0], ref, bound)
    for d in dnns:
        d.close()


def test_captured_call_follows_lengths_and_tables(gpu):
    """Two captured calls with a workspace each, replayed in turn with eager work
    between, after the lengths, the table and the queries have changed."""
    gen = torch.Generator().manual_seed(18)
    dnn = g.Dnn()
    calls, ad = [], g.AttnDesc(True, 0.125)
    for weights in (True, False):
        c = Cache(gen, F16, [600, 4, 90], 2, 16, 64, True)     # lengths 0 .. 3 below
        q = query(gen, 3, 4, 64, F16)
        o = torch.empty_like(q)
        w = torch.zeros((3, 2, c.width * 16), device="cuda") if weights else None
        kd, vd, td = c.descs()
        qd, wd = desc(q), desc(w) if weights else None
        ws = Workspace(dnn.paged_attention_workspace(qd, kd, td, wd))
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            dnn.set_stream(torch.cuda.current_stream().cuda_stream)
            st = dnn.paged_attention(ad, qd, q.data_ptr(), kd, c.k.data_ptr(), vd, c.v.data_ptr(), td,
                                     c.table.data_ptr(), c.lengths.data_ptr(), 0.0, wd,
                                     w.data_ptr() if weights else None, qd, o.data_ptr(), ws.p, ws.size)
        assert st == g.SUCCESS
        calls.append((c, q, o, w, graph, (kd, vd, td, qd, wd, ws)))
    dnn.set_stream(None)
    for rep in range(4):
        for c, q, o, w, graph, _ in calls:
            n = [600 - 131 * rep, rep, 90 - rep]
            c.lengths.copy_(ints(n))
            q.copy_(query(gen, 3, 4, 64, F16))
            if rep == 2:       # the first sequence moves to the pages of the third
                pages = c.table[2].clone()
                c.table[0, :6] = pages[:6]
                n[0] = 80
                c.lengths.copy_(ints(n))
                c.K[0], c.V[0] = c.K[2][:, :90], c.V[2][:, :90]
            if rep == 3:
                n[0] = 40
                c.lengths.copy_(ints(n))
            torch.cuda.synchronize()
            say(f"replay {rep}")
            graph.replay()
            torch.cuda.synchronize()
            for i in range(3):
                ref, p, bound, _ = attention_ref(q[i, :, 0].cpu(), c.K[i][:, :n[i]], c.V[i][:, :n[i]], 0.125)
                assert within(o[i, :, 0], ref, bound), (rep, i)
                if w is not None:
                    got = w[i, :, :n[i]].cpu().double()
                    assert torch.allclose(got, p.reshape(2, 2, n[i]).sum(1), rtol=1e-4, atol=1e-7), (rep, i)
            eager = torch.full_like(q, math.nan)
            attend(dnn, c, q, eager, 0.125)      # a workspace of its own
            assert torch.equal(eager, o), rep
    dnn.close()


def test_same_bits_every_time(dnn):
    gen = torch.Generator().manual_seed(19)
    c = Cache(gen, BF16, [5000, 12, 700], 2, 16, 128, True)
    q = query(gen, 3, 8, 128, BF16)
    outs = []
    for _ in range(3):
        o, w = torch.empty_like(q), torch.zeros((3, 2, c.width * 16), device="cuda")
        attend(dnn, c, q, o, 128 ** -0.5, w)
        outs.append((o, w))
    assert all(torch.equal(o, outs[0][0]) and torch.equal(w, outs[0][1]) for o, w in outs)


@pytest.mark.parametrize("b,H,heads,d,room,tokmajor,weights,kernel", [
    (3, 8, 2, 64, 256, True, False, "whole1"), (40, 8, 4, 64, 512, True, True, "whole1"),
    (3, 8, 2, 128, 512, True, False, "split1"),
    (20, 4, 4, 64, 700, True, True, "split1"), (64, 4, 4, 64, 700, True, True, "split4"),
    (20, 4, 4, 64, 700, False, True, "split1"), (40, 12, 6, 64, 600, True, False, "split2"),
    (2, 66, 2, 128, 600, True, True, "split1"), (40, 132, 4, 64, 640, True, False, "split4"),
])
def test_every_kernel_choice(dnn, capfd, monkeypatch, b, H, heads, d, room, tokmajor, weights, kernel):
    """The choice that GRXDNN_LOG names, on ragged lengths from none to the room's."""
    gen = torch.Generator().manual_seed(20)
    lengths = [0, 1, room] + torch.randint(0, room + 1, (max(0, b - 3),), generator=gen).tolist()
    c = Cache(gen, BF16, lengths[:b], heads, 20 if room % 20 == 0 else 16, d, tokmajor, room=room)
    capfd.readouterr()
    monkeypatch.setenv("GRXDNN_LOG", "1")
    check(dnn, c, query(gen, b, H, d, BF16), d ** -0.5, weights=weights, decay=0.5)
    monkeypatch.delenv("GRXDNN_LOG")
    log = [x for x in capfd.readouterr().err.splitlines() if x.startswith("grxdnn: paged attention ")]
    assert len(log) == 1 and log[0].endswith(f"weights={int(weights)} kernel={kernel}"), log


@pytest.mark.parametrize("room", [8, 640])      # one launch, split and joined
def test_more_sequences_than_a_grid_has_rows(dnn, room):
    """70000 sequences over shared pages, most of them short; 40 are held to 64 bits, the
    empty ones to 0."""
    gen = torch.Generator().manual_seed(21)
    b, heads, d, page, pages = 70000, 1, 64, 8, 90
    k, v = (torch.randn((pages, heads, page, d), generator=gen).to(BF16) for _ in range(2))
    table = torch.randint(0, pages, (b, room // page), generator=gen).int()
    lengths = torch.randint(0, 9, (b,), generator=gen).int()
    some = torch.cat([torch.randint(0, b, (35,), generator=gen), torch.tensor([0, 65534, 65535, 65536, b - 1])])
    lengths[some] = torch.randint(1, room + 1, (40,), generator=gen).int()
    q = query(gen, b, 2, d, BF16)
    o, w = torch.full_like(q, math.nan), torch.zeros((b, heads, room), device="cuda")
    kc, vc, tc, lc = (t.cuda() for t in (k, v, table, lengths))
    kd, td, qd, wd = desc(kc), desc(tc), desc(q), desc(w)
    ws = Workspace(dnn.paged_attention_workspace(qd, kd, td, wd))
    say(f"paged attention of {b} sequences, room {room}")
    g.check(dnn.paged_attention(g.AttnDesc(True, 0.125), qd, q.data_ptr(), kd, kc.data_ptr(), kd, vc.data_ptr(), td,
                                tc.data_ptr(), lc.data_ptr(), 1.0, wd, w.data_ptr(), qd, o.data_ptr(), ws.p, ws.size))
    torch.cuda.synchronize()
    for i in some.tolist():
        n = lengths[i].item()
        K, V = (t[table[i].long()].transpose(0, 1).reshape(heads, room, d)[:, :n] for t in (k, v))
        ref, p, bound, pbound = attention_ref(q[i, :, 0].cpu(), K, V, 0.125)
        assert within(o[i, :, 0], ref, bound), i
        assert ((w[i, 0, :n].cpu().double() - p.sum(0)).abs() <= pbound.sum(0) + 2.0 ** -21 * p.sum(0)).all(), i
    assert (o[lengths == 0] == 0).all() and torch.isfinite(o).all()
    # every query's weights sum to 1 within their fp32 roundings
    assert torch.allclose(w.sum((1, 2)).cpu(), 2.0 * (lengths > 0), rtol=2.0 ** -14, atol=0)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("H,heads,room", [(4, 2, 64), (40, 1, 64), (4, 2, 6000), (64, 2, 6000)])
def test_values_are_weighted_by_more_than_16_bits(dnn, dtype, H, heads, room):
    """Values of either sign that nearly cancel: o's one rounding is small there, and what
    16-bit weights would cost stands far above it. As attention_ref, but for the weights,
    which are held to 2^-15."""
    gen = torch.Generator().manual_seed(22)
    c = Cache(gen, dtype, [5, 16, 40, 3], heads, 16, 64, True, room=room)
    q, scale = query(gen, 4, H, 64, dtype), 0.125 / 8
    o = torch.full_like(q, math.nan)
    say(f"weights of the values, {dtype}, {H} on {heads} heads, room {room}")
    attend(dnn, c, q, o, scale)
    for i, n in enumerate(c.n):
        k, v = (t[i].double().repeat_interleave(H // heads, 0) for t in (c.K, c.V))
        qi = q[i, :, 0].cpu().double()
        ref, p, _, _ = attention_ref(q[i, :, 0].cpu(), c.K[i], c.V[i], scale)
        size = torch.matmul(k.abs(), qi.abs()[:, :, None])[..., 0] * scale
        rel = 2 * (64 + 3) * 2.0 ** -24 * size.amax(1, keepdim=True) + 2.0 ** -18
        u = HALF_STEP[dtype]
        mass = torch.matmul(p[:, None], v.abs())[:, 0]
        assert within(o[i, :, 0], ref, u * ref.abs() + (1 + u) * (2.0 ** -15 + rel) * mass + 2.0 ** -25), i


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("room", [80, 800])
def test_an_infinite_value_shows_whatever_it_weighs(dnn, dtype, room):
    """Infinite values of slots that weigh much, little, and as much as the heaviest (a power
    of two: no bits behind the first)."""
    gen = torch.Generator().manual_seed(23)
    c = Cache(gen, dtype, [70, 70, 1, 70], 2, 16, 64, True, room=room)
    for t in (c.K[0], c.K[3]):
        t[:] = 0.0
    c.K[3][:, 40:, 0] = -80 * math.log(2)                 # scores of -10 log 2, about 2^-10
    c.V[0][0, 3, 5], c.V[0][1, 69, 6] = math.inf, -math.inf
    c.V[1][0, :, 5] = math.inf
    c.V[1][1, 33, 7] = -math.inf
    c.V[2][1, 0, 9] = math.inf
    c.V[3][0, 50, 5], c.V[3][1, 1, 6] = -math.inf, math.inf
    c.store()
    q = query(gen, 4, 4, 64, dtype)
    q[..., 0] = 1.0
    check(dnn, c, q, 0.125)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("b,H,heads,d", [(1, 4, 2, 64), (40, 16, 2, 128), (40, 16, 2, 64), (3, 16, 16, 128)])
def test_infinite_values_in_the_last_part(dnn, capfd, monkeypatch, dtype, b, H, heads, d):
    """Sequences in every number of parts whose last slots hold infinite values: these show,
    and nothing turns into NaN."""
    gen = torch.Generator().manual_seed(24)
    lengths = [1500 - 37 * (i % 23) for i in range(b)]
    c = Cache(gen, dtype, lengths, heads, 16, d, False)
    for v in c.V:
        v[0, -1, 5], v[heads - 1, -20:, d - 1] = math.inf, -math.inf
    c.store()
    capfd.readouterr()
    monkeypatch.setenv("GRXDNN_LOG", "1")
    check(dnn, c, query(gen, b, H, d, dtype), 0.5 * d ** -0.5)
    assert "kernel=split" in capfd.readouterr().err
