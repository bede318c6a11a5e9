"""A paged key-value cache in torch tensors, and its operators in 64 bits (host)."""
import math

import torch

import grxcp_amd as g

GRX = {torch.bfloat16: g.GRX_R_16BF, torch.float16: g.GRX_R_16F, torch.float32: g.GRX_R_32F,
       torch.int32: g.GRX_R_32I}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32 = 2.0 ** -24          # half a step of fp32


def desc(t):
    return g.TensorDesc(GRX[t.dtype], list(t.shape), list(t.stride()))


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def guarded(pages, page, heads, d, dtype, tokmajor=False, fill=math.nan):
    """A pool of `pages` pages with one more on either side: [pages + 2, heads, page, d]."""
    shape = (pages + 2, page, heads, d) if tokmajor else (pages + 2, heads, page, d)
    p = torch.full(shape, fill, dtype=dtype, device="cuda")
    return p.transpose(1, 2) if tokmajor else p


class Cache:
    """Pools whose every slot holds `fill` (NaN: what no call may read) but for the
    first lengths[b] slots of each sequence. tokmajor: memory is [pages, page, heads,
    d]. room: slots that a table row has room for (the longest sequence's, rounded
    up to pages, if None)."""

    def __init__(self, gen, dtype, lengths, heads, page, d, tokmajor=False, fill=math.nan, room=None, spare=3,
                 scale=1.0):
        b = len(lengths)
        self.dtype, self.heads, self.page, self.d = dtype, heads, page, d
        self.width = max(1, -(-max([room or 0, *lengths]) // page))
        total = b * self.width + spare
        self.guarded = [guarded(total, page, heads, d, dtype, tokmajor, fill) for _ in range(2)]
        self.k, self.v = (p[1:-1] for p in self.guarded)
        order = torch.randperm(total, generator=gen)
        self.spare = order[b * self.width:]
        table = order[: b * self.width].reshape(b, self.width).int()
        self.table = table.cuda()
        self.lengths = ints(lengths)
        self.n = list(lengths)
        self.K = [torch.randn((heads, n, d), generator=gen).mul(scale).to(dtype) for n in lengths]
        self.V = [torch.randn((heads, n, d), generator=gen).to(dtype) for n in lengths]
        self.store()

    def places(self, i, slots):
        return self.table[i, slots // self.page].long(), slots % self.page

    def store(self):
        """The host rows into the pools."""
        for i, n in enumerate(self.n):
            if n:
                page, row = self.places(i, torch.arange(n, device="cuda"))
                self.k[page, :, row] = self.K[i].transpose(0, 1).cuda()
                self.v[page, :, row] = self.V[i].transpose(0, 1).cuda()

    def descs(self):
        return desc(self.k), desc(self.v), desc(self.table)


def attention_ref(q, K, V, scale, skip=()):
    """o, p, the bound on o's error and the one on p's, of one sequence: q [H, d], K
    and V [heads, n, d] (host). skip: slots that are not there.

    A score is a sum of d products of 16-bit values in fp32 (every product exact):
    off by at most (d + 1) half steps of sum |q k|, and two more for the scale
    (softmaxScale * log2 e, rounded once, and the product with it); e^x moves by that
    much, relatively. 2^-18 covers exp2, the fp32 sums and rescalings and the division.
    The values' weights are rounded to the 16-bit type (half a step each), o once."""
    H, d = q.shape
    heads, n, _ = K.shape
    group = H // heads
    live = torch.ones(n, dtype=torch.bool)
    live[list(skip)] = False
    k = K.double().repeat_interleave(group, 0)[:, live]
    v = V.double().repeat_interleave(group, 0)[:, live]
    if not k.shape[1]:
        zero = torch.zeros(H, n, dtype=torch.float64)
        return torch.zeros(H, d, dtype=torch.float64), zero, torch.zeros(H, d, dtype=torch.float64), zero
    s = torch.matmul(k, q.double()[:, :, None])[..., 0] * scale
    p = torch.softmax(s, 1)
    o = torch.matmul(p[:, None], v)[:, 0]
    size = torch.matmul(k.abs().nan_to_num(posinf=0.0), q.double().abs()[:, :, None])[..., 0] * scale
    delta = (d + 3) * F32 * size.amax(1, keepdim=True)
    rel = 2 * delta + 2.0 ** -18
    u = HALF_STEP[q.dtype]
    # sum p |v|: what relative errors of the weights act on
    mass = torch.matmul(p[:, None], v.abs())[:, 0]
    bound = u * o.abs() + (1 + u) * (u + rel) * mass + (2.0 ** -25 if q.dtype == torch.float16 else 0.0)
    full = torch.zeros(H, n, dtype=torch.float64)
    full[:, live] = p
    fullrel = torch.zeros(H, n, dtype=torch.float64)
    fullrel[:, live] = rel * p
    return o, full, bound, fullrel


def evict_ref(w, budget, recent):
    """Slots that stay, in order: w is one head's weights (host fp32)."""
    n = w.numel()
    if n <= budget:
        return list(range(n))
    old = max(0, n - recent)
    rank = [(-math.inf if math.isnan(x) else -x, j) for j, x in enumerate(w[:old].tolist())]
    # NaN before +inf
    rank.sort(key=lambda t: (0 if math.isnan(w[t[1]]) else 1, t[0], t[1]))
    return sorted(j for _, j in rank[:budget - recent]) + list(range(old, n))


class Workspace:
    """Device bytes that hold 0xFF (NaN) before a call."""

    def __init__(self, size):
        self.t = torch.full((max(size, 16),), 0xFF, dtype=torch.uint8, device="cuda")
        self.size = size
        self.p = self.t.data_ptr()


def attend(dnn, c, q, o, scale, weights=None, decay=1.0, expect=g.SUCCESS):
    kd, vd, td = c.descs()
    qd, od = desc(q), desc(o)
    wd = None if weights is None else desc(weights)
    ws = Workspace(dnn.paged_attention_workspace(qd, kd, td, wd))
    st = dnn.paged_attention(g.AttnDesc(True, scale), qd, q.data_ptr(), kd, c.k.data_ptr(), vd, c.v.data_ptr(),
                             td, c.table.data_ptr(), c.lengths.data_ptr(), decay, wd,
                             None if weights is None else weights.data_ptr(), od, o.data_ptr(), ws.p, ws.size)
    assert st == expect, g.STATUS[st]
    torch.cuda.synchronize()


def append(dnn, c, k, v, counts=None):
    kd, vd, td = c.descs()
    g.check(dnn.paged_append(desc(k), k.data_ptr(), desc(v), v.data_ptr(), kd, c.k.data_ptr(), vd, c.v.data_ptr(),
                             td, c.table.data_ptr(), c.lengths.data_ptr(),
                             None if counts is None else counts.data_ptr()), "append")
    torch.cuda.synchronize()


def evict(dnn, c, w, budget, recent, new_table, new_w, new_lengths):
    kd, vd, td = c.descs()
    kept = torch.full((len(c.n), c.heads, budget), -7, dtype=torch.int32, device="cuda")
    g.check(dnn.paged_evict(kd, c.k.data_ptr(), vd, c.v.data_ptr(), td, c.table.data_ptr(), c.lengths.data_ptr(),
                            desc(w), w.data_ptr(), budget, recent, kept.data_ptr(), desc(new_table),
                            new_table.data_ptr(), new_lengths.data_ptr(), desc(new_w), new_w.data_ptr()), "evict")
    torch.cuda.synchronize()
    return kept
