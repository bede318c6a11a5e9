"""A paged key-value cache in 8 bits in torch tensors, and its operators in 64 bits (host)."""
import math

import torch

import grxcp_amd as g
from paged_cases import desc as float_desc
from paged_cases import ints

I8 = torch.int8


def desc(t):
    if t.dtype == I8:
        return g.TensorDesc(g.GRX_R_8I, list(t.shape), list(t.stride()))
    return float_desc(t)


def least8(x):
    """The least number of 8 significant bits, and at least 2^-126, that is not below x >= 0
    (64 bits); 0 for 0, NaN for what is not finite."""
    fraction, power = torch.frexp(x)
    up = torch.ldexp(torch.ceil(fraction * 256) / 256, power).clamp(min=2.0 ** -126)
    return torch.where(torch.isfinite(x), torch.where(x > 0, up, 0.0), math.nan)


def over(x, s):
    """x / s to the nearest code; 0 where s is 0 or not finite."""
    fine = (s > 0) & torch.isfinite(s)
    q = torch.round(x / torch.where(fine, s, 1.0))
    return torch.where(fine, q, 0.0).nan_to_num().to(I8)


class QuantCache:
    """Pools of codes and scales. Every slot that holds no token has code 77, every block that
    holds none the scale `unset` (NaN: what no call may look at). One page more on either
    side. Sequences begin with lengths[b] rows of normal values, appended by `append_ref`, or
    (quick) of any codes and scales."""

    def __init__(self, gen, lengths, heads, page, block, d, tokmajor=False, room=None, spare=3, unset=math.nan,
                 dtype=torch.bfloat16, scale=1.0, quick=False):
        b = len(lengths)
        self.heads, self.page, self.block, self.d = heads, page, block, d
        self.width = max(1, -(-max([room or 0, *lengths]) // page))
        total = b * self.width + spare
        shape = (total + 2, page, heads, d) if tokmajor else (total + 2, heads, page, d)
        order = torch.randperm(total, generator=gen)
        self.table = order[: b * self.width].reshape(b, self.width).int().cuda()
        self.spare = order[b * self.width:]
        self.pools = [torch.full(shape, 77, dtype=I8) for _ in range(2)]
        self.scales = [torch.full((total + 2, heads, page // block), unset) for _ in range(2)]
        self.n = [0] * b
        self.cuda(tokmajor)
        if quick:
            self.n = list(lengths)
            self.fill(gen, scale)
            self.lengths = ints(self.n)
            return
        new = [torch.randn((b, heads, max([*lengths, 1]), d), generator=gen).mul(scale).to(dtype) for _ in range(2)]
        self.lengths = ints(self.n)
        want = self.append_ref(*new, lengths)
        self.store(*want)
        self.n = [min(n, self.width * page) for n in lengths]
        self.lengths = ints(self.n)

    def cuda(self, tokmajor):
        self.guarded = [p.cuda() for p in self.pools]
        self.guarded_scales = [s.cuda() for s in self.scales]
        if tokmajor:
            self.guarded = [p.transpose(1, 2) for p in self.guarded]
        self.k, self.v = (p[1:-1] for p in self.guarded)
        self.ks, self.vs = (s[1:-1] for s in self.guarded_scales)
        del self.pools, self.scales

    def fill(self, gen, scale):
        """Codes of normal values and scales around them for every slot that holds a token."""
        k, v, ks, vs = self.state()
        table = self.table.cpu()
        for i, n in enumerate(self.n):
            at = torch.arange(n)
            page, row = table[i, at // self.page].long(), at % self.page
            for pool, scales in ((k, ks), (v, vs)):
                rows = torch.randn((n, self.heads, self.d), generator=gen).mul(36).round().clamp(-127, 127)
                pool[page, :, row] = rows.to(I8)
                by = torch.randn((n, self.heads), generator=gen).mul(0.3).exp().mul(3 * scale / 127)
                scales[page, :, row // self.block] = by
        self.store(k, v, ks, vs)

    def store(self, k, v, ks, vs):
        for to, x in ((self.k, k), (self.v, v), (self.ks, ks), (self.vs, vs)):
            to.copy_(x)

    def state(self):
        """k, v, ks, vs on the host."""
        return [t.cpu().clone() for t in (self.k, self.v, self.ks, self.vs)]

    def args(self):
        return (desc(self.k), self.k.data_ptr(), desc(self.v), self.v.data_ptr(), desc(self.ks), self.ks.data_ptr(),
                self.vs.data_ptr(), desc(self.table), self.table.data_ptr(), self.lengths.data_ptr())

    def append_ref(self, k, v, counts):
        """k, v, ks, vs (host) after rows of k, v [b, heads, T, d] behind the sequences."""
        out = self.state()
        table, pages, room = self.table.cpu(), self.k.shape[0], self.width * self.page
        for i, n in enumerate(self.n):
            n = min(max(n, 0), room)
            c = min(max(counts[i], 0), k.shape[2], room - n)
            for lo in range(n // self.block * self.block, n + c if c else 0, self.block):
                at, row = int(table[i, lo // self.page]), lo % self.page
                if not 0 <= at < pages:
                    continue
                old, end = max(0, n - lo), min(self.block, n + c - lo)
                for pool, scale, rows in ((out[0], out[2], k), (out[1], out[3], v)):
                    x = rows[i, :, lo + old - n:lo + end - n].cpu().double()
                    need = least8(x.abs().nan_to_num(nan=math.inf, posinf=math.inf).amax((1, 2)) / 127)
                    was = scale[at, :, row // self.block].double()
                    s = torch.where(torch.isnan(need) | torch.isnan(was), math.nan, torch.maximum(need, was)) if old else need
                    held = pool[at, :, row:row + old]
                    again = over(held.double() * was[:, None, None], s[:, None, None])
                    grew = (s > was) if old else torch.zeros_like(s, dtype=torch.bool)
                    pool[at, :, row:row + old] = torch.where(grew[:, None, None], again, held)
                    pool[at, :, row + old:row + end] = over(x, s[:, None, None])
                    scale[at, :, row // self.block] = s.float()
        return out

    def rows(self, i, n=None):
        """Keys and values of sequence i in 64 bits, [heads, n, d] each (host), and which of its
        slots are there."""
        n = self.n[i] if n is None else n
        k, v, ks, vs = self.state()
        at = torch.arange(n)
        page, row = self.table[i].cpu()[at // self.page].long(), at % self.page
        there = (page >= 0) & (page < k.shape[0])
        page = torch.where(there, page, 0)
        out = []
        for pool, scale in ((k, ks), (v, vs)):
            x = pool[page, :, row].double() * scale[page, :, row // self.block].double()[..., None]
            out.append(x.transpose(0, 1))
        return (*out, there)

    def check(self, want):
        """Codes, scales and guard pages after a call."""
        for name, got, ref in zip(("k", "v", "ks", "vs"), self.state(), want):
            if got.dtype == I8:
                bad = (got != ref).nonzero()
                assert not len(bad), f"{name}: {len(bad)} codes, first at {bad[0].tolist()}"
            else:
                assert torch.equal(got.view(torch.int32), ref.contiguous().view(torch.int32)) or (
                    torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(got.nan_to_num(-1), ref.nan_to_num(-1))
                ), name
        assert all((p[[0, -1]] == 77).all() for p in self.guarded)


def append(dnn, c, k, v, counts=None):
    g.check(dnn.paged_append_quantized(desc(k), k.data_ptr(), desc(v), v.data_ptr(), *c.args(),
                                       None if counts is None else counts.data_ptr()), "append")
    torch.cuda.synchronize()


def read(dnn, c, k, v, first=None):
    g.check(dnn.paged_read_quantized(*c.args(), None if first is None else first.data_ptr(), desc(k), k.data_ptr(),
                                     desc(v), v.data_ptr()), "read")
    torch.cuda.synchronize()


def attend(dnn, c, q, o, scale, expect=g.SUCCESS):
    from paged_cases import Workspace
    args = c.args()
    qd, od = desc(q), desc(o)
    ws = Workspace(dnn.paged_attention_quantized_workspace(qd, args[0], args[7]))
    st = dnn.paged_attention_quantized(g.AttnDesc(True, scale), qd, q.data_ptr(), *args, od, o.data_ptr(), ws.p, ws.size)
    assert st == expect, g.STATUS[st]
    torch.cuda.synchronize()


def attention_ref(q, K, V, scale, there=None):
    """o of one sequence and the bound on its error: q [H, d], K and V [heads, n, d] in 64 bits
    (host), there: which slots are.

    A query's value is off by at most 2^-22 of its row's largest one, a product with a code is
    exact, three fp32 roundings join the digits, three more the scales (softmaxScale * log2 e, the
    slot's, their product): a score is off by 2^-22 max|q| sum|k| and 8 half steps of sum |q k|, and
    e^x moves by that much, relatively. 2^-18 covers exp2, the fp32 sums and rescalings and the
    division. The weights keep 21 bits, but at least 2^-24 of 2^-11 of the largest scale of a
    value (and a power of two above); o is rounded once."""
    H, d = q.shape
    heads, n, _ = K.shape
    group = H // heads
    live = torch.ones(n, dtype=torch.bool) if there is None else there
    k, v = (x.repeat_interleave(group, 0)[:, live] for x in (K, V))
    if not k.shape[1]:
        zero = torch.zeros(H, d, dtype=torch.float64)
        return zero, zero
    q64 = q.double()
    s = torch.matmul(k, q64[:, :, None])[..., 0] * scale
    p = torch.softmax(s, 1)
    o = torch.matmul(p[:, None], v)[:, 0]
    size = torch.matmul(k.abs(), q64.abs()[:, :, None])[..., 0]
    off = 2.0 ** -22 * q64.abs().amax(1, keepdim=True) * k.abs().sum(2)
    delta = (off + 8 * 2.0 ** -24 * size).amax(1, keepdim=True) * scale
    rel = 2 * delta + 2.0 ** -18 + 2.0 ** -20
    u = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[q.dtype]
    mass = torch.matmul(p[:, None], v.abs())[:, 0]
    floor = k.shape[1] * 2.0 ** -34 * 2 * v.abs().amax((1, 2))[:, None]
    return o, u * o.abs() + (1 + u) * (rel * mass + floor) + (2.0 ** -25 if q.dtype == torch.float16 else 0.0)
