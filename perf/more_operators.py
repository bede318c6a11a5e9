"""Serving and training work between a projection and a key-value cache in 8 bits, as
cases that can be prepared, run, counted and checked.

The operators are grxDNN's

  rope          queries and keys, each head's row normalised (root mean square) and
                rotated by its token's position, in one pass
  rope_grad     the gradient of that in queries, keys and gains
  append8       rows of new keys and values into the pages of their sequences in 8 bits,
                with one scale for each block of slots and head
  read8         rows of such a cache back in 16 bits
  attend8       attention of one new token per sequence over such a cache

Where `own` is false the same work is done with elementary torch operations in 32 bits
(angles and quotients in 64). A pool is [pages, heads, page, d] int8, or [pages, page,
heads, d] where a case says tokmajor; scales are [pages, heads, page / block].

What append8 gives back are the cache's codes and scales: a code is a whole number, and
every code has to be the same on both sides. A block's scale is its largest magnitude
/ 127, rounded up to 8 significant bits, so a quotient of a 16-bit value and a scale is
either half way between two codes or further from there than fp32 can lose.
"""
import math

import torch

own = False

TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6


def listed():
    return [
        # One token for each of 64 running sequences, far along their contexts: the step
        # before each decoding attention, where latency is all.
        dict(name="rope_step", kind="rope", dtype="bf16", b=64, s=1, hq=32, hkv=8, d=128, rotary=128, pairs=False,
             norm=True, base=1e6, ctx=100000),
        # The queries and keys of a batch of prompts.
        dict(name="rope_prompts", kind="rope", dtype="bf16", b=4, s=4096, hq=32, hkv=8, d=128, rotary=128,
             pairs=False, norm=True, base=5e5, ctx=0),
        # fp32, neighbouring pairs, half of each head rotated, no norm, an odd length.
        dict(name="rope_pairs_odd", kind="rope", dtype="f32", b=3, s=1001, hq=16, hkv=16, d=64, rotary=32,
             pairs=True, norm=False, base=1e4, ctx=7),
        # The gradient of a small step with one key head and wide heads.
        dict(name="rope_grad_odd", kind="rope_grad", dtype="f16", b=1, s=777, hq=5, hkv=1, d=256, rotary=256,
             pairs=False, norm=True, base=1e4, ctx=0),
        # The gradient of a training step.
        dict(name="rope_grad_train", kind="rope_grad", dtype="bf16", b=4, s=2048, hq=32, hkv=8, d=128, rotary=128,
             pairs=False, norm=True, base=5e5, ctx=0),
        # One token for each of 64 sequences into half-filled blocks.
        dict(name="append8_step", kind="append8", dtype="bf16", b=64, hkv=8, d=128, page=16, block=16, tokmajor=True,
             ctx=1000, tokens=1, ragged=False),
        # The keys and values of a batch of prompts of different lengths, just computed.
        dict(name="append8_prompts", kind="append8", dtype="f16", b=8, hkv=8, d=128, page=64, block=32, tokmajor=False,
             ctx=0, tokens=4000, ragged=True),
        # A few short sequences back in 16 bits, a scale for each token.
        dict(name="read8_few", kind="read8", dtype="f16", b=3, hkv=8, d=64, page=16, block=1, tokmajor=True,
             lo=1001, hi=1500),
        # The earlier tokens of long prompts, for the attention of their next chunk.
        dict(name="read8_prompts", kind="read8", dtype="bf16", b=8, hkv=8, d=128, page=16, block=16, tokmajor=True,
             lo=5000, hi=8192),
        # One user with a short conversation: the smallest call.
        dict(name="attend8_one_short", kind="attend8", dtype="bf16", b=1, hq=32, hkv=8, d=128, page=16, block=16,
             tokmajor=True, lo=201, hi=201),
        # A serving batch of grouped heads, sequences of 33 to 4096 tokens.
        dict(name="attend8_batch", kind="attend8", dtype="bf16", b=48, hq=32, hkv=8, d=128, page=16, block=16,
             tokmajor=True, lo=33, hi=4096),
        # Two long documents, a scale for each token: few rows, all of the work along the cache.
        dict(name="attend8_long", kind="attend8", dtype="f16", b=2, hq=32, hkv=4, d=128, page=64, block=1,
             tokmajor=False, lo=131072, hi=131072),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "rope_grad", "rope_grad", "append8", "append8", "read8", "attend8", "attend8",
                       "attend8"])
    if kind in ("rope", "rope_grad"):
        while True:
            c = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), b=_log(rng, 1, 128),
                     s=1 if rng.random() < 0.3 else _log(rng, 1, 8192), hkv=_log(rng, 1, 16),
                     d=rng.choice([64, 128, 128, 256]), pairs=rng.random() < 0.3, norm=rng.random() < 0.7,
                     base=rng.choice([1e4, 5e5, 1e6]), ctx=rng.randrange(0, 200000))
            c["hq"] = c["hkv"] * rng.choice([1, 2, 4, 5, 8])
            c["rotary"] = c["d"] if rng.random() < 0.6 else 16 * rng.randint(1, c["d"] // 16)
            values = c["b"] * c["s"] * (c["hq"] + c["hkv"]) * c["d"] * SIZE[c["dtype"]]
            if c["hq"] <= 64 and values <= (2 ** 27 if kind == "rope" else 2 ** 26):
                return c
    while True:
        page = rng.choice([1, 7, 16, 32, 64, 256])
        c = dict(kind=kind, dtype=rng.choice(["bf16", "f16"]), b=_log(rng, 1, 128), hkv=rng.choice([1, 2, 4, 8, 16, 32]),
                 d=rng.choice([64, 128]), page=page, block=rng.choice([x for x in (1, 4, 7, 16, 64, 256) if page % x == 0]),
                 tokmajor=rng.random() < 0.5)
        if kind == "append8":
            c.update(ctx=rng.randrange(0, 2000), tokens=1 if rng.random() < 0.3 else _log(rng, 1, 8192),
                     ragged=rng.random() < 0.5)
            rows, most = c["b"] * (c["ctx"] + c["tokens"]), 2 ** 24
        else:
            hi = _log(rng, 1, 131072 if kind == "attend8" else 16384)
            c.update(lo=hi if rng.random() < 0.4 else rng.randrange(0, hi + 1), hi=hi)
            rows, most = c["b"] * hi, 2 ** 26 if kind == "attend8" else 2 ** 25
            if kind == "attend8":
                c["hq"] = c["hkv"] * rng.choice([1, 2, 4, 5, 8, 16])
                rows *= 1 if c["hq"] <= 64 else 4
        if rows * c["hkv"] * c["d"] <= most:
            return c


# ---- preparing -------------------------------------------------------------

def _lengths(case):
    """The sequences' lengths, evenly from lo to hi; the seed gives their order."""
    b, lo, hi = case["b"], case["lo"], case["hi"]
    return [hi if b == 1 else lo + (hi - lo) * i // (b - 1) for i in range(b)]


def _counts(case):
    """New tokens per sequence: all of them, or evenly from none to all."""
    b, t = case["b"], case["tokens"]
    return [t if b == 1 or not case["ragged"] else t * (i + 1) // b for i in range(b)]


class _Rand:
    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, shape, dtype="f32", scale=1.0):
        x = torch.randn(shape, generator=self.gen, device="cuda", dtype=torch.float32)
        return x.mul_(scale).to(TORCH[dtype])

    def ints(self, lo, hi, shape, dtype=torch.int32):
        return torch.randint(lo, hi, shape, generator=self.gen, device="cuda", dtype=dtype)

    def order(self, n):
        return torch.randperm(n, generator=self.gen, device="cuda")


def _ints(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def _heads(r, case, heads, dtype):
    """What a projection gives for `heads` heads: [b, heads, s, d], a view of [b, s, heads, d]."""
    return r.normal((case["b"], case["s"], heads, case["d"]), dtype).transpose(1, 2)


def _codes(case, r, pages):
    h, n, d = case["hkv"], case["page"], case["d"]
    # what normal values of a block of largest magnitude 3 to 4 have
    if case["tokmajor"]:
        return r.normal((pages, n, h, d), scale=36.0).round_().clamp_(-127, 127).to(torch.int8).transpose(1, 2)
    return r.normal((pages, h, n, d), scale=36.0).round_().clamp_(-127, 127).to(torch.int8)


def _scales(case, r, pages):
    """Scales of 8 significant bits, those of blocks of normal values."""
    x = r.normal((pages, case["hkv"], case["page"] // case["block"])).mul_(0.1).exp_().mul_(3.0 / 127)
    return x.bfloat16().float()


def _tables(needs, pages):
    """Page tables: sequence i has needs[i] of `pages` (an order of the pool), then
    entries of -1."""
    need, width = _ints(needs).long(), max(1, max(needs))
    at = torch.arange(width, device="cuda")
    first = need.cumsum(0) - need
    own_page = pages[(first[:, None] + at).clamp(max=pages.numel() - 1)]
    return torch.where(at < need[:, None], own_page, -1).int()


def prepare(case, seed):
    r, s = _Rand(seed), dict(case)
    kind, dtype, b, hkv, d = case["kind"], case["dtype"], case["b"], case["hkv"], case["d"]
    if kind in ("rope", "rope_grad"):
        hq = case["hq"]
        # queries, keys and values come side by side out of one projection
        packed = r.normal((b, case["s"], hq + 2 * hkv, d), dtype)
        s["q"], s["k"] = packed[:, :, :hq].transpose(1, 2), packed[:, :, hq:hq + hkv].transpose(1, 2)
        s["qg"], s["kg"] = ((1.0 + r.normal((d,), scale=0.2)).to(TORCH[dtype]) for _ in range(2))
        # a sequence's tokens follow one another from where its context ends
        start = r.ints(case["ctx"] // 2, case["ctx"] + 1, (b, 1)) if case["ctx"] else _ints([[0]] * b)
        s["positions"] = (start + torch.arange(case["s"], device="cuda", dtype=torch.int32)).contiguous()
        i = torch.arange(0, case["rotary"], 2, device="cuda", dtype=torch.float64)
        s["inv_freq"] = (case["base"] ** (-i / case["rotary"])).float()
        if kind == "rope":
            s["yq"], s["yk"] = (torch.empty((b, case["s"], h, d), device="cuda", dtype=TORCH[dtype]).transpose(1, 2)
                                for h in (hq, hkv))
        else:
            s["dyq"], s["dyk"] = _heads(r, case, hq, dtype), _heads(r, case, hkv, dtype)
            s["dq"], s["dk"] = torch.empty_like(s["dyq"]), torch.empty_like(s["dyk"])
            if case["norm"]:
                s["dqg"], s["dkg"] = (torch.empty(d, device="cuda") for _ in range(2))
        return s

    page, block = case["page"], case["block"]
    perm = r.order(b)
    if kind == "append8":
        before = [case["ctx"]] * b
        # room for the new tokens and the block behind them
        needs = [-(-(n + case["tokens"] + 2 * block) // page) for n in before]
        s["lengths"], s["counts"] = _ints(before), _ints(_counts(case))[perm]
        shape = (b, case["tokens"], hkv, d)      # as the projection gives them
        s["k_new"], s["v_new"] = (r.normal(shape, dtype).transpose(1, 2) for _ in range(2))
    else:
        s["lengths"] = _ints(_lengths(case))[perm]
        needs = [-(-n // page) for n in s["lengths"].tolist()]
    pages = r.order(max(1, sum(needs)))
    s["k"], s["v"] = _codes(case, r, pages.numel()), _codes(case, r, pages.numel())
    s["ks"], s["vs"] = _scales(case, r, pages.numel()), _scales(case, r, pages.numel())
    s["table"] = _tables(needs, pages)
    if kind == "read8":
        s["k_out"], s["v_out"] = (torch.empty((b, hkv, case["hi"], d), device="cuda", dtype=TORCH[dtype])
                                  for _ in range(2))
    elif kind == "attend8":
        s["q"] = r.normal((b, case["hq"], 1, d), dtype, 2.0)
        s["o"] = torch.empty_like(s["q"])
    return s


# ---- the plain forms ---------------------------------------------------------

def _cos_sin(s):
    """Of every token's angles, [b, 1, s, rotary / 2]."""
    angle = s["positions"].double()[:, None, :, None] * s["inv_freq"].double()
    return angle.cos().float(), angle.sin().float()


def _rotate(x, s, cos, sin):
    n = s["rotary"]
    y = x.clone()
    if s["pairs"]:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        y[..., 0:n:2], y[..., 1:n:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :n // 2], x[..., n // 2:n]
        y[..., :n // 2], y[..., n // 2:n] = a * cos - b * sin, b * cos + a * sin
    return y


def _inverse_rms(x):
    return (x.square().mean(-1, keepdim=True) + EPS).rsqrt()


def _plain_rope(s):
    cos, sin = _cos_sin(s)
    for x, gain, y in ((s["q"], s["qg"], s["yq"]), (s["k"], s["kg"], s["yk"])):
        x = x.float()
        if s["norm"]:
            x = x * _inverse_rms(x) * gain.float()
        y.copy_(_rotate(x, s, cos, sin))
    return [s["yq"], s["yk"]]


def _plain_rope_grad(s):
    cos, sin = _cos_sin(s)
    out = []
    for x, gain, dy, dx, dgain in ((s["q"], s["qg"], s["dyq"], s["dq"], s.get("dqg")),
                                   (s["k"], s["kg"], s["dyk"], s["dk"], s.get("dkg"))):
        g = _rotate(dy.float(), s, cos, -sin)
        if s["norm"]:
            x = x.float()
            r = _inverse_rms(x)
            n = x * r
            dgain.copy_((g * n).sum((0, 1, 2), dtype=torch.float64))
            g = g * gain.float()
            g = r * (g - n * (g * n).mean(-1, keepdim=True))
            out.append(dgain)
        dx.copy_(g)
        out.append(dx)
    return out


def _places(table, slots, page):
    """(page, row in it) of each sequence's slots [b, t]."""
    at = torch.gather(table.long(), 1, (slots // page).clamp(max=table.shape[1] - 1))
    return at.clamp(min=0), slots % page


def _round_up_8(x):
    """The least number of 8 significant bits that is not below x >= 0, and not below
    2^-126 where x is not 0."""
    up = ((x.contiguous().view(torch.int32) + 0xffff) & ~0xffff).view(torch.float32)
    return torch.where(x > 0, up.clamp(min=2.0 ** -126), 0.0)


def _plain_append8(s):
    page, block, d, heads = s["page"], s["block"], s["d"], s["hkv"]
    n = s["lengths"].long()[:, None]
    blocks = (2 * block - 2 + s["tokens"]) // block                # that a sequence's new rows can touch
    slot = n // block * block + torch.arange(blocks * block, device="cuda")
    old, new = slot < n, (slot >= n) & (slot < n + s["counts"][:, None])
    at, row = _places(s["table"], slot, page)
    first = slice(None, None, block)                               # of each block
    live, held = new.reshape(-1, blocks, block).any(2)[..., None], old[:, first, None]
    t = (slot - n).clamp(0, s["tokens"] - 1)[:, None, :, None].expand(-1, heads, -1, d)
    for pool, scales, rows in ((s["k"], s["ks"], s["k_new"]), (s["v"], s["vs"], s["v_new"])):
        x = torch.gather(rows, 2, t).transpose(1, 2).double() * new[..., None, None]   # [b, slots, heads, d]
        most = x.abs().reshape(-1, blocks, block, heads, d).amax((2, 4))
        before = scales[at[:, first], :, row[:, first] // block]    # [b, blocks, heads]
        scale = _round_up_8((most / 127).float())
        scale = torch.where(held, torch.maximum(scale, before), scale)
        wide, was = (z.double().repeat_interleave(block, 1)[..., None] for z in (scale, before))
        wide = wide.clamp(min=2.0 ** -126)
        code = pool[at, :, row]
        code = torch.where(old[..., None, None], (code * was / wide).round().clamp(-127, 127).to(torch.int8), code)
        code = torch.where(new[..., None, None], (x / wide).round().clamp(-127, 127).to(torch.int8), code)
        keep = live.repeat_interleave(block, 1)[..., None]
        pool[at, :, row] = torch.where(keep, code, pool[at, :, row])
        scales[at[:, first], :, row[:, first] // block] = torch.where(live, scale, before)
    return [s["k"], s["v"], s["ks"], s["vs"]]


def _plain_read8(s):
    slot = torch.arange(s["hi"], device="cuda").expand(s["b"], -1)
    at, row = _places(s["table"], slot, s["page"])
    live = (slot < s["lengths"][:, None])[..., None, None]
    for pool, scales, out in ((s["k"], s["ks"], s["k_out"]), (s["v"], s["vs"], s["v_out"])):
        x = pool[at, :, row].float() * scales[at, :, row // s["block"]][..., None]
        out.copy_(torch.where(live, x, 0.0).transpose(1, 2))
    return [s["k_out"], s["v_out"]]


def _plain_attend8(s):
    b, hq, hkv, d = s["b"], s["hq"], s["hkv"], s["d"]
    table = s["table"].long().clamp(min=0)
    width = table.shape[1] * s["page"]

    def rows(pool, scales):
        x = pool[table].float() * scales[table].repeat_interleave(s["block"], 3)[..., None]
        return x.transpose(1, 2).reshape(b, hkv, width, d)

    k, v = rows(s["k"], s["ks"]), rows(s["v"], s["vs"])
    live = (torch.arange(width, device="cuda") < s["lengths"][:, None])[:, None, None, :]
    q = s["q"].float().reshape(b, hkv, hq // hkv, d)
    score = (torch.matmul(q, k.transpose(2, 3)) * d ** -0.5).masked_fill(~live, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = (score - top).exp()
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-38)
    s["o"].copy_(torch.matmul(p, v).reshape(b, hq, 1, d))
    return [s["o"]]


# ---- the framework's calls -----------------------------------------------------

class _Lib:
    """The process's handle, on the stream that torch uses, and its workspace."""
    g = dnn = workspace = None

    @classmethod
    def get(cls):
        if cls.g is None:
            import grxcp_amd
            cls.g, cls.dnn = grxcp_amd, grxcp_amd.Dnn()
            cls.types = {torch.bfloat16: grxcp_amd.GRX_R_16BF, torch.float16: grxcp_amd.GRX_R_16F,
                         torch.float32: grxcp_amd.GRX_R_32F, torch.int32: grxcp_amd.GRX_R_32I,
                         torch.int8: grxcp_amd.GRX_R_8I}
            cls.dnn.set_stream(torch.cuda.current_stream().cuda_stream)
        return cls

    @classmethod
    def room(cls, size):
        if size and (cls.workspace is None or cls.workspace.numel() < size):
            cls.workspace = torch.empty(size, device="cuda", dtype=torch.uint8)
        return cls.workspace.data_ptr() if size else None


DESCRIBED = ("q", "k", "yq", "yk", "dyq", "dyk", "dq", "dk", "qg", "v", "ks", "k_new", "v_new", "k_out", "v_out",
             "table", "o")


def _describe(s, L):
    """The descriptors of a state's shapes and the workspace they need: made once, as a
    program does for the buffers that it decodes or trains with."""
    d = {n: L.g.TensorDesc(L.types[s[n].dtype], list(s[n].shape), list(s[n].stride())) for n in DESCRIBED if n in s}
    d["size"] = 0
    if s["kind"] == "attend8":
        d["attn"] = L.g.AttnDesc(True, s["d"] ** -0.5)
        d["size"] = L.dnn.paged_attention_quantized_workspace(d["q"], d["k"], d["table"])
    elif s["kind"] == "rope_grad" and s["norm"]:
        d["size"] = L.dnn.qk_norm_rope_workspace(d["q"], d["k"], d["qg"])
    return d


def _own(s):
    L = _Lib.get()
    kind, dnn, check = s["kind"], L.dnn, L.g.check
    d = s.get("descs")
    if d is None:
        d = s["descs"] = _describe(s, L)

    def p(name):
        return s[name].data_ptr()

    if kind in ("rope", "rope_grad"):
        norm = s["norm"]
        gains = (d["qg"], p("qg"), p("kg")) if norm else (None, None, None)
        mode = L.g.ROPE_PAIRS if s["pairs"] else L.g.ROPE_HALVES
        angles = (mode, s["rotary"], p("positions"), p("inv_freq"))
        if kind == "rope":
            check(dnn.qk_norm_rope(d["q"], p("q"), d["k"], p("k"), *gains, EPS, *angles, d["yq"], p("yq"), d["yk"],
                                   p("yk")))
            return [s["yq"], s["yk"]]
        check(dnn.qk_norm_rope_backward(d["q"], p("q"), d["k"], p("k"), *gains, EPS, *angles, d["dyq"], p("dyq"),
                                        d["dyk"], p("dyk"), d["dq"], p("dq"), d["dk"], p("dk"),
                                        p("dqg") if norm else None, p("dkg") if norm else None, L.room(d["size"]),
                                        d["size"]))
        return [s["dqg"], s["dq"], s["dkg"], s["dk"]] if norm else [s["dq"], s["dk"]]
    cache = (d["k"], p("k"), d["v"], p("v"), d["ks"], p("ks"), p("vs"), d["table"], p("table"), p("lengths"))
    if kind == "append8":
        check(dnn.paged_append_quantized(d["k_new"], p("k_new"), d["v_new"], p("v_new"), *cache, p("counts")))
        return [s["k"], s["v"], s["ks"], s["vs"]]
    if kind == "read8":
        check(dnn.paged_read_quantized(*cache, None, d["k_out"], p("k_out"), d["v_out"], p("v_out")))
        return [s["k_out"], s["v_out"]]
    check(dnn.paged_attention_quantized(d["attn"], d["q"], p("q"), *cache, d["o"], p("o"), L.room(d["size"]),
                                        d["size"]))
    return [s["o"]]


def run(state):
    if own:
        return _own(state)
    return {"rope": _plain_rope, "rope_grad": _plain_rope_grad, "append8": _plain_append8, "read8": _plain_read8,
            "attend8": _plain_attend8}[state["kind"]](state)


# ---- counting --------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind in ("rope", "rope_grad"):
        tokens = case["b"] * case["s"]
        n, size = tokens * (case["hq"] + case["hkv"]) * case["d"], SIZE[case["dtype"]]
        small = 4 * tokens + 2 * case["rotary"] + (2 * case["d"] * size if case["norm"] else 0)
        if kind == "rope":
            return {"bytes": 2 * n * size + small, "flops": (7.0 if case["norm"] else 3.0) * n}
        if not case["norm"]:
            return {"bytes": 2 * n * size + small, "flops": 3.0 * n}
        return {"bytes": 3 * n * size + small + 8 * case["d"], "flops": 14.0 * n}
    values, block = 2 * case["hkv"] * case["d"], case["block"]    # of a token's key and value
    if kind == "append8":
        # each new row read and its codes written, the scales of the blocks that get rows
        counts = _counts(case)
        scales = sum(-(-(case["ctx"] % block + c) // block) for c in counts if c) * 8 * case["hkv"]
        return {"bytes": 3 * values * sum(counts) + scales + 8 * case["b"], "flops": 3.0 * values * sum(counts)}
    lengths = _lengths(case)
    t, pages = sum(lengths), sum(-(-n // case["page"]) for n in lengths)
    scales = 8 * case["hkv"] * sum(-(-n // block) for n in lengths)
    if kind == "read8":
        return {"bytes": values * t + scales + 4 * pages + 2 * values * case["b"] * case["hi"], "flops": 1.0 * values * t}
    return {"bytes": values * t + scales + 4 * pages + 4 * case["b"] * case["hq"] * case["d"],
            "flops": 4.0 * case["hq"] * case["d"] * t}


# ---- in 64 bits ----------------------------------------------------------------

def _turn(x, case, positions, inv_freq, way):
    """Each pair of x [b, h, s, d] as a complex number, times e^(i way angle)."""
    n = case["rotary"]
    pair = x[..., :n].unflatten(-1, (n // 2, 2) if case["pairs"] else (2, n // 2))
    pair = pair.movedim(-1 if case["pairs"] else -2, -1)
    angle = positions.double()[:, None, :, None] * inv_freq.double()
    z = torch.complex(pair[..., 0], pair[..., 1]) * torch.polar(torch.ones_like(angle), way * angle)
    both = torch.stack([z.real, z.imag], -1 if case["pairs"] else -2).flatten(-2)
    return torch.cat([both, x[..., n:]], -1)


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "rope":
        out = []
        for x, gain in ((s["q"], s["qg"]), (s["k"], s["kg"])):
            x = x.double()
            if case["norm"]:
                x = x / torch.sqrt(torch.sum(x * x, -1, keepdim=True) / case["d"] + EPS) * gain.double()
            out.append(_turn(x, case, s["positions"], s["inv_freq"], 1.0))
        return out
    if kind == "rope_grad":
        out = []
        for x, gain, dy in ((s["q"], s["qg"], s["dyq"]), (s["k"], s["kg"], s["dyk"])):
            u = _turn(dy.double(), case, s["positions"], s["inv_freq"], -1.0)
            if not case["norm"]:
                out.append(u)
                continue
            x = x.double()
            length = torch.sqrt(torch.sum(x * x, -1, keepdim=True) / case["d"] + EPS)
            out.append((u * (x / length)).sum((0, 1, 2)))
            w = u * gain.double()
            out.append(w / length - x * torch.sum(w * x, -1, keepdim=True) / (case["d"] * length ** 3))
        return out
    page, block = case["page"], case["block"]
    if kind == "append8":
        if case["b"] * (1 + case["tokens"] // block) > 4000:
            return None                      # block by block, it would take too long
        out = []
        for pool, scales, rows in ((s["k"], s["ks"], s["k_new"]), (s["v"], s["vs"], s["v_new"])):
            pool, scales = pool.clone(), scales.double()
            for i, (n, c) in enumerate(zip(s["lengths"].tolist(), s["counts"].tolist())):
                table = s["table"][i].tolist()
                for lo in range(n // block * block, n + c if c else 0, block):
                    at, row = table[lo // page], lo % page
                    old, hi = max(0, n - lo), min(block, n + c - lo)
                    x = rows[i, :, lo + old - n:lo + hi - n].double()             # [heads, new, d]
                    most = x.abs().amax((1, 2))
                    fraction, power = torch.frexp(torch.div(most, torch.full_like(most, 127.0)))
                    need = torch.ldexp(torch.ceil(fraction * 256), power - 8)
                    was = scales[at, :, row // block].clone()
                    now = torch.maximum(was, need) if old else need
                    by = now.clamp(min=1e-300)[:, None, None]
                    kept = pool[at, :, row:row + old].double() * was[:, None, None]
                    pool[at, :, row:row + old] = torch.round(kept / by).to(torch.int8)
                    pool[at, :, row + old:row + hi] = torch.round(x / by).to(torch.int8)
                    scales[at, :, row // block] = now
            out.append((pool, scales))
        return [out[0][0], out[1][0], out[0][1], out[1][1]]

    def sequence(pool, scales, i, n):
        """Rows 0 .. n-1 of sequence i, [heads, n, d]."""
        pages = s["table"][i, :-(-n // page)].long()
        x = torch.cat(list(pool[pages]), 1)[:, :n].double()
        by = torch.cat(list(scales[pages]), 1).double()
        return x * by[:, torch.arange(n, device="cuda") // page * (page // block)
                      + torch.arange(n, device="cuda") % page // block, None]

    lengths = s["lengths"].tolist()
    if kind == "read8":
        out = []
        for pool, scales in ((s["k"], s["ks"]), (s["v"], s["vs"])):
            x = torch.zeros(s["k_out"].shape, device="cuda", dtype=torch.float64)
            for i, n in enumerate(lengths):
                if n:
                    x[i, :, :n] = sequence(pool, scales, i, n)
            out.append(x)
        return out
    o = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    group = case["hq"] // case["hkv"]
    for i, n in enumerate(lengths):
        if n:
            k, v = sequence(s["k"], s["ks"], i, n), sequence(s["v"], s["vs"], i, n)
            for h in range(case["hkv"]):
                q = s["q"][i, h * group:(h + 1) * group, 0].double()
                p = torch.softmax(torch.mm(k[h], q.T).T / math.sqrt(case["d"]), dim=1)
                o[i, h * group:(h + 1) * group, 0] = torch.mm(p, v[h])
    return [o]
