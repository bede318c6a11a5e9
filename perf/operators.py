"""Serving and policy-training work on a paged key-value cache and a vocabulary, as
cases that can be prepared, run, counted and checked.

The operators are grxDNN's

  append        rows of new keys and values into the pages of their sequences
  attend        attention of one new token per sequence over the pages, with the
                weights that the cache's slots received where the case asks for them
  evict         the slots of largest accumulated weight and the newest ones into
                pages of their own, in order
  logprob       log probabilities of given tokens, with log-sum-exp, entropy and
                the top alternatives
  logprob_grad  the gradient of log probabilities and entropies in the logits

Where `own` is false the same work is done with elementary torch operations in 32
bits. A pool is [pages, heads, page, d], or [pages, page, heads, d] where a case
says tokmajor; both are handed on as [pages, heads, page, d] views.
"""
import math

import torch

own = False

TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
DECAY = 0.98


def listed():
    return [
        # One token for each of 64 running sequences: the step before each decoding
        # attention, where latency is all.
        dict(name="append_step", kind="append", dtype="bf16", b=64, hkv=8, d=128, page=16, tokmajor=True,
             ctx=1000, tokens=1, ragged=False),
        # The keys and values of a batch of prompts of different lengths, just computed.
        dict(name="append_prompts", kind="append", dtype="f16", b=8, hkv=8, d=128, page=32, tokmajor=False,
             ctx=0, tokens=4000, ragged=True),
        # One user with a short conversation: the smallest call.
        dict(name="attend_one_short", kind="attend", dtype="bf16", b=1, hq=32, hkv=8, d=128, page=16,
             tokmajor=True, lo=201, hi=201, weights=False),
        # A serving batch of grouped heads, sequences of 33 to 4096 tokens.
        dict(name="attend_batch", kind="attend", dtype="bf16", b=48, hq=32, hkv=8, d=128, page=16,
             tokmajor=True, lo=33, hi=4096, weights=False),
        # One long document: few rows, all of the work along the cache.
        dict(name="attend_long", kind="attend", dtype="bf16", b=2, hq=32, hkv=4, d=128, page=64,
             tokmajor=False, lo=131072, hi=131072, weights=False),
        # A head per query head, and the weights that eviction goes by.
        dict(name="attend_weights", kind="attend", dtype="f16", b=24, hq=16, hkv=16, d=64, page=32,
             tokmajor=True, lo=500, hi=3001, weights=True),
        # A few sequences back to half of their slots.
        dict(name="evict_few", kind="evict", dtype="f16", b=3, hkv=8, d=64, page=16, tokmajor=True,
             lo=1001, hi=1500, budget=512, recent=64),
        # A batch of long contexts back to a quarter.
        dict(name="evict_batch", kind="evict", dtype="bf16", b=16, hkv=8, d=128, page=16, tokmajor=False,
             lo=6000, hi=8192, budget=2048, recent=256),
        # What a decoding step answers with: the sampled tokens and 8 alternatives.
        dict(name="logprob_step", kind="logprob", dtype="bf16", rows=32, vocab=131072, top=8),
        # fp32 logits of a batch of answers over a vocabulary of odd size.
        dict(name="logprob_answers", kind="logprob", dtype="f32", rows=4096, vocab=32001, top=0),
        # The gradient of a small step, odd vocabulary.
        dict(name="logprob_grad_odd", kind="logprob_grad", dtype="f16", rows=500, vocab=50001, entropy=False),
        # The gradient of a large training step with an entropy bonus.
        dict(name="logprob_grad_large", kind="logprob_grad", dtype="bf16", rows=8192, vocab=65536, entropy=True),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "evict", "evict", "logprob",
                       "logprob", "logprob_grad", "logprob_grad"])
    half = rng.choice(["bf16", "f16"])
    if kind in ("logprob", "logprob_grad"):
        while True:
            c = dict(kind=kind, dtype=rng.choice(["bf16", "f16", "f32"]), rows=_log(rng, 1, 8192),
                     vocab=_log(rng, 1000, 262144))
            if c["rows"] * c["vocab"] <= (2 ** 27 if kind == "logprob" else 2 ** 28):
                break
        if kind == "logprob":
            c["top"] = rng.choice([0, 1, 5, 20, 64])
        else:
            c["entropy"] = rng.random() < 0.5
        return c
    while True:
        c = dict(kind=kind, dtype=half, b=_log(rng, 1, 128), hkv=rng.choice([1, 2, 4, 8, 16, 32]),
                 d=rng.choice([64, 128]), page=rng.choice([1, 7, 16, 32, 64, 256]), tokmajor=rng.random() < 0.5)
        if kind == "append":
            c.update(ctx=rng.randrange(0, 2000), tokens=_log(rng, 1, 8192), ragged=rng.random() < 0.5)
            rows = c["b"] * (c["ctx"] + c["tokens"])
        else:
            hi = _log(rng, 1, 131072) if kind == "attend" else _log(rng, 64, 16384)
            c.update(lo=hi if rng.random() < 0.4 else rng.randrange(0 if kind == "attend" else 1, hi + 1), hi=hi)
            rows = c["b"] * hi
            if kind == "attend":
                c["hq"] = c["hkv"] * rng.choice([1, 2, 4, 5, 8, 16])
                c["weights"] = rng.random() < 0.4
                rows *= 1 if c["hq"] <= 64 else 4
            else:
                c["budget"] = rng.randrange(1, hi + 1)
                c["recent"] = rng.randrange(0, c["budget"] + 1)
        if rows * c["hkv"] * c["d"] <= 2 ** 27:
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

    def ints(self, lo, hi, shape):
        return torch.randint(lo, hi, shape, generator=self.gen, device="cuda", dtype=torch.int32)

    def order(self, n):
        return torch.randperm(n, generator=self.gen, device="cuda")


def _ints(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def _pool(case, r, pages):
    """A pool of keys or values as a [pages, heads, page, d] view of its layout."""
    h, n, d = case["hkv"], case["page"], case["d"]
    if case["tokmajor"]:
        return r.normal((pages, n, h, d), case["dtype"]).transpose(1, 2)
    return r.normal((pages, h, n, d), case["dtype"])


def _tables(needs, pages):
    """Page tables: sequence i has needs[i] of `pages` (an order of the pool), then
    entries of -1. The pages that are left come back too."""
    need, width = _ints(needs).long(), max(1, max(needs))
    at = torch.arange(width, device="cuda")
    first = need.cumsum(0) - need
    own_page = pages[(first[:, None] + at).clamp(max=pages.numel() - 1)]
    table = torch.where(at < need[:, None], own_page, -1).int()
    return table, pages[sum(needs):]


def prepare(case, seed):
    r, s = _Rand(seed), dict(case)
    kind = case["kind"]
    if kind in ("logprob", "logprob_grad"):
        rows, vocab = case["rows"], case["vocab"]
        s["x"] = r.normal((rows, vocab), case["dtype"], 3.0)
        # sampled tokens; the last rows of a batch are padding
        s["tokens"] = r.ints(0, vocab, (rows,))
        s["tokens"][rows - rows // 16:] = -1
        if kind == "logprob":
            s["logprob"], s["lse"], s["entropy"] = (torch.empty(rows, device="cuda") for _ in range(3))
            s["top_logprob"] = torch.empty((rows, case["top"]), device="cuda")
            s["top_index"] = torch.empty((rows, case["top"]), device="cuda", dtype=torch.int32)
            return s
        logp = s["x"].double().log_softmax(1)
        s["lse"] = (s["x"][:, 0].double() - logp[:, 0]).float()
        s["entropy_in"] = -(logp.exp() * logp).sum(1).float()
        s["dlogprob"] = r.normal((rows,))
        if case["entropy"]:
            s["dentropy"] = r.normal((rows,), scale=0.1)
        s["dx"] = torch.empty_like(s["x"])
        return s

    b, hkv, d, page, dtype = case["b"], case["hkv"], case["d"], case["page"], case["dtype"]
    perm = r.order(b)
    if kind == "append":
        before = [case["ctx"]] * b
        after = [x + case["tokens"] for x in before]
        s["lengths"], s["counts"] = _ints(before), _ints(_counts(case))[perm]
        shape = (b, case["tokens"], hkv, d)      # as the projection gives them
        s["k_new"], s["v_new"] = (r.normal(shape, dtype).transpose(1, 2) for _ in range(2))
    else:
        s["lengths"] = _ints(_lengths(case))[perm]
        after = s["lengths"].tolist()
    needs = [-(-n // page) for n in after]
    more = 0
    if kind == "evict":
        more = b * -(-case["budget"] // page)
    pages = r.order(sum(needs) + more)
    if pages.numel() == 0:
        pages = r.order(1)
    s["k"], s["v"] = _pool(case, r, pages.numel()), _pool(case, r, pages.numel())
    s["table"], left = _tables(needs, pages)
    slots = s["table"].shape[1] * page
    if kind == "attend" and case["weights"] or kind == "evict":
        # what past steps gave the slots, and nothing behind the sequences' ends
        w = r.normal((b, hkv, slots), scale=1.5).exp_()
        w *= torch.arange(slots, device="cuda") < s["lengths"][:, None, None]
        s["w"] = w
    if kind == "attend":
        s["q"] = r.normal((b, case["hq"], 1, d), dtype, 2.0)
        s["o"] = torch.empty_like(s["q"])
    elif kind == "evict":
        s["new_table"] = left.reshape(b, -1).int()
        s["kept"] = torch.empty((b, hkv, case["budget"]), device="cuda", dtype=torch.int32)
        s["new_lengths"] = torch.empty_like(s["lengths"])
        s["new_w"] = torch.empty((b, hkv, s["new_table"].shape[1] * page), device="cuda")
    return s


# ---- the plain forms ---------------------------------------------------------

def _slot_places(table, slots, page):
    """(page, place in it) of each sequence's slots [b, t]."""
    at = torch.gather(table.long(), 1, (slots // page).clamp(max=table.shape[1] - 1))
    return at.clamp(min=0), slots % page


def _plain_append(s):
    t = torch.arange(s["tokens"], device="cuda")
    page, place = _slot_places(s["table"], s["lengths"].long()[:, None] + t, s["page"])
    new = (t < s["counts"][:, None])[:, :, None, None]
    for pool, rows in ((s["k"], s["k_new"]), (s["v"], s["v_new"])):
        old = pool[page, :, place]                       # [b, t, heads, d]
        pool[page, :, place] = torch.where(new, rows.transpose(1, 2), old)
    return [s["k"], s["v"]]


def _plain_attend(s):
    b, hq, hkv, d = s["b"], s["hq"], s["hkv"], s["d"]
    table = s["table"].long().clamp(min=0)
    width = table.shape[1] * s["page"]
    k = s["k"][table].float().transpose(1, 2).reshape(b, hkv, width, d)
    v = s["v"][table].float().transpose(1, 2).reshape(b, hkv, width, d)
    live = (torch.arange(width, device="cuda") < s["lengths"][:, None])[:, None, None, :]
    q = s["q"].float().reshape(b, hkv, hq // hkv, d)
    score = torch.matmul(q, k.transpose(2, 3)) * d ** -0.5
    score = score.masked_fill(~live, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = (score - top).exp()
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-38)
    v = v.masked_fill(~live.transpose(2, 3), 0.0)
    s["o"].copy_(torch.matmul(p, v).reshape(b, hq, 1, d))
    if not s["weights"]:
        return [s["o"]]
    s["w"].copy_(torch.where(live[:, 0], DECAY * s["w"] + p.sum(2), s["w"]))
    return [s["o"], s["w"]]


def _plain_evict(s):
    b, hkv, budget, page = s["b"], s["hkv"], s["budget"], s["page"]
    n = s["lengths"].long()[:, None, None]
    slot = torch.arange(s["w"].shape[2], device="cuda")
    rank = s["w"].masked_fill(slot >= n - s["recent"], math.inf).masked_fill(slot >= n, -math.inf)
    order = rank.sort(dim=2, descending=True, stable=True).indices
    order = torch.nn.functional.pad(order, (0, max(0, budget - order.shape[2])), value=slot.numel())[:, :, :budget]
    live = torch.arange(budget, device="cuda") < n.clamp(max=budget)
    kept = order.masked_fill(~live, slot.numel()).sort(dim=2).values
    inside = kept.clamp(max=slot.numel() - 1)
    head = torch.arange(hkv, device="cuda")[:, None]
    width = s["table"].shape[1]
    src = torch.gather(s["table"].long(), 1, (inside // page).reshape(b, -1).clamp(max=width - 1))
    src, place = src.reshape(b, hkv, budget).clamp(min=0), inside % page
    to = torch.arange(budget, device="cuda")
    dst = s["new_table"].long()[:, to // page][:, None].expand(b, hkv, budget)
    to = (to % page).expand(b, hkv, budget)
    for pool in (s["k"], s["v"]):
        pool[dst, head, to] = torch.where(live[..., None], pool[src, head, place], pool[dst, head, to])
    s["kept"].copy_(kept.masked_fill(~live, -1))
    s["new_lengths"].copy_(s["lengths"].clamp(max=budget))
    s["new_w"].zero_()
    s["new_w"][:, :, :budget] = torch.gather(s["w"], 2, inside) * live
    return [s["k"], s["v"], s["kept"], s["new_lengths"], s["new_w"]]


def _plain_logprob(s):
    x = s["x"].float()
    top = x.amax(1, keepdim=True)
    e = (x - top).exp()
    total = e.sum(1, keepdim=True)
    lse = top + total.log()
    entropy = total.log() - (e * (x - top)).sum(1, keepdim=True) / total
    token = s["tokens"].long()[:, None]
    logprob = (torch.gather(x, 1, token.clamp(min=0)) - lse) * (token >= 0)
    out = [logprob[:, 0], lse[:, 0], entropy[:, 0]]
    if s["top"]:
        # the values as they are, so that equal ones stay equal
        best = x.sort(dim=1, descending=True, stable=True)
        out += [best.values[:, :s["top"]] - lse, best.indices[:, :s["top"]].int()]
    return out


def _plain_logprob_grad(s):
    x, token = s["x"].float(), s["tokens"].long()[:, None]
    logp = x - s["lse"][:, None]
    p = logp.exp()
    g = s["dlogprob"][:, None] * (token >= 0)
    dx = -g * p
    dx.scatter_add_(1, token.clamp(min=0), g)
    if s["entropy"]:
        dx -= s["dentropy"][:, None] * p * (logp + s["entropy_in"][:, None])
    s["dx"].copy_(dx)
    return [s["dx"]]


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
                         torch.float32: grxcp_amd.GRX_R_32F, torch.int32: grxcp_amd.GRX_R_32I}
            cls.dnn.set_stream(torch.cuda.current_stream().cuda_stream)
        return cls

    @classmethod
    def room(cls, size):
        if size and (cls.workspace is None or cls.workspace.numel() < size):
            cls.workspace = torch.empty(size, device="cuda", dtype=torch.uint8)
        return cls.workspace.data_ptr() if size else None


DESCRIBED = ("x", "dx", "q", "o", "k", "v", "k_new", "v_new", "table", "new_table", "w", "new_w")


def _describe(s, L):
    """The descriptors of a state's shapes and the workspace they need: made once, as a
    program does for the buffers that it decodes or trains with."""
    d = {n: L.g.TensorDesc(L.types[s[n].dtype], list(s[n].shape), list(s[n].stride())) for n in DESCRIBED if n in s}
    d["size"] = 0
    if s["kind"] == "attend":
        d["attn"] = L.g.AttnDesc(True, s["d"] ** -0.5)
        d["size"] = L.dnn.paged_attention_workspace(d["q"], d["k"], d["table"], d.get("w"))
    elif s["kind"] == "logprob":
        d["size"] = L.dnn.token_logprob_workspace(d["x"], s["top"])
    return d


def _own(s):
    L = _Lib.get()
    kind, dnn, check = s["kind"], L.dnn, L.g.check
    d = s.get("descs")
    if d is None:
        d = s["descs"] = _describe(s, L)

    def p(name):
        return s[name].data_ptr()

    if kind == "append":
        check(dnn.paged_append(d["k_new"], p("k_new"), d["v_new"], p("v_new"), d["k"], p("k"), d["v"], p("v"),
                               d["table"], p("table"), p("lengths"), p("counts")))
        return [s["k"], s["v"]]
    if kind == "attend":
        w = s["weights"]
        check(dnn.paged_attention(d["attn"], d["q"], p("q"), d["k"], p("k"), d["v"], p("v"), d["table"], p("table"),
                                  p("lengths"), DECAY, d["w"] if w else None, p("w") if w else None, d["o"], p("o"),
                                  L.room(d["size"]), d["size"]))
        return [s["o"], s["w"]] if w else [s["o"]]
    if kind == "evict":
        check(dnn.paged_evict(d["k"], p("k"), d["v"], p("v"), d["table"], p("table"), p("lengths"), d["w"], p("w"),
                              s["budget"], s["recent"], p("kept"), d["new_table"], p("new_table"), p("new_lengths"),
                              d["new_w"], p("new_w")))
        return [s["k"], s["v"], s["kept"], s["new_lengths"], s["new_w"]]
    if kind == "logprob":
        top = s["top"]
        check(dnn.token_logprob(d["x"], p("x"), p("tokens"), p("logprob"), p("lse"), p("entropy"), top,
                                p("top_logprob") if top else None, p("top_index") if top else None,
                                L.room(d["size"]), d["size"]))
        return [s["logprob"], s["lse"], s["entropy"]] + ([s["top_logprob"], s["top_index"]] if top else [])
    check(dnn.token_logprob_backward(d["x"], p("x"), p("tokens"), p("lse"), p("entropy_in"), p("dlogprob"),
                                     p("dentropy") if s["entropy"] else None, d["dx"], p("dx")))
    return [s["dx"]]


def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict, "logprob": _plain_logprob,
            "logprob_grad": _plain_logprob_grad}[state["kind"]](state)


# ---- counting --------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind in ("logprob", "logprob_grad"):
        rows, n, size = case["rows"], case["rows"] * case["vocab"], SIZE[case["dtype"]]
        if kind == "logprob":
            # x once; the tokens, three statistics and the alternatives
            return {"bytes": n * size + rows * (16 + 8 * case["top"]), "flops": 6.0 * n}
        return {"bytes": 2 * n * size + rows * (12 + (8 if case["entropy"] else 0)),
                "flops": (6.0 if case["entropy"] else 4.0) * n}
    row = 2 * case["hkv"] * case["d"] * 2                # a token's key and value
    if kind == "append":
        t = sum(_counts(case))
        return {"bytes": 2 * row * t + 8 * case["b"], "flops": 0.0}
    lengths = _lengths(case)
    pages = sum(-(-n // case["page"]) for n in lengths)
    if kind == "attend":
        t = sum(lengths)
        extra = 8 * case["hkv"] * t if case["weights"] else 0
        return {"bytes": row * t + 4 * case["b"] * case["hq"] * case["d"] + 4 * pages + extra,
                "flops": 4.0 * case["hq"] * case["d"] * t}
    kept = sum(min(n, case["budget"]) for n in lengths)
    # the weights; the rows that stay, read and written; their slots and new weights
    return {"bytes": 4 * case["hkv"] * sum(lengths) + 2 * row * kept + 8 * case["hkv"] * kept + 4 * pages,
            "flops": float(case["hkv"] * sum(lengths))}


# ---- in 64 bits ----------------------------------------------------------------

def _rows_of(pool, table, n, page):
    """Rows 0 .. n-1 of one sequence, [heads, n, d] in 64 bits."""
    pages = table[: -(-n // page)].long()
    return torch.cat(list(pool[pages]), dim=1)[:, :n].double() if n else pool.new_zeros(
        (pool.shape[1], 0, pool.shape[3]), dtype=torch.float64)


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "append":
        pools = []
        for pool, rows in ((s["k"], s["k_new"]), (s["v"], s["v_new"])):
            pool = pool.double()
            for i, (n, c) in enumerate(zip(s["lengths"].tolist(), s["counts"].tolist())):
                slots = torch.arange(n, n + c, device="cuda")
                if c:
                    pool[s["table"][i, slots // case["page"]].long(), :, slots % case["page"]] = \
                        rows[i, :, :c].transpose(0, 1).double()
            pools.append(pool)
        return pools
    if kind == "attend":
        o = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
        w = s["w"].double() if case["weights"] else None
        group = case["hq"] // case["hkv"]
        for i, n in enumerate(s["lengths"].tolist()):
            if not n:
                continue
            k, v = (_rows_of(s[x], s["table"][i], n, case["page"]) for x in "kv")
            for h in range(case["hkv"]):
                q = s["q"][i, h * group:(h + 1) * group, 0].double()
                p = torch.softmax(torch.mm(k[h], q.T).T / math.sqrt(case["d"]), dim=1)
                o[i, h * group:(h + 1) * group, 0] = torch.mm(p, v[h])
                if w is not None:
                    w[i, h, :n] = DECAY * w[i, h, :n] + p.sum(0)
        return [o] if w is None else [o, w]
    if kind == "evict":
        pools, page = [s["k"].double(), s["v"].double()], case["page"]
        kept = torch.full(s["kept"].shape, -1, device="cuda", dtype=torch.int32)
        new_w = torch.zeros(s["new_w"].shape, device="cuda", dtype=torch.float64)
        lengths = s["lengths"].tolist()
        for i, n in enumerate(lengths):
            m = min(n, case["budget"])
            old = max(0, n - case["recent"])
            rows = [_rows_of(pool, s["table"][i], n, page) for pool in pools]
            for h in range(case["hkv"]):
                best = torch.argsort(-s["w"][i, h, :old].double(), stable=True)[: m - (n - old)]
                stay = torch.zeros(n, dtype=torch.bool, device="cuda")
                stay[best] = True
                stay[old:] = True
                stay = stay.nonzero()[:, 0]
                to = torch.arange(m, device="cuda")
                for pool, row in zip(pools, rows):
                    pool[s["new_table"][i, to // page].long(), h, to % page] = row[h, stay]
                kept[i, h, :m] = stay.int()
                new_w[i, h, :m] = s["w"][i, h, stay].double()
        return pools + [kept, _ints([min(n, case["budget"]) for n in lengths]), new_w]
    x, token = s["x"].double(), s["tokens"].long()
    rows = torch.arange(case["rows"], device="cuda")
    if kind == "logprob":
        lse = torch.logsumexp(x, 1)
        logp = x - lse[:, None]
        entropy = -(logp.exp() * logp).sum(1)
        logprob = torch.where(token >= 0, logp[rows, token.clamp(min=0)], 0.0)
        out = [logprob, lse, entropy]
        if case["top"]:
            index = torch.argsort(-x, dim=1, stable=True)[:, :case["top"]]
            out += [logp.gather(1, index), index.int()]
        return out
    p = torch.exp(x - s["lse"].double()[:, None])
    logp = x - s["lse"].double()[:, None]
    one = torch.zeros_like(p)
    one[rows, token.clamp(min=0)] = 1.0
    dx = (one - p) * torch.where(token >= 0, s["dlogprob"].double(), 0.0)[:, None]
    if case["entropy"]:
        dx -= s["dentropy"].double()[:, None] * p * (logp + s["entropy_in"].double()[:, None])
    return [dx]
