"""The paged cache's and the log probabilities' entry points without a GPU: index
arithmetic, argument checks and workspace sizes."""
import ctypes
import os
import subprocess

import pytest

import grxcp_amd as g
from grxcp_amd import build as B

HERE = os.path.dirname(os.path.abspath(__file__))
BF16, F16, F32, I32, I8 = g.GRX_R_16BF, g.GRX_R_16F, g.GRX_R_32F, g.GRX_R_32I, g.GRX_R_8I
INVALID, UNSUPPORTED = g.INVALID_VALUE, g.NOT_SUPPORTED


def test_index_arithmetic(tmp_path):
    exe = tmp_path / "paged_index"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror",
                    "-fsanitize=undefined,address", "-fno-sanitize-recover", os.path.join(HERE, "paged_index_main.cpp"),
                    "-I", B.CSRC, "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.stdout.strip() == "ok", r.stdout + r.stderr


@pytest.fixture(scope="module")
def dnn():
    d = g.Dnn()
    yield d
    d.close()


def at(i):
    """An address that no call below follows: 1 GiB apart."""
    return 0x100000000 + (i << 30)


# What a call that passes every check returns: no device here, or nothing to check
# on a machine that has one (the addresses are not real).
needs_no_gpu = pytest.mark.skipif(g.device_count() > 0, reason="checks the no-device path")
OK = g.ARCH_MISMATCH
T = g.TensorDesc
POOL = [40, 4, 16, 64]          # pages, heads, page, d
TABLE = [3, 8]


def append(dnn, **kw):
    a = dict(kd=T(BF16, [3, 4, 5, 64]), k=at(1), vd=T(BF16, [3, 4, 5, 64]), v=at(2), kcd=T(BF16, POOL), kc=at(3),
             vcd=T(BF16, POOL), vc=at(4), td=T(I32, TABLE), table=at(5), lengths=at(6), counts=at(7))
    assert set(kw) <= set(a)
    a.update(kw)
    return dnn.paged_append(*a.values())


def attend(dnn, size=1 << 20, **kw):
    a = dict(ad=g.AttnDesc(True, 0.125), qd=T(BF16, [3, 8, 1, 64]), q=at(1), kcd=T(BF16, POOL), kc=at(3),
             vcd=T(BF16, POOL), vc=at(4), td=T(I32, TABLE), table=at(5), lengths=at(6), decay=1.0,
             wd=T(F32, [3, 4, 128]), w=at(7), od=T(BF16, [3, 8, 1, 64]), o=at(2), ws=at(8))
    assert set(kw) <= set(a)
    a.update(kw)
    return dnn.paged_attention(*a.values(), size)


def evict(dnn, **kw):
    a = dict(kcd=T(BF16, POOL), kc=at(3), vcd=T(BF16, POOL), vc=at(4), td=T(I32, TABLE), table=at(5),
             lengths=at(6), wd=T(F32, [3, 4, 128]), w=at(7), budget=30, recent=4, kept=at(8), ntd=T(I32, [3, 2]),
             new_table=at(9), new_lengths=at(10), nwd=T(F32, [3, 4, 30]), new_w=at(11))
    assert set(kw) <= set(a)
    a.update(kw)
    return dnn.paged_evict(*a.values())


def logprob(dnn, size=1 << 20, **kw):
    a = dict(xd=T(BF16, [6, 1000]), x=at(1), tokens=at(2), logprob=at(3), lse=at(4), entropy=at(5), top=3,
             top_logprob=at(6), top_index=at(7), ws=at(8))
    assert set(kw) <= set(a)
    a.update(kw)
    return dnn.token_logprob(*a.values(), size)


def gradient(dnn, **kw):
    a = dict(xd=T(BF16, [6, 1000]), x=at(1), tokens=at(2), lse=at(4), entropy=at(5), dlogprob=at(6), dentropy=at(7),
             dxd=T(BF16, [6, 1000]), dx=at(8))
    assert set(kw) <= set(a)
    a.update(kw)
    return dnn.token_logprob_backward(*a.values())


class Unset:
    """A descriptor that was created and never set."""

    def __init__(self):
        self.L, self.d = g.load().dnn, ctypes.c_void_p()
        g.check(self.L.grxdnnCreateTensorDescriptor(ctypes.byref(self.d)))

    def __del__(self):
        self.L.grxdnnDestroyTensorDescriptor(self.d)


class Null:
    d = None


@needs_no_gpu
def test_valid_calls_reach_the_device_check(dnn):
    assert append(dnn) == OK and append(dnn, counts=None) == OK
    assert attend(dnn) == OK and attend(dnn, wd=None, w=None) == OK
    assert evict(dnn) == OK
    assert logprob(dnn) == OK
    assert logprob(dnn, tokens=None, logprob=None, entropy=None, top=0, top_logprob=None, top_index=None) == OK
    assert gradient(dnn) == OK
    assert gradient(dnn, entropy=None, dentropy=None) == OK and gradient(dnn, dentropy=None) == OK
    assert gradient(dnn, tokens=None, dlogprob=None) == OK
    # [pages, page, heads, d] memory, q and o as rows of a packed projection, o over q
    tok = T(BF16, POOL, [4096, 64, 256, 1])
    assert append(dnn, kcd=tok, vcd=tok) == OK
    # the two pools as halves of one array
    both = T(BF16, POOL, [8192, 64, 512, 1])
    assert append(dnn, kcd=both, vcd=both, vc=at(3) + 512) == OK
    row = T(BF16, [3, 8, 1, 64], [1536, 64, 1536, 1])
    assert attend(dnn, qd=row, od=row) == OK and attend(dnn, qd=row, od=row, o=at(1)) == OK
    assert attend(dnn, ad=g.AttnDesc(False, 0.125)) == OK
    # one group of many heads, lengths in place, one table row for all, dx over x
    assert attend(dnn, qd=T(BF16, [3, 4096, 1, 64]), od=T(BF16, [3, 4096, 1, 64]), size=1 << 40) == OK
    assert evict(dnn, new_lengths=at(6)) == OK
    assert attend(dnn, td=T(I32, TABLE, [0, 1])) == OK
    assert gradient(dnn, dx=at(1)) == OK
    assert logprob(dnn, xd=T(F32, [2, 3, 1000], [3300, 1100, 1])) == OK


def test_null_handle():
    class H:
        L, h = g.load().dnn, None
    for call in (append, attend, evict, logprob, gradient):
        d = g.Dnn()
        h, d.h = d.h, None
        assert call(d) == g.NOT_INITIALIZED
        d.h = h
        d.close()
    n = ctypes.c_size_t()
    assert H.L.grxdnnPagedAttentionGetWorkspaceSize(None, None, None, None, None, ctypes.byref(n)) == g.NOT_INITIALIZED
    assert H.L.grxdnnTokenLogProbGetWorkspaceSize(None, None, 0, ctypes.byref(n)) == g.NOT_INITIALIZED


@pytest.mark.parametrize("call,names", [
    (append, ["kd", "vd", "kcd", "vcd", "td"]), (attend, ["qd", "kcd", "vcd", "td", "od", "wd"]),
    (evict, ["kcd", "vcd", "td", "wd", "ntd", "nwd"]), (logprob, ["xd"]), (gradient, ["xd", "dxd"])])
def test_missing_and_unset_descriptors(dnn, call, names):
    for n in names:
        assert call(dnn, **{n: Unset()}) == INVALID, n
        assert call(dnn, **{n: Null()}) == INVALID, n


@pytest.mark.parametrize("call,names", [
    (append, ["k", "v", "kc", "vc", "table", "lengths"]),
    (attend, ["q", "kc", "vc", "table", "lengths", "o", "w"]),
    (evict, ["kc", "vc", "table", "lengths", "w", "kept", "new_table", "new_lengths", "new_w"]),
    (logprob, ["x", "tokens", "logprob", "lse", "top_logprob", "top_index"]),
    (gradient, ["x", "tokens", "lse", "entropy", "dlogprob", "dx"])])
def test_null_pointers(dnn, call, names):
    for n in names:
        assert call(dnn, **{n: None}) == INVALID, n


def test_shapes_that_do_not_belong_together(dnn):
    assert append(dnn, kd=T(BF16, [2, 4, 5, 64]), vd=T(BF16, [2, 4, 5, 64])) == INVALID
    assert append(dnn, kd=T(BF16, [3, 3, 5, 64]), vd=T(BF16, [3, 3, 5, 64])) == INVALID
    assert append(dnn, kd=T(BF16, [3, 4, 5, 128]), vd=T(BF16, [3, 4, 5, 128])) == INVALID
    assert append(dnn, vd=T(BF16, [3, 4, 6, 64])) == INVALID
    assert append(dnn, kd=T(BF16, [3, 20, 64]), vd=T(BF16, [3, 20, 64])) == INVALID
    for call in (append, attend, evict):
        assert call(dnn, vcd=T(BF16, [41, 4, 16, 64])) == INVALID
        assert call(dnn, kcd=T(BF16, [640, 4, 64]), vcd=T(BF16, [640, 4, 64])) == INVALID
        assert call(dnn, kcd=T(BF16, [0, 4, 16, 64]), vcd=T(BF16, [0, 4, 16, 64])) == INVALID
        assert call(dnn, td=T(I32, [3, 8, 1])) == INVALID
        assert call(dnn, td=T(F32, TABLE)) == INVALID
        assert call(dnn, td=T(I32, [3, 0])) == INVALID
        assert call(dnn, td=T(I32, TABLE, [16, 2])) == INVALID
        assert call(dnn, td=T(I32, [2, 8])) == INVALID
    assert attend(dnn, qd=T(BF16, [3, 6, 1, 64]), od=T(BF16, [3, 6, 1, 64])) == INVALID
    assert attend(dnn, qd=T(BF16, [3, 0, 1, 64]), od=T(BF16, [3, 0, 1, 64])) == INVALID
    assert attend(dnn, od=T(BF16, [3, 4, 1, 64])) == INVALID
    assert attend(dnn, wd=T(F32, [3, 4, 127])) == INVALID
    assert attend(dnn, wd=T(F32, [3, 8, 128])) == INVALID
    assert attend(dnn, wd=T(BF16, [3, 4, 128])) == INVALID
    assert attend(dnn, wd=T(F32, [3, 4, 128], [1024, 256, 2])) == INVALID
    assert attend(dnn, wd=T(F32, [3, 4, 128], [256, 64, 1])) == INVALID
    assert attend(dnn, wd=None) == INVALID
    assert evict(dnn, ntd=T(I32, [3, 1])) == INVALID             # 16 slots for a budget of 30
    assert evict(dnn, ntd=T(I32, [2, 2])) == INVALID
    assert evict(dnn, nwd=T(F32, [3, 4, 29])) == INVALID
    assert evict(dnn, nwd=T(F32, [3, 4, 30], [30, 0, 1])) == INVALID
    assert evict(dnn, wd=T(F32, [3, 4, 120])) == INVALID
    assert gradient(dnn, dxd=T(BF16, [6, 999])) == INVALID
    assert gradient(dnn, dxd=T(BF16, [6, 1000], [500, 1])) in (INVALID, UNSUPPORTED)


def test_scalars(dnn):
    for budget, recent in ((0, 0), (-1, 0), (30, -1), (30, 31)):
        assert evict(dnn, budget=budget, recent=recent) == INVALID
    for decay in (-0.5, float("nan"), float("inf")):
        assert attend(dnn, decay=decay) == INVALID
    assert logprob(dnn, top=-1) == INVALID
    assert logprob(dnn, xd=T(BF16, [6, 2]), top=3) == INVALID
    assert logprob(dnn, top=65) == UNSUPPORTED
    assert logprob(dnn, top=0) == INVALID                        # the arrays have to be NULL


def test_types_and_layouts_that_are_not_served(dnn):
    for call in (append, attend, evict):
        for t in (F32, I8):
            assert call(dnn, kcd=T(t, POOL), vcd=T(t, POOL)) == UNSUPPORTED
        assert call(dnn, vcd=T(F16, POOL)) == UNSUPPORTED
        for strides in ([4096, 1024, 64, 2], [4100, 1024, 64, 1], [4608, 1152, 68, 1]):
            assert call(dnn, kcd=T(BF16, POOL, strides), vcd=T(BF16, POOL, strides)) == UNSUPPORTED
        assert call(dnn, kc=at(3) + 8) == UNSUPPORTED
        assert call(dnn, vc=at(4) + 2) == UNSUPPORTED
        assert call(dnn, td=T(I32, [3, 1 << 27])) != OK          # 2^31 slots
    assert append(dnn, kd=T(F16, [3, 4, 5, 64]), vd=T(F16, [3, 4, 5, 64])) == UNSUPPORTED
    assert append(dnn, k=at(1) + 2) == UNSUPPORTED
    assert attend(dnn, qd=T(F16, [3, 8, 1, 64])) == UNSUPPORTED
    assert attend(dnn, qd=T(BF16, [3, 8, 2, 64]), od=T(BF16, [3, 8, 2, 64])) == UNSUPPORTED
    assert attend(dnn, qd=T(BF16, [3, 4100, 1, 64]), od=T(BF16, [3, 4100, 1, 64]), size=1 << 40) == UNSUPPORTED
    assert attend(dnn, q=at(1) + 4) == UNSUPPORTED and attend(dnn, ws=at(8) + 4) == UNSUPPORTED
    d96 = T(BF16, [40, 4, 16, 96])
    assert attend(dnn, kcd=d96, vcd=d96, qd=T(BF16, [3, 8, 1, 96]), od=T(BF16, [3, 8, 1, 96])) == UNSUPPORTED
    for call, n in ((logprob, "xd"), (gradient, "xd")):
        more = {"dxd": T(I8, [6, 1000])} if call is gradient else {}
        assert call(dnn, **{n: T(I8, [6, 1000])}, **more) == UNSUPPORTED
        more = {"dxd": T(F32, [6, 1000], [2000, 2])} if call is gradient else {}
        assert call(dnn, **{n: T(F32, [6, 1000], [2000, 2])}, **more) == UNSUPPORTED
        more = {"dxd": T(F32, [2, 3, 1000], [5000, 1100, 1])} if call is gradient else {}
        assert call(dnn, **{n: T(F32, [2, 3, 1000], [5000, 1100, 1])}, **more) == UNSUPPORTED
    big = T(BF16, [1, (1 << 24) + 1])
    assert logprob(dnn, xd=big) == UNSUPPORTED and gradient(dnn, xd=big, dxd=big) == UNSUPPORTED
    assert gradient(dnn, dxd=T(F32, [6, 1000])) == UNSUPPORTED


def test_empty_calls_succeed_without_a_device(dnn):
    none = T(I32, [0, 8])
    assert append(dnn, kd=T(BF16, [0, 4, 5, 64]), vd=T(BF16, [0, 4, 5, 64]), td=none, k=None) == g.SUCCESS
    assert append(dnn, kd=T(BF16, [3, 4, 0, 64]), vd=T(BF16, [3, 4, 0, 64]), k=None, v=None) == g.SUCCESS
    assert attend(dnn, qd=T(BF16, [0, 8, 1, 64]), od=T(BF16, [0, 8, 1, 64]), td=none, wd=T(F32, [0, 4, 128]),
                  q=None) == g.SUCCESS
    assert evict(dnn, td=none, ntd=T(I32, [0, 2]), wd=T(F32, [0, 4, 128]), nwd=T(F32, [0, 4, 30])) == g.SUCCESS
    assert logprob(dnn, xd=T(BF16, [0, 1000]), x=None) == g.SUCCESS
    assert gradient(dnn, xd=T(BF16, [0, 1000]), dxd=T(BF16, [0, 1000]), x=None) == g.SUCCESS


def test_overlaps_are_refused(dnn):
    page = 2 * 4 * 16 * 64
    for call in (append, evict):
        assert call(dnn, vc=at(3)) == INVALID                     # one pool for both
        assert call(dnn, vc=at(3) + 39 * page) == INVALID
        same = T(BF16, POOL, [0, 1024, 64, 1])
        assert call(dnn, kcd=same, vcd=same) == INVALID           # pages that share addresses
    assert append(dnn, k=at(3)) == INVALID and append(dnn, v=at(4) + page) == INVALID
    assert append(dnn, table=at(3)) == INVALID and append(dnn, lengths=at(4)) == INVALID
    assert append(dnn, counts=at(4)) == INVALID
    assert attend(dnn, o=at(3)) == INVALID and attend(dnn, o=at(4) + page) == INVALID
    assert attend(dnn, o=at(1) + 128) == INVALID                  # over other rows of q
    assert attend(dnn, o=at(5)) == INVALID and attend(dnn, o=at(7)) == INVALID
    assert attend(dnn, w=at(1)) == INVALID and attend(dnn, w=at(3)) == INVALID and attend(dnn, w=at(6)) == INVALID
    for p in (1, 2, 3, 4, 5, 6, 7):
        assert attend(dnn, ws=at(p)) == INVALID, p
    shared = T(BF16, [3, 8, 1, 64], [0, 64, 64, 1])
    assert attend(dnn, od=shared) == INVALID
    for n in ("kept", "new_lengths", "new_w"):
        for p in (3, 4, 5, 6, 7, 9):
            if (n, p) != ("new_lengths", 6):
                assert evict(dnn, **{n: at(p)}) == INVALID, (n, p)
    assert evict(dnn, new_lengths=at(6) + 4) == INVALID
    assert evict(dnn, kept=at(10)) == INVALID and evict(dnn, kept=at(11)) == INVALID
    for n in ("logprob", "lse", "entropy", "top_logprob", "top_index"):
        for p in (1, 2):
            assert logprob(dnn, **{n: at(p)}) == INVALID, (n, p)
    assert logprob(dnn, lse=at(3)) == INVALID and logprob(dnn, top_index=at(6) + 8) == INVALID
    assert gradient(dnn, dx=at(1) + 2000) == INVALID
    for p in (2, 4, 5, 6, 7):
        assert gradient(dnn, dx=at(p)) == INVALID, p
    assert gradient(dnn, xd=T(BF16, [6, 1000], [1100, 1]), dx=at(1)) == INVALID


def test_optional_pairs(dnn):
    assert gradient(dnn, tokens=None) == INVALID and gradient(dnn, dlogprob=None) == INVALID
    assert gradient(dnn, entropy=None) == INVALID
    assert gradient(dnn, tokens=None, dlogprob=None, entropy=None, dentropy=None) == INVALID
    assert gradient(dnn, tokens=None, dlogprob=None, dentropy=None) == INVALID
    assert logprob(dnn, tokens=None) == INVALID and logprob(dnn, logprob=None) == INVALID


def test_workspace_sizes(dnn):
    q, pool, table = T(BF16, [3, 8, 1, 64]), T(BF16, POOL), T(I32, TABLE)
    w = T(F32, [3, 4, 128])
    plain, weighted = dnn.paged_attention_workspace(q, pool, table), dnn.paged_attention_workspace(q, pool, table, w)
    assert weighted >= plain + 4 * 3 * 8 * 128
    assert attend(dnn, size=weighted - 1) == INVALID
    if plain:
        assert attend(dnn, wd=None, w=None, size=plain - 1) == INVALID
        assert attend(dnn, wd=None, w=None, ws=None) == INVALID
    assert attend(dnn, ws=None) == INVALID
    n = dnn.token_logprob_workspace(T(BF16, [6, 100000]), 3)
    if n:
        assert logprob(dnn, xd=T(BF16, [6, 100000]), size=n - 1) == INVALID
        assert logprob(dnn, xd=T(BF16, [6, 100000]), ws=None) == INVALID
    L, out = g.load().dnn, ctypes.c_size_t()
    ask = L.grxdnnPagedAttentionGetWorkspaceSize
    assert ask(dnn.h, q.d, pool.d, table.d, None, None) == INVALID
    assert ask(dnn.h, None, pool.d, table.d, None, ctypes.byref(out)) == INVALID
    assert ask(dnn.h, T(BF16, [3, 6, 1, 64]).d, pool.d, table.d, None, ctypes.byref(out)) == INVALID
    assert L.grxdnnTokenLogProbGetWorkspaceSize(dnn.h, T(BF16, [6, 2]).d, 3, ctypes.byref(out)) == INVALID
    assert L.grxdnnTokenLogProbGetWorkspaceSize(dnn.h, None, 0, ctypes.byref(out)) == INVALID


@needs_no_gpu
def test_strides_of_a_dimension_of_one_do_not_matter(dnn):
    """[B, 1, V] views of the last tokens' logits, of rows first and of transposed ones: the
    pitch is the batch's, whatever the dimension of one has for a stride."""
    for strides in ([7000, 1000, 1], [7000, 5, 1], [1000, 6000, 1], [1000, 0, 1]):
        x = T(BF16, [6, 1, 1000], strides)
        assert logprob(dnn, xd=x) == OK and gradient(dnn, xd=x, dxd=x) == OK, strides
    assert logprob(dnn, xd=T(BF16, [6, 1, 1000], [500, 1000, 1])) == UNSUPPORTED       # rows that overlap
    assert logprob(dnn, xd=T(BF16, [2, 1, 3, 1000], [5000, 9, 1100, 1])) == UNSUPPORTED
    assert logprob(dnn, xd=T(BF16, [2, 1, 3, 1000], [3300, 9, 1100, 1])) == OK


@needs_no_gpu
def test_more_joining_workgroups_than_one_launch_takes(dnn):
    """Refused before anything is launched: 17 heads of 2^30 slots have 2^24 + 2^20 chunks of
    1024 weights. As many slots without weights, or fewer heads, pass."""
    far = dict(kcd=T(BF16, [40, 17, 16, 64]), vcd=T(BF16, [40, 17, 16, 64]), td=T(I32, [1, 1 << 26]),
               qd=T(BF16, [1, 17, 1, 64]), od=T(BF16, [1, 17, 1, 64]), table=1 << 43, ws=1 << 45, size=1 << 44)
    w = dict(wd=T(F32, [1, 17, 1 << 30], [0, 1 << 30, 1]), w=1 << 44)
    assert attend(dnn, **far, **w) == UNSUPPORTED
    assert attend(dnn, **far, wd=None, w=None) == OK
    few = dict(far, kcd=T(BF16, [40, 15, 16, 64]), vcd=T(BF16, [40, 15, 16, 64]), qd=T(BF16, [1, 15, 1, 64]),
               od=T(BF16, [1, 15, 1, 64]))
    assert attend(dnn, **few, wd=T(F32, [1, 15, 1 << 30], [0, 1 << 30, 1]), w=1 << 44) == OK
