"""The 8-bit paged cache's entry points without a GPU: argument checks."""
import ctypes

import pytest

import grxcp_amd as g
from test_paged_host import Null, Unset, at

BF16, F16, F32, I32, I8 = g.GRX_R_16BF, g.GRX_R_16F, g.GRX_R_32F, g.GRX_R_32I, g.GRX_R_8I
INVALID, UNSUPPORTED = g.INVALID_VALUE, g.NOT_SUPPORTED
needs_no_gpu = pytest.mark.skipif(g.device_count() > 0, reason="checks the no-device path")
OK = g.ARCH_MISMATCH
T = g.TensorDesc
POOL, TABLE, SCALES = [40, 4, 16, 64], [3, 8], [40, 4, 2]


@pytest.fixture(scope="module")
def dnn():
    d = g.Dnn()
    yield d
    d.close()


def cache():
    return dict(kcd=T(I8, POOL), kc=at(3), vcd=T(I8, POOL), vc=at(4), sd=T(F32, SCALES), ks=at(5), vs=at(6),
                td=T(I32, TABLE), table=at(7), lengths=at(8))


def append(dnn, **kw):
    a = dict(kd=T(BF16, [3, 4, 5, 64]), k=at(1), vd=T(BF16, [3, 4, 5, 64]), v=at(2), **cache(), counts=at(9))
    assert set(kw) <= set(a)
    a.update(kw)
    return dnn.paged_append_quantized(*a.values())


def read(dnn, **kw):
    a = dict(**cache(), first=at(9), kd=T(BF16, [3, 4, 5, 64]), k=at(1), vd=T(BF16, [3, 4, 5, 64]), v=at(2))
    assert set(kw) <= set(a)
    a.update(kw)
    return dnn.paged_read_quantized(*a.values())


def attend(dnn, size=1 << 24, **kw):
    a = dict(ad=g.AttnDesc(True, 0.125), qd=T(BF16, [3, 8, 1, 64]), q=at(1), **cache(), od=T(BF16, [3, 8, 1, 64]),
             o=at(2), ws=at(10))
    assert set(kw) <= set(a)
    a.update(kw)
    return dnn.paged_attention_quantized(*a.values(), size)


BOTH = (append, read)


@needs_no_gpu
def test_valid_calls_reach_the_device_check(dnn):
    assert append(dnn) == OK and append(dnn, counts=None) == OK
    assert read(dnn) == OK and read(dnn, first=None) == OK
    f32 = T(F32, [3, 4, 5, 64])
    assert read(dnn, kd=f32, vd=f32) == OK
    for call in BOTH:
        tok = T(I8, POOL, [4096, 64, 256, 1])                # [pages, page, heads, d] memory
        assert call(dnn, kcd=tok, vcd=tok) == OK
        both = T(I8, POOL, [8192, 64, 512, 1])               # the two pools as halves of one array
        assert call(dnn, kcd=both, vcd=both, vc=at(3) + 256) == OK
        for n in (1, 4, 16):
            assert call(dnn, sd=T(F32, [40, 4, n])) == OK
        pair = T(F32, SCALES, [16, 2, 1])                    # two scale arrays side by side
        assert call(dnn, sd=pair, vs=at(5) + 32) == OK
        assert call(dnn, td=T(I32, TABLE, [0, 1])) == OK
        row = T(BF16, [3, 4, 5, 64], [12 * 320, 64, 768, 1])  # a packed projection
        assert call(dnn, kd=row, vd=row, v=at(1) + 512) == OK
    # one pool's rows read into one array, and read twice
    assert read(dnn, vcd=T(I8, POOL), vc=at(3)) == OK


def test_null_handle_descriptors_and_pointers(dnn):
    for call in BOTH:
        d = g.Dnn()
        h, d.h = d.h, None
        assert call(d) == g.NOT_INITIALIZED
        d.h = h
        d.close()
        for n in ("kd", "vd", "kcd", "vcd", "sd", "td"):
            assert call(dnn, **{n: Unset()}) == INVALID, n
            assert call(dnn, **{n: Null()}) == INVALID, n
        for n in ("k", "v", "kc", "vc", "ks", "vs", "table", "lengths"):
            assert call(dnn, **{n: None}) == INVALID, n


def test_shapes_and_types(dnn):
    for call in BOTH:
        assert call(dnn, kd=T(BF16, [2, 4, 5, 64]), vd=T(BF16, [2, 4, 5, 64])) == INVALID
        assert call(dnn, kd=T(BF16, [3, 3, 5, 64]), vd=T(BF16, [3, 3, 5, 64])) == INVALID
        assert call(dnn, kd=T(BF16, [3, 4, 5, 128]), vd=T(BF16, [3, 4, 5, 128])) == INVALID
        assert call(dnn, vd=T(BF16, [3, 4, 6, 64])) == INVALID
        assert call(dnn, kd=T(BF16, [3, 20, 64]), vd=T(BF16, [3, 20, 64])) == INVALID
        assert call(dnn, vcd=T(I8, [41, 4, 16, 64])) == INVALID
        assert call(dnn, kcd=T(I8, [0, 4, 16, 64]), vcd=T(I8, [0, 4, 16, 64])) == INVALID
        assert call(dnn, td=T(F32, TABLE)) == INVALID and call(dnn, td=T(I32, [2, 8])) == INVALID
        for s in ([41, 4, 2], [40, 3, 2], [40, 4, 0], [40, 4, 3], [40, 4, 32], [40, 8]):
            assert call(dnn, sd=T(F32, s)) == INVALID, s
        assert call(dnn, sd=T(BF16, SCALES)) == UNSUPPORTED
        for t in (BF16, F32, I32):
            assert call(dnn, kcd=T(t, POOL), vcd=T(t, POOL)) == UNSUPPORTED
        assert call(dnn, vcd=T(BF16, POOL)) == UNSUPPORTED
        assert call(dnn, vd=T(F16, [3, 4, 5, 64])) == UNSUPPORTED
        assert call(dnn, kd=T(I8, [3, 4, 5, 64]), vd=T(I8, [3, 4, 5, 64])) == UNSUPPORTED
        for strides in ([4096, 1024, 64, 2], [4104, 1024, 64, 1], [4608, 1152, 72, 1]):
            assert call(dnn, kcd=T(I8, POOL, strides), vcd=T(I8, POOL, strides)) == UNSUPPORTED
        for n in ("k", "v", "kc", "vc"):
            assert call(dnn, **{n: at(20) + 8}) == UNSUPPORTED, n
        wide = T(I8, [40, 4, 512, 64])                       # blocks of 512 slots
        assert call(dnn, kcd=wide, vcd=wide, sd=T(F32, [40, 4, 1])) == UNSUPPORTED
        d96 = T(I8, [40, 4, 16, 96])
        assert call(dnn, kcd=d96, vcd=d96, kd=T(BF16, [3, 4, 5, 96]), vd=T(BF16, [3, 4, 5, 96])) == UNSUPPORTED
        assert call(dnn, td=T(I32, [3, 1 << 27])) == UNSUPPORTED   # 2^31 slots
        many = T(BF16, [3, 4, 1 << 29, 64], [0, 0, 64, 1])
        assert call(dnn, kd=many, vd=many) == UNSUPPORTED
    assert append(dnn, kd=T(F32, [3, 4, 5, 64]), vd=T(F32, [3, 4, 5, 64])) == UNSUPPORTED
    shared = T(BF16, [3, 4, 5, 64], [0, 320, 64, 1])
    assert read(dnn, kd=shared) == INVALID                   # rows that share addresses


def test_empty_calls_succeed_without_a_device(dnn):
    for call in BOTH:
        none = T(BF16, [0, 4, 5, 64])
        assert call(dnn, kd=none, vd=none, td=T(I32, [0, 8]), k=None) == g.SUCCESS
        none = T(BF16, [3, 4, 0, 64])
        assert call(dnn, kd=none, vd=none, k=None, v=None) == g.SUCCESS


def test_overlaps_are_refused(dnn):
    page, scales = 4 * 16 * 64, 40 * 4 * 2 * 4
    assert append(dnn, vc=at(3)) == INVALID and append(dnn, vc=at(3) + 39 * page) == INVALID
    assert append(dnn, vs=at(5)) == INVALID and append(dnn, vs=at(5) + scales - 4) == INVALID
    same = T(I8, POOL, [0, 1024, 64, 1])
    assert append(dnn, kcd=same, vcd=same) == INVALID        # pages that share addresses
    assert append(dnn, sd=T(F32, SCALES, [8, 2, 0])) == INVALID
    for n in ("kc", "vc", "ks", "vs"):
        for p in (1, 2, 3, 4, 5, 6, 7, 8, 9):
            if at(p) != cache()[n]:
                assert append(dnn, **{n: at(p)}) == INVALID, (n, p)
    for n in ("k", "v"):
        for p in (1, 2, 3, 4, 5, 6, 7, 8, 9):
            if (n, p) not in (("k", 1), ("v", 2)):
                assert read(dnn, **{n: at(p)}) == INVALID, (n, p)


# ---- attention -----------------------------------------------------------------

@needs_no_gpu
def test_valid_attention_calls_reach_the_device_check(dnn):
    assert attend(dnn) == OK and attend(dnn, ad=g.AttnDesc(False, 0.125)) == OK
    half = T(F16, [3, 8, 1, 64])
    assert attend(dnn, qd=half, od=half) == OK
    tok = T(I8, POOL, [4096, 64, 256, 1])
    assert attend(dnn, kcd=tok, vcd=tok) == OK
    row = T(BF16, [3, 8, 1, 64], [1536, 64, 1536, 1])
    assert attend(dnn, qd=row, od=row) == OK and attend(dnn, qd=row, od=row, o=at(1)) == OK
    many = T(BF16, [3, 4096, 1, 64])
    assert attend(dnn, qd=many, od=many, size=1 << 40) == OK
    assert attend(dnn, td=T(I32, TABLE, [0, 1])) == OK and attend(dnn, vc=at(3), vs=at(5)) == OK


def test_refused_attention_calls(dnn):
    d = g.Dnn()
    h, d.h = d.h, None
    assert attend(d) == g.NOT_INITIALIZED
    d.h = h
    d.close()
    for n in ("ad", "qd", "kcd", "vcd", "sd", "td", "od"):
        if n != "ad":
            assert attend(dnn, **{n: Unset()}) == INVALID, n
        assert attend(dnn, **{n: Null()}) == INVALID, n
    for n in ("q", "kc", "vc", "ks", "vs", "table", "lengths", "o"):
        assert attend(dnn, **{n: None}) == INVALID, n
    for h in (0, 6):
        assert attend(dnn, qd=T(BF16, [3, h, 1, 64]), od=T(BF16, [3, h, 1, 64])) == INVALID
    assert attend(dnn, od=T(BF16, [3, 4, 1, 64])) == INVALID
    assert attend(dnn, qd=T(BF16, [2, 8, 1, 64]), od=T(BF16, [2, 8, 1, 64])) == INVALID
    assert attend(dnn, sd=T(F32, [40, 4, 3])) == INVALID and attend(dnn, vcd=T(I8, [41, 4, 16, 64])) == INVALID
    assert attend(dnn, od=T(F16, [3, 8, 1, 64])) == UNSUPPORTED
    assert attend(dnn, qd=T(F32, [3, 8, 1, 64]), od=T(F32, [3, 8, 1, 64])) == UNSUPPORTED
    assert attend(dnn, kcd=T(BF16, POOL), vcd=T(BF16, POOL)) == UNSUPPORTED
    assert attend(dnn, qd=T(BF16, [3, 8, 2, 64]), od=T(BF16, [3, 8, 2, 64])) == UNSUPPORTED
    wide = T(BF16, [3, 4100, 1, 64])
    assert attend(dnn, qd=wide, od=wide, size=1 << 40) == UNSUPPORTED
    for n in ("q", "kc", "vc", "o", "ws"):
        assert attend(dnn, **{n: at(20) + 8}) == UNSUPPORTED or dnn.paged_attention_quantized_workspace(
            T(BF16, [3, 8, 1, 64]), T(I8, POOL), T(I32, TABLE)) == 0, n
    assert attend(dnn, od=T(BF16, [3, 8, 1, 64], [0, 64, 64, 1])) == INVALID
    none = T(BF16, [0, 8, 1, 64])
    assert attend(dnn, qd=none, od=none, td=T(I32, [0, 8]), q=None) == g.SUCCESS
    for p in (3, 4, 5, 6, 7, 8):
        assert attend(dnn, o=at(p)) == INVALID, p
    assert attend(dnn, o=at(1) + 128) == INVALID
    # a table long enough for shares
    far = dict(td=T(I32, [3, 400]))
    need = dnn.paged_attention_quantized_workspace(T(BF16, [3, 8, 1, 64]), T(I8, POOL), far["td"])
    assert need > 0 and attend(dnn, **far, size=need - 1) == INVALID and attend(dnn, **far, ws=None) == INVALID
    assert attend(dnn, **far, ws=at(10) + 4) == UNSUPPORTED
    for p in range(1, 9):
        assert attend(dnn, **far, ws=at(p)) == INVALID, p
    L, out = g.load().dnn, ctypes.c_size_t()
    ask = L.grxdnnPagedAttentionQuantizedGetWorkspaceSize
    q, pool, table = T(BF16, [3, 8, 1, 64]), T(I8, POOL), T(I32, TABLE)
    assert ask(None, q.d, pool.d, table.d, ctypes.byref(out)) == g.NOT_INITIALIZED
    assert ask(dnn.h, q.d, pool.d, table.d, None) == INVALID
    assert ask(dnn.h, None, pool.d, table.d, ctypes.byref(out)) == INVALID
    assert ask(dnn.h, T(BF16, [3, 6, 1, 64]).d, pool.d, table.d, ctypes.byref(out)) == INVALID
    assert ask(dnn.h, q.d, T(BF16, POOL).d, table.d, ctypes.byref(out)) == UNSUPPORTED


def test_misaligned_attention_pointers(dnn):
    """With room for 128 slots, where no workspace is needed and its alignment is not looked at."""
    assert dnn.paged_attention_quantized_workspace(T(BF16, [3, 8, 1, 64]), T(I8, POOL), T(I32, TABLE)) == 0
    for n in ("q", "kc", "vc", "o"):
        for off in (2, 8):
            assert attend(dnn, **{n: at(20) + off}) == UNSUPPORTED, (n, off)
