"""grxdnnQkNormRopeForward / Backward without a GPU: argument checks and workspace sizes."""
import ctypes

import pytest

import grxcp_amd as g
from test_paged_host import Null, Unset, at

BF16, F16, F32, I32, I8 = g.GRX_R_16BF, g.GRX_R_16F, g.GRX_R_32F, g.GRX_R_32I, g.GRX_R_8I
INVALID, UNSUPPORTED = g.INVALID_VALUE, g.NOT_SUPPORTED
needs_no_gpu = pytest.mark.skipif(g.device_count() > 0, reason="checks the no-device path")
OK = g.ARCH_MISMATCH
T = g.TensorDesc
Q, K = [2, 6, 5, 64], [2, 3, 5, 64]


@pytest.fixture(scope="module")
def dnn():
    d = g.Dnn()
    yield d
    d.close()


def forward(dnn, **kw):
    a = dict(qd=T(BF16, Q), q=at(1), kd=T(BF16, K), k=at(2), wd=T(BF16, [64]), qg=at(3), kg=at(4), eps=1e-6,
             mode=g.ROPE_HALVES, rotary=64, positions=at(5), freq=at(6), yqd=T(BF16, Q), yq=at(7), ykd=T(BF16, K),
             yk=at(8))
    assert set(kw) <= set(a)
    a.update(kw)
    return dnn.qk_norm_rope(*a.values())


def backward(dnn, **kw):
    a = dict(qd=T(BF16, Q), q=at(1), kd=T(BF16, K), k=at(2), wd=T(BF16, [64]), qg=at(3), kg=at(4), eps=1e-6,
             mode=g.ROPE_HALVES, rotary=64, positions=at(5), freq=at(6), dyqd=T(BF16, Q), dyq=at(9),
             dykd=T(BF16, K), dyk=at(10), yqd=T(BF16, Q), yq=at(7), ykd=T(BF16, K), yk=at(8), dqg=at(11), dkg=at(12),
             ws=at(13), size=1 << 24)
    assert set(kw) <= set(a)
    a.update(kw)
    return dnn.qk_norm_rope_backward(*a.values())


NO_KEYS = dict(kd=None, k=None, kg=None, ykd=None, yk=None)
NO_KEYS_BACK = dict(NO_KEYS, dykd=None, dyk=None, dkg=None)
NO_NORM = dict(wd=None, qg=None, kg=None)


@needs_no_gpu
def test_valid_calls_reach_the_device_check(dnn):
    for call, none in ((forward, NO_KEYS), (backward, NO_KEYS_BACK)):
        more = {"dqg": None, "dkg": None, "ws": None, "size": 0} if call is backward else {}
        assert call(dnn) == OK and call(dnn, **none) == OK
        assert call(dnn, **NO_NORM, **more) == OK
        assert call(dnn, **NO_NORM, **more, eps=float("nan")) == OK          # not looked at
        assert call(dnn, mode=g.ROPE_PAIRS, rotary=16) == OK
        assert call(dnn, rotary=0, positions=None, freq=None) == OK
        # packed projections [2, 5, 6 + 2 * 3, 64]: queries and keys side by side, outputs over them
        row = [12 * 64 * 5, 64, 12 * 64, 1]
        q, k = T(BF16, Q, row), T(BF16, K, row)
        over = dict(qd=q, kd=k, k=at(1) + 2 * 6 * 64, yqd=q, yq=at(1), ykd=k, yk=at(1) + 2 * 6 * 64)
        assert call(dnn, **over) == OK
        assert call(dnn, **dict(over, yk=at(1) + 2 * 9 * 64)) == OK           # over the values, not the keys
        # more key heads than query heads beside each other
        q, k = T(BF16, K, row), T(BF16, Q, row)
        swapped = dict(qd=q, kd=k, k=at(1) + 2 * 3 * 64, yqd=q, yq=at(1), ykd=k, yk=at(1) + 2 * 3 * 64)
        grads = dict(dyqd=T(BF16, K), dykd=T(BF16, Q)) if call is backward else {}
        assert call(dnn, **swapped, **grads) == OK
    assert backward(dnn, yq=at(9), yk=at(10)) == OK and backward(dnn, dqg=None) == OK
    assert backward(dnn, dqg=None, dkg=None, ws=None, size=0) == OK
    assert backward(dnn, **NO_NORM, q=None, k=None, dqg=None, dkg=None, ws=None, size=0) == OK
    # one key head for all, of any stride; a dimension of one has none
    shared = T(BF16, [2, 3, 5, 64], [320, 0, 64, 1])
    assert forward(dnn, kd=shared) == OK
    one = [2, 6, 1, 64]
    assert forward(dnn, **NO_KEYS, qd=T(BF16, one, [384, 64, 7, 1]), yqd=T(BF16, one, [384, 64, 3, 1])) == OK


def test_null_handle_descriptors_and_pointers(dnn):
    for call in (forward, backward):
        d = g.Dnn()
        h, d.h = d.h, None
        assert call(d) == g.NOT_INITIALIZED
        d.h = h
        d.close()
        names = ["qd", "kd", "wd", "yqd", "ykd"] + (["dyqd", "dykd"] if call is backward else [])
        for n in names:
            assert call(dnn, **{n: Unset()}) == INVALID, n
            assert call(dnn, **{n: Null()}) == INVALID, n
        names = ["q", "k", "qg", "kg", "positions", "freq", "yq", "yk"]
        names += ["dyq", "dyk", "ws"] if call is backward else []
        for n in names:
            assert call(dnn, **{n: None}) == INVALID, n
    n = ctypes.c_size_t()
    ask = g.load().dnn.grxdnnQkNormRopeGetWorkspaceSize
    assert ask(None, T(BF16, Q).d, None, None, ctypes.byref(n)) == g.NOT_INITIALIZED
    assert ask(dnn.h, None, None, None, ctypes.byref(n)) == INVALID
    assert ask(dnn.h, T(BF16, Q).d, None, None, None) == INVALID


def test_shapes_types_and_scalars(dnn):
    for call in (forward, backward):
        assert call(dnn, kd=T(BF16, [2, 3, 4, 64]), ykd=T(BF16, [2, 3, 4, 64])) == INVALID
        assert call(dnn, yqd=T(BF16, [2, 6, 5, 128])) == INVALID
        assert call(dnn, qd=T(BF16, [2, 30, 64])) == INVALID
        assert call(dnn, wd=T(BF16, [128])) == INVALID
        assert call(dnn, wd=T(BF16, [64, 1])) == INVALID
        assert call(dnn, wd=T(F32, [64])) == UNSUPPORTED
        assert call(dnn, wd=T(BF16, [64], [2])) == UNSUPPORTED
        assert call(dnn, kd=T(F16, K)) == UNSUPPORTED
        assert call(dnn, yqd=T(F32, Q)) == UNSUPPORTED
        assert call(dnn, qd=T(I8, Q)) == UNSUPPORTED
        d96 = [2, 6, 5, 96]
        assert forward(dnn, **NO_KEYS, qd=T(BF16, d96), yqd=T(BF16, d96), wd=T(BF16, [96])) == UNSUPPORTED
        for eps in (-1e-6, float("nan"), float("inf")):
            assert call(dnn, eps=eps) == INVALID
        for rotary in (-16, 80):
            assert call(dnn, rotary=rotary) == INVALID
        for rotary in (8, 24, 63):
            assert call(dnn, rotary=rotary) == UNSUPPORTED
        assert call(dnn, mode=2) == INVALID
        more = {"dqg": None, "dkg": None} if call is backward else {}
        assert call(dnn, **NO_NORM, **more, rotary=0) == INVALID             # nothing to do
        assert call(dnn, wd=None) == INVALID                                 # gains without a descriptor
        for strides in ([1920, 320, 64, 2], [1920, 320, 68, 1], [1924, 320, 64, 1]):
            assert call(dnn, qd=T(BF16, Q, strides)) == UNSUPPORTED
            assert call(dnn, yqd=T(BF16, Q, strides)) == UNSUPPORTED
        for n in ("q", "k", "qg", "kg", "yq", "yk") + (("dyq", "dyk", "ws") if call is backward else ()):
            assert call(dnn, **{n: at(20) + 8}) == UNSUPPORTED, n
        many = [1 << 16, 1, 1 << 15, 64]
        far = T(BF16, many, [0, 0, 64, 1])
        more = dict(dyqd=far, dykd=None, dyk=None, dkg=None) if call is backward else {}
        assert call(dnn, **NO_KEYS, qd=far, yqd=far, **more) == UNSUPPORTED   # 2^31 tokens
        heads = T(BF16, [1, (1 << 20) + 1, 1, 64])
        more = dict(dyqd=heads, dykd=None, dyk=None, dkg=None) if call is backward else {}
        assert call(dnn, **NO_KEYS, qd=heads, yqd=heads, **more) == UNSUPPORTED
    assert backward(dnn, **NO_NORM) == INVALID                               # gradients of no gains
    assert backward(dnn, dyqd=T(BF16, [2, 6, 4, 64])) == INVALID
    # parts of the keys' arguments
    for n in NO_KEYS:
        if n != "kd":
            keep = {x: v for x, v in NO_KEYS.items() if x != n}
            assert forward(dnn, **keep) == INVALID, n
    assert backward(dnn, **{x: v for x, v in NO_KEYS_BACK.items() if x != "dkg"}) == INVALID


def test_empty_calls_succeed_without_a_device(dnn):
    for shape in ([0, 6, 5, 64], [2, 0, 5, 64], [2, 6, 0, 64]):
        x = T(BF16, shape)
        assert forward(dnn, **NO_KEYS, qd=x, yqd=x, q=None, yq=None) == g.SUCCESS
        assert backward(dnn, **NO_KEYS_BACK, qd=x, yqd=x, dyqd=x, q=None, dqg=None, ws=None, size=0) == g.SUCCESS


def test_overlaps_are_refused(dnn):
    for call in (forward, backward):
        assert call(dnn, yq=at(8)) == INVALID                                # one output for both
        for p in (2, 3, 4, 5, 6):
            assert call(dnn, yq=at(p)) == INVALID, p
        for p in (1, 3, 4, 5, 6):
            assert call(dnn, yk=at(p)) == INVALID, p
        assert call(dnn, yq=at(1) + 128) == INVALID                          # over other rows of q
        assert call(dnn, yqd=T(BF16, Q, [1920, 64, 384, 1]), yq=at(1)) == INVALID   # over q, in another order
        assert call(dnn, yqd=T(BF16, Q, [1920, 0, 64, 1])) == INVALID        # rows that share addresses
        row = [12 * 64 * 5, 64, 12 * 64, 1]
        q, k = T(BF16, Q, row), T(BF16, K, row)
        assert call(dnn, qd=q, kd=k, k=at(1) + 2 * 6 * 64, yqd=q, yq=at(1) + 2 * 64, ykd=k) == INVALID
    for n in ("dqg", "dkg", "ws"):
        for p in (1, 2, 3, 4, 5, 6, 7, 8, 9, 10):
            assert backward(dnn, **{n: at(p)}) == INVALID, (n, p)
    assert backward(dnn, dqg=at(12)) == INVALID and backward(dnn, ws=at(11)) == INVALID
    assert backward(dnn, yq=at(10)) == INVALID and backward(dnn, yk=at(9)) == INVALID


def test_workspace_sizes(dnn):
    q, k, w = T(BF16, Q), T(BF16, K), T(BF16, [64])
    n = dnn.qk_norm_rope_workspace(q, k, w)
    assert n > 0 and dnn.qk_norm_rope_workspace(q, k, None) == 0
    assert dnn.qk_norm_rope_workspace(T(BF16, [0, 6, 5, 64]), None, w) == 0
    assert backward(dnn, size=n - 1) == INVALID and backward(dnn, ws=None) == INVALID
    # it does not grow with the tokens past what fills the GPU
    assert dnn.qk_norm_rope_workspace(T(BF16, [64, 32, 8192, 128], [0, 128, 4096, 1]), None, T(BF16, [128])) < 1 << 22
