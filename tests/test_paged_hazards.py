"""The paged attention's inline assembly, checked on the code that the build produces (CPU).

The kernel's loads into LDS are inline assembly, of which the compiler knows neither the
counter nor M0. Checked in every kernel that has them: a wait state between M0's write and
the load, in the same statement; no s_barrier (behind which waves take over each other's
LDS) with such a load or an LDS access outstanding; a wait for all loads between the first
of them and the first transposing read of what they bring. The general rules on inline
assembly's wait states hold too."""
import os
import subprocess

import pytest

from grxcp_amd import build as B
from test_kernel_hazards import _barrier_waits, _body, _check, _kernels, _waits

SRC = "kernels/paged_attention.hip"


def as_buffer_loads(body):
    """The stream with the global form of a load into LDS under the name that the barrier
    rule knows."""
    return [("buffer_load_dwordx4", ["lds"], a) if mn.startswith("global_load_lds") else (mn, ops, a)
            for mn, ops, a in body]


def m0_problems(body):
    out = []
    for i, (mn, _, a) in enumerate(body):
        if a and mn.startswith("global_load_lds"):
            before = [(m, o[:1]) for m, o, _ in body[max(0, i - 2):i]]
            if before[-1][0] != "s_nop" or before[0] != ("s_mov_b32", ["m0"]):
                out.append(f"#{i}: {before}")
    return out


def unwaited_reads(body):
    """The transposing reads before which no load into LDS was waited for."""
    loads = waits = 0
    out = []
    for i, (mn, ops, _) in enumerate(body):
        if mn.startswith("global_load_lds"):
            loads += 1
        elif mn == "s_waitcnt" and loads and _waits(ops).get("vmcnt") == 0:
            waits += 1
        elif mn.startswith("ds_read_b64_tr") and not waits:
            out.append(f"#{i}: after {loads} loads")
    return out


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    dst = tmp_path_factory.mktemp("asm") / "paged_attention.s"
    r = subprocess.run([B.HIPCC, *B.HIP_FLAGS, *B.EXTRA.get(SRC, []), *B.INCLUDES, "--cuda-device-only", "-S",
                        os.path.join(B.CSRC, SRC), "-o", str(dst)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    return _kernels(dst.read_text())


def test_wait_states_and_barriers(kernels):
    split = [(n, b) for n, b in kernels if any(m.startswith("global_load_lds") for m, _, _ in b)]
    assert len(split) >= 8, [n for n, _ in kernels]
    bad = []
    for name, body in split:
        assert any(m.startswith("ds_read_b64_tr") for m, _, _ in body) and any(m == "s_barrier" for m, _, _ in body)
        for p in _check(body) + m0_problems(body) + unwaited_reads(body) + _barrier_waits(as_buffer_loads(body)):
            bad.append(f"{name[:70]}: {p}")
    assert not bad, f"{len(bad)}: " + "\n".join(bad[:10])


def test_no_packed_fp32(kernels):
    for name, body in kernels:
        assert not [m for m, _, _ in body if m in ("v_pk_add_f32", "v_pk_mul_f32", "v_pk_fma_f32")], name


def test_the_checks_find_what_they_are_for():
    load = "s_mov_b32 m0, s3\n{nop}global_load_lds_dwordx4 v[2:3], off\n"
    good, bare = load.format(nop="s_nop 0\n"), "s_nop 0\n" + load.format(nop="")
    assert not m0_problems(_body(good, {0, 1, 2})) and m0_problems(_body(bare, {0, 1, 2}))
    read = "ds_read_b64_tr_b16 v[0:1], v4\n"
    assert unwaited_reads(_body(good + read, {0, 1, 2}))
    assert unwaited_reads(_body(good + "s_waitcnt vmcnt(2)\n" + read, {0, 1, 2}))
    assert not unwaited_reads(_body(good + "s_waitcnt vmcnt(0) lgkmcnt(0)\n" + read, {0, 1, 2}))
    bar = good + "s_waitcnt vmcnt({n}) lgkmcnt(0)\ns_barrier\n"
    assert _barrier_waits(as_buffer_loads(_body(bar.format(n=4), {0, 1, 2})))
    assert not _barrier_waits(as_buffer_loads(_body(bar.format(n=0), {0, 1, 2})))
