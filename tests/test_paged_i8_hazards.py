"""The 8-bit paged attention's inline assembly, checked on the code that the build produces
(CPU), by the rules of the 16-bit one's test."""
import os
import subprocess

import pytest

from grxcp_amd import build as B
from test_kernel_hazards import _barrier_waits, _body, _check, _kernels, _waits
from test_paged_hazards import as_buffer_loads, m0_problems, unwaited_reads


def assembled(src, tmp_path_factory):
    dst = tmp_path_factory.mktemp("asm") / "kernel.s"
    r = subprocess.run([B.HIPCC, *B.HIP_FLAGS, *B.EXTRA.get(src, []), *B.INCLUDES, "--cuda-device-only", "-S",
                        os.path.join(B.CSRC, src), "-o", str(dst)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    return _kernels(dst.read_text())


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    return assembled("kernels/paged_attention_i8.hip", tmp_path_factory)


def test_wait_states_and_barriers(kernels):
    split = [(n, b) for n, b in kernels if any(m.startswith("global_load_lds") for m, _, _ in b)]
    assert len(split) >= 8, [n for n, _ in kernels]
    bad = []
    for name, body in split:
        assert any(m.startswith("ds_read_b64_tr_b8") for m, _, _ in body) and any(m == "s_barrier" for m, _, _ in body)
        for p in _check(body) + m0_problems(body) + unwaited_reads(body) + _barrier_waits(as_buffer_loads(body)):
            bad.append(f"{name[:70]}: {p}")
    assert not bad, f"{len(bad)}: " + "\n".join(bad[:10])


def reads_in_flight(body):
    """Loads into LDS that are issued before the transposing reads of what lies there have been
    waited for."""
    out, open_reads = [], False
    for i, (mn, ops, _) in enumerate(body):
        if mn.startswith("ds_read_b64_tr"):
            open_reads = True
        elif mn == "s_waitcnt" and _waits(ops).get("lgkmcnt") == 0:
            open_reads = False
        elif mn.startswith("global_load_lds") and open_reads:
            out.append(f"#{i}")
    return out


def test_a_tile_is_read_before_its_place_is_written(kernels):
    split = [(n, b) for n, b in kernels if any(m.startswith("ds_read_b64_tr") for m, _, _ in b)]
    assert len(split) >= 8
    for name, body in split:
        assert not reads_in_flight(body), name[:70]
    load = "s_mov_b32 m0, s3\ns_nop 0\nglobal_load_lds_dwordx4 v[2:3], off\n"
    read = "ds_read_b64_tr_b8 v[0:1], v4\n"
    assert reads_in_flight(_body(read + load, {0, 1, 2}))
    assert reads_in_flight(_body(read + "s_waitcnt lgkmcnt(1)\n" + load, {0, 1, 2}))
    assert not reads_in_flight(_body(read + "s_waitcnt lgkmcnt(0)\n" + load, {0, 1, 2}))


@pytest.mark.parametrize("src", ["paged_attention_i8", "paged_cache_i8", "qk_norm_rope"])
def test_no_packed_fp32(src, tmp_path_factory):
    for name, body in assembled(f"kernels/{src}.hip", tmp_path_factory):
        assert not [m for m, _, _ in body if m in ("v_pk_add_f32", "v_pk_mul_f32", "v_pk_fma_f32")], name
