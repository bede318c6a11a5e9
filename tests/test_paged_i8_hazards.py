"""The 8-bit paged attention's inline assembly, checked on the code that the build produces
(CPU), by the rules of the 16-bit one's test."""
import os
import subprocess

import pytest

from grxcp_amd import build as B
from test_kernel_hazards import _barrier_waits, _check, _kernels
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


@pytest.mark.parametrize("src", ["paged_attention_i8", "paged_cache_i8", "qk_norm_rope"])
def test_no_packed_fp32(src, tmp_path_factory):
    for name, body in assembled(f"kernels/{src}.hip", tmp_path_factory):
        assert not [m for m, _, _ in body if m in ("v_pk_add_f32", "v_pk_mul_f32", "v_pk_fma_f32")], name
