"""Refusals of di_attn_encoder, di_qk_norm_rope and di_linear_lora: every check
of their arguments, on the host alone (the program sees no device)."""
import os
import subprocess

import pytest

from test_gemm_plans import CSRC, HIPCC, LIB, REPO


def test_refusals(tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("needs hipcc")
    exe = tmp_path / "refusals"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-x", "hip", "-std=c++17", "-O1", "-I", CSRC,
                    os.path.join(REPO, "tests", "attention_layer_refusals.cpp"), "-o", str(exe), "-L", LIB,
                    "-l:libdrawinstant_hip.so", "-Wl,-rpath," + LIB], check=True, timeout=300)
    env = dict(os.environ, HIP_VISIBLE_DEVICES="-1", ROCR_VISIBLE_DEVICES="-1")
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60, env=env)
    assert r.returncode == 0 and r.stdout.strip() == "OK", r.stdout + r.stderr


def test_python_views():
    from drawinstant.attention import BHSD, Rope, heads
    class B:  # noqa: E306  (a view only takes the handle)
        handle = 7
    v = heads(B, 10, 3, 8, start=2)
    assert (v.buf, v.offset, v.token, v.head, v.batch) == (7, 48, 24, 8, 240)
    v = heads(B, 10, 3, 8, BHSD, start=2)
    assert (v.offset, v.token, v.head, v.batch) == (16, 8, 80, 240)
    v = heads(B, 10, 3, 8, token=72, batch=0, offset=24)
    assert (v.offset, v.token, v.head, v.batch) == (24, 72, 8, 0)
    r = Rope([16, 24], [1e4, 2e4], halves=True, one_spectrum=True, pos_batch=5)
    assert (r.axes, list(r.dim), list(r.theta), r.flags, r.pos_batch) == (2, [16, 24, 0, 0], [1e4, 2e4, 0, 0], 3, 5)
    with pytest.raises(ValueError):
        Rope([2] * 5)
    with pytest.raises(ValueError):
        Rope([2, 2], [1e4])
