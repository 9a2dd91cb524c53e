"""The 8-bit cache's index arithmetic on the CPU (tests/cpp/pages_i8_check.cpp), which its kernels share, and the refusals
of the 8-bit cache, the norms of queries and keys and the page tables that need no device."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not on PATH")
def test_pages_i8_index(tmp_path):
    exe = str(tmp_path / "pages_i8_check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-I", os.path.join(ROOT, "neuralnet.cpp_amd", "csrc"), "-o", exe,
                    os.path.join(ROOT, "tests", "cpp", "pages_i8_check.cpp")], check=True)
    out = subprocess.run([exe], check=False, capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.strip().endswith("wrong 0"), out.stdout + out.stderr


def test_null_context_is_refused(nnhip):
    L = nnhip.lib()
    for st in (L.nnhip_kv_pages_fill_i8(None, None, None, None, 1, None, None, 1, None, None, 0),
               L.nnhip_kv_pages_read_i8(None, None, 1, None, None, 1, None, None),
               L.nnhip_attention_pages_decode_i8(None, None, None, None, None, 1, 1, None, 1, None, None, 0, 1.0, 0.0, None, 0, None),
               L.nnhip_attention_pages_prefill_i8(None, None, None, 1, None, None, 1, 1, 1, None, None, 0, 1.0, 0.0, None, None,
                                                  0, None),
               L.nnhip_qk_norm_rope(None, None, None, 1, 1, 1, 64, None, None, 1e-5, None, None, None, 0, 0, None, None),
               L.nnhip_pages_assign(None, None, 1, 16, 1, 1, None, None, None, None, None, None, 0, None, None),
               L.nnhip_pages_slots(None, None, 1, 16, 1, None, None, 1, 1, None, None),
               L.nnhip_pages_release(None, None, 1, 16, 1, 1, None, None, None, None)):
        assert st == 1 and "null context" in L.nnhip_last_error().decode()


def test_handle_refuses(nnhip):
    import torch
    k, v = torch.zeros(4, 2, 1, 4, 16, 16, dtype=torch.int8), torch.zeros(4, 2, 1, 64, 16, dtype=torch.int8)
    s, t = torch.zeros(4, 2, 1), torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(nnhip.NNHipError, match="device tensor"):
        nnhip.KVPagesI8(k, v, s, s.clone(), t)
    with pytest.raises(nnhip.NNHipError, match="codes must be"):
        nnhip.KVPagesI8(k[0], v, s, s, t)
    with pytest.raises(nnhip.NNHipError, match="codes must be"):
        nnhip.KVPagesI8(k, v, s[0], s, t)
    for bad in ((24, 64, 16), (16, 72, 16), (32, 64, 24), (0, 64, 16), (16, 64, 0)):
        with pytest.raises(nnhip.NNHipError, match="multiples of 16"):
            nnhip.KVPagesI8.empty(4, 2, *bad, t)
