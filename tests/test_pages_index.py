"""The paged cache's index arithmetic on the CPU (tests/cpp/pages_index_check.cpp): pages that end inside
a chunk, bad ids, packings that are not in order, limits. The kernels use the same functions. And the
refusals of the Python handles that need no device."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not on PATH")
def test_pages_index(tmp_path):
    exe = str(tmp_path / "pages_index_check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-I", os.path.join(ROOT, "neuralnet.cpp_amd", "csrc"), "-o", exe,
                    os.path.join(ROOT, "tests", "cpp", "pages_index_check.cpp")], check=True)
    out = subprocess.run([exe], check=False, capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.strip().endswith("wrong 0"), out.stdout + out.stderr


def test_null_context_is_refused(nnhip):
    L = nnhip.lib()
    assert L.nnhip_kv_pages_fill(None, None, None, None, 1, None, None, 1, None, None, 0) == 1
    assert "null context" in L.nnhip_last_error().decode()
    assert L.nnhip_attention_pages_decode(None, None, None, None, None, 1, 1, None, 1, None, None, 0, 1.0, 0.0, None, 0,
                                          None) == 1
    assert L.nnhip_logits_adjust_rows(None, None, 1, 1, None, None, None, None) == 1
    assert L.nnhip_token_counts_add(None, None, 1, None, 1, 1, None) == 1
    assert L.nnhip_attention_pages_workspace_bytes(None, 1, 1, 1, 64, 1000) == 0
    assert L.nnhip_logits_workspace_bytes(None, 1000, 1) == 0


def test_handles_refuse(nnhip):
    import torch
    pool = torch.zeros(4, 2, 16, 64)
    with pytest.raises(nnhip.NNHipError, match="device tensor"):
        nnhip.KVPages(pool, pool.clone(), torch.zeros(1, 4, dtype=torch.int32))
    with pytest.raises(nnhip.NNHipError, match="num_pages, Hkv"):
        nnhip.KVPages(pool[0], pool[0], torch.zeros(1, 4, dtype=torch.int32))
    with pytest.raises(nnhip.NNHipError, match="rows"):
        nnhip.LogitRules(10, counts=torch.zeros(2, 10, dtype=torch.int32), repeat=torch.ones(3))
    with pytest.raises(nnhip.NNHipError, match="device tensor"):
        nnhip.LogitRules(10, bias=torch.zeros(1, 10))
