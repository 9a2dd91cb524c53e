"""Python binding (ctypes) of libnn-hip.so — the MI355X BitLinear W1.58A8 engine.

The product is the C ABI in include/nnhip.h and the C++ nn:: engine layer built into the
same library; this module is plumbing for the tests and bench.py. Device memory comes from
torch (CUDA/HIP tensors), and every call runs on torch's current stream, so it is ordered
with torch's own work. There is no CPU fallback: if libnn-hip.so is missing or no gfx950
device is visible, the calls raise.

The directory name contains a dot, so load it by path:
    spec = importlib.util.spec_from_file_location(
        "nnhip_py", "neuralnet.cpp_amd/__init__.py",
        submodule_search_locations=["neuralnet.cpp_amd"])
"""
from __future__ import annotations

import ctypes
import os
import subprocess

_HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(_HERE)
LIB_PATH = os.path.join(_HERE, "libnn-hip.so")
HEADER_PATH = os.path.join(ROOT, "include", "nnhip.h")

TILE_K = 256
TILE_ROWS = 16
GEMV_MAX_M = 16


class NNHipError(RuntimeError):
    """A libnn-hip.so call returned a status other than NNHIP_OK."""

    def __init__(self, status: int, message: str):
        super().__init__(f"[status {status}] {message}")
        self.status = status


def build(jobs: int = 8) -> None:
    """Compile libnn-hip.so in-tree with neuralnet.cpp_amd/Makefile (hipcc, gfx950)."""
    subprocess.run(["make", "-s", "-C", _HERE, f"-j{jobs}"], check=True)


_vp = ctypes.c_void_p
_sz = ctypes.c_size_t
_st = ctypes.c_int
_f = ctypes.c_float


class GemvDesc(ctypes.Structure):
    _fields_ = [("rp", _vp), ("tau", _vp), ("xi", _vp), ("s", _vp), ("rowsum", _vp),
                ("bias", _vp), ("y", _vp), ("N", ctypes.c_uint64), ("K", ctypes.c_uint64),
                ("M", ctypes.c_uint64)]


class _KVPagesDesc(ctypes.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("table", _vp), ("num_pages", _sz), ("page_size", _sz),
                ("table_stride", _sz), ("Hkv", _sz), ("dk", _sz), ("f16", _st)]


class _KVPagesI8Desc(ctypes.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("k_scale", _vp), ("v_scale", _vp), ("table", _vp), ("num_pages", _sz),
                ("page_size", _sz), ("block", _sz), ("table_stride", _sz), ("Hkv", _sz), ("dk", _sz)]


class _LogitRulesDesc(ctypes.Structure):
    _fields_ = [("counts", _vp), ("repeat", _vp), ("presence", _vp), ("frequency", _vp), ("bias", _vp),
                ("bias_stride", _sz), ("allowed", _vp), ("allowed_stride", _sz), ("count_choice", _st)]


# name -> (restype, argtypes); every nnhip_* symbol of include/nnhip.h
SIGNATURES = {
    "nnhip_last_error": (ctypes.c_char_p, []),
    "nnhip_version": (ctypes.c_char_p, []),
    "nnhip_fnv1a64": (ctypes.c_uint64, [_vp, _sz]),
    "nnhip_device_count": (_st, [ctypes.POINTER(ctypes.c_int)]),
    "nnhip_ctx_create": (_st, [ctypes.c_int, ctypes.POINTER(_vp)]),
    "nnhip_ctx_destroy": (_st, [_vp]),
    "nnhip_ctx_set_stream": (_st, [_vp, _vp]),
    "nnhip_ctx_reset_stream": (_st, [_vp]),
    "nnhip_ctx_get_stream": (_st, [_vp, ctypes.POINTER(_vp)]),
    "nnhip_sync": (_st, [_vp]),
    "nnhip_ctx_set_gemm_tile": (_st, [_vp, _st]),
    "nnhip_ctx_prefetch_next": (_st, [_vp, _sz, ctypes.POINTER(_vp), ctypes.POINTER(_sz)]),
    "nnhip_malloc": (_st, [_vp, _sz, ctypes.POINTER(_vp)]),
    "nnhip_free": (_st, [_vp, _vp]),
    "nnhip_memcpy_h2d": (_st, [_vp, _vp, _vp, _sz]),
    "nnhip_memcpy_d2h": (_st, [_vp, _vp, _vp, _sz]),
    "nnhip_memcpy_d2d": (_st, [_vp, _vp, _vp, _sz]),
    "nnhip_fill_u32": (_st, [_vp, _vp, ctypes.c_uint32, _sz]),
    "nnhip_device_name": (_st, [ctypes.c_int, ctypes.c_char_p, _sz]),
    "nnhip_convert_f32_f16": (_st, [_vp, _vp, _sz, _vp]),
    "nnhip_convert_f16_f32": (_st, [_vp, _vp, _sz, _vp]),
    "nnhip_row_absmean": (_st, [_vp, _vp, _sz, _sz, _vp]),
    "nnhip_trit_pack": (_st, [_vp, _vp, _vp, _sz, _sz, _vp]),
    "nnhip_col_reduce_max": (_st, [_vp, _vp, _sz, _sz, _vp]),
    "nnhip_abs": (_st, [_vp, _vp, _sz, _vp]),
    "nnhip_scale_inplace": (_st, [_vp, _vp, _sz, _f]),
    "nnhip_act_scale": (_st, [_vp, _vp, _sz, _sz, _vp]),
    "nnhip_quantize_i8": (_st, [_vp, _vp, _vp, _sz, _sz, ctypes.c_int, _vp]),
    "nnhip_unpack_i8": (_st, [_vp, _vp, _sz, _sz, _vp]),
    "nnhip_matmul_q_i8": (_st, [_vp, _vp, _vp, _vp, _vp, _sz, _sz, _sz, _vp]),
    "nnhip_matmul_q_i8_noalloc": (_st, [_vp, _vp, _vp, _vp, _vp, _sz, _sz, _sz, _vp]),
    "nnhip_add_row_broadcast": (_st, [_vp, _vp, _vp, _sz, _sz]),
    "nnhip_matmul_q": (_st, [_vp, _vp, _vp, _vp, ctypes.c_int, _sz, _sz, _sz, _vp, ctypes.c_int]),
    "nnhip_matmul_q_t": (_st, [_vp, _vp, _vp, _vp, ctypes.c_int, _sz, _sz, _sz, _vp, ctypes.c_int]),
    "nnhip_rmsnorm": (_st, [_vp, _vp, _vp, _f, _sz, _sz, _vp]),
    "nnhip_layernorm": (_st, [_vp, _vp, _vp, _vp, _f, _sz, _sz, _vp]),
    "nnhip_repacked_bytes": (_sz, [_sz, _sz]),
    "nnhip_repack_ternary": (_st, [_vp, _vp, _sz, _sz, _vp]),
    "nnhip_unrepack_ternary": (_st, [_vp, _vp, _sz, _sz, _vp]),
    "nnhip_act_i8_bytes": (_sz, [_sz, _sz]),
    "nnhip_act_quant_i8": (_st, [_vp, _vp, _sz, _sz, _vp, _vp, _vp, _vp]),
    "nnhip_rmsnorm_quant_i8": (_st, [_vp, _vp, _vp, _f, _sz, _sz, _vp, _vp, _vp, _vp]),
    "nnhip_act_i8_from_container": (_st, [_vp, _vp, _sz, _sz, _vp, _vp]),
    "nnhip_act_i8_to_container": (_st, [_vp, _vp, _sz, _sz, _vp]),
    "nnhip_ternary_matmul": (_st, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _sz, _sz, _sz, _vp]),
    "nnhip_ternary_matmul_f": (_st, [_vp, _vp, _vp, _vp, ctypes.c_int, _sz, _sz, _sz, _vp, ctypes.c_int]),
    "nnhip_ternary_matmul_t_f": (_st, [_vp, _vp, _vp, _vp, ctypes.c_int, _sz, _sz, _sz, _vp, ctypes.c_int]),
    "nnhip_trit_transpose": (_st, [_vp, _vp, _sz, _sz, _vp]),
    "nnhip_stream_xor": (_st, [_vp, _vp, _sz, _vp]),
    "nnhip_device_info": (_st, [ctypes.c_int] + [ctypes.POINTER(ctypes.c_int)] * 4),
    "nnhip_ternary_matmul_add": (_st, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _sz, _sz, _sz, _vp]),
    "nnhip_ternary_matmul_add_tokens": (_st, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _sz, _sz, _sz, _vp]),
    "nnhip_ternary_matmul_partial": (_st, [_vp, _vp, _vp, _sz, _sz, _sz, _sz, _vp]),
    "nnhip_partial_residual_quant_i8": (_st, [_vp, _vp, _sz, _vp, _vp, _vp, _vp, _vp, _sz, _sz, _vp, _vp, _f, _vp,
                                              _vp, _vp]),
    "nnhip_partial_residual_quant_i8_tokens": (_st, [_vp, _vp, _sz, _vp, _vp, _vp, _vp, _vp, _sz, _sz, _vp, _vp, _f, _vp,
                                              _vp, _vp]),
    "nnhip_ternary_matmul_n": (_st, [_vp, _sz, ctypes.POINTER(_vp), ctypes.POINTER(_vp), ctypes.POINTER(_vp),
                                     ctypes.POINTER(_sz), ctypes.POINTER(_vp), _vp, _vp, _vp, _sz, _sz]),
    "nnhip_ternary_matmul_n_tokens": (_st, [_vp, _sz, ctypes.POINTER(_vp), ctypes.POINTER(_vp), ctypes.POINTER(_vp),
                                     ctypes.POINTER(_sz), ctypes.POINTER(_vp), _vp, _vp, _vp, _sz, _sz]),
    "nnhip_ffn_glu_i8_add": (_st, [_vp, _vp, _vp, _f, _sz, _sz, _sz, ctypes.c_int, _vp, _vp, _vp, _vp, _f, _vp, _vp,
                                   _vp, _vp, _vp]),
    "nnhip_group_create": (_st, [_vp, ctypes.POINTER(GemvDesc), _sz, ctypes.POINTER(_vp)]),
    "nnhip_group_run": (_st, [_vp, _vp]),
    "nnhip_group_destroy": (_st, [_vp, _vp]),
    "nnhip_gemv_grid_waves": (_sz, [_vp, _sz]),
    "nnhip_group_info": (_st, [_vp, ctypes.POINTER(ctypes.c_int), ctypes.POINTER(_sz), ctypes.POINTER(_sz)]),
    "nnhip_glu": (_st, [_vp, _vp, _sz, _sz, ctypes.c_int, _vp]),
    "nnhip_glu_rows": (_sz, [_sz]),
    "nnhip_glu_interleave": (_st, [_vp, _vp, _vp, _vp, _sz, _sz, _vp, _vp, _vp]),
    "nnhip_ternary_matmul_glu": (_st, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _sz, _sz, _sz, ctypes.c_int, _vp]),
    "nnhip_ternary_matmul_glu_tokens": (_st, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _sz, _sz, _sz, ctypes.c_int,
                                              _vp]),
    "nnhip_rmsnorm_quant_i8_tokens": (_st, [_vp, _vp, _vp, _f, _sz, _sz, _vp, _vp, _vp]),
    "nnhip_embedding_rmsnorm_quant_i8_tokens": (_st, [_vp, _vp, _vp, _sz, _sz, _sz, _vp, _f, _vp, _vp, _vp, _vp]),
    "nnhip_ffn_glu_workspace_bytes": (_sz, [_sz, _sz, _sz]),
    "nnhip_ffn_glu_i8": (_st, [_vp, _vp, _vp, _f, _sz, _sz, _sz, ctypes.c_int, _vp, _vp, _vp, _vp, _f, _vp, _vp,
                               _vp, _vp]),
    "nnhip_rope_table": (_st, [_sz, _sz, _vp, _vp]),
    "nnhip_attention_workspace_bytes": (_sz, [_sz, _sz, _sz, _sz, _sz]),
    "nnhip_attention_decode": (_st, [_vp, _vp, _vp, _vp, _sz, _sz, _sz, _sz, _vp, _sz, _vp, _vp, _vp, _vp, _sz, _f,
                                     _vp]),
    "nnhip_attention_decode_tokens": (_st, [_vp, _vp, _vp, _vp, _sz, _sz, _sz, _sz, _vp, _sz, _vp, _vp, _vp, _vp, _sz,
                                            _f, _vp]),
    "nnhip_attention_decode_h": (_st, [_vp, _vp, _vp, _vp, _sz, _sz, _sz, _sz, _vp, _sz, _vp, _vp, _vp, _vp, _sz, _f,
                                       _vp]),
    "nnhip_attention_decode_tokens_h": (_st, [_vp, _vp, _vp, _vp, _sz, _sz, _sz, _sz, _vp, _sz, _vp, _vp, _vp, _vp,
                                              _sz, _f, _vp]),
    "nnhip_add": (_st, [_vp, _vp, _vp, _sz, _vp]),
    "nnhip_kv_cache_fill": (_st, [_vp, _vp, _vp, _sz, _sz, _sz, _sz, _sz, _vp, _vp, _vp, _vp, _sz]),
    "nnhip_kv_cache_fill_h": (_st, [_vp, _vp, _vp, _sz, _sz, _sz, _sz, _sz, _vp, _vp, _vp, _vp, _sz]),
    "nnhip_attention_prefill": (_st, [_vp, _vp, _vp, _vp, _sz, _sz, _sz, _sz, _sz, _sz, _vp, _vp, _sz, _f, _vp]),
    "nnhip_attention_prefill_h": (_st, [_vp, _vp, _vp, _vp, _sz, _sz, _sz, _sz, _sz, _sz, _vp, _vp, _sz, _f, _vp]),
    "nnhip_copy_columns": (_st, [_vp, _vp, _sz, _sz, _sz, _sz, _sz, _vp]),
    "nnhip_embedding_gather": (_st, [_vp, _vp, _vp, _sz, _sz, _sz, _vp]),
    "nnhip_embedding_gather_tokens": (_st, [_vp, _vp, _vp, _sz, _sz, _sz, _vp]),
    "nnhip_argmax_cols": (_st, [_vp, _vp, _sz, _sz, _vp]),
    "nnhip_argmax_rows": (_st, [_vp, _vp, _sz, _sz, _vp, _vp]),
    "nnhip_kv_pages_fill": (_st, [_vp, _vp, _vp, _vp, _sz, _vp, _vp, _sz, _vp, _vp, _sz]),
    "nnhip_attention_pages_decode": (_st, [_vp, _vp, _vp, _vp, _vp, _sz, _sz, _vp, _sz, _vp, _vp, _sz, _f, _f, _vp,
                                           _st, _vp]),
    "nnhip_attention_pages_prefill": (_st, [_vp, _vp, _vp, _sz, _vp, _vp, _sz, _sz, _sz, _vp, _vp, _sz, _f, _f, _vp,
                                            _vp, _vp]),
    "nnhip_attention_pages_prefill_distance": (_st, [_vp, _vp, _vp, _sz, _vp, _vp, _sz, _sz, _sz, _vp, _vp, _sz, _f, _f,
                                                     _vp, _vp, _vp]),
    "nnhip_kv_pages_fill_i8": (_st, [_vp, _vp, _vp, _vp, _sz, _vp, _vp, _sz, _vp, _vp, _sz]),
    "nnhip_kv_pages_read_i8": (_st, [_vp, _vp, _sz, _vp, _vp, _sz, _vp, _vp]),
    "nnhip_attention_pages_decode_i8": (_st, [_vp, _vp, _vp, _vp, _vp, _sz, _sz, _vp, _sz, _vp, _vp, _sz, _f, _f, _vp,
                                              _st, _vp]),
    "nnhip_attention_pages_prefill_i8": (_st, [_vp, _vp, _vp, _sz, _vp, _vp, _sz, _sz, _sz, _vp, _vp, _sz, _f, _f, _vp,
                                               _vp, _st, _vp]),
    "nnhip_qk_norm_rope": (_st, [_vp, _vp, _vp, _sz, _sz, _sz, _sz, _vp, _vp, _f, _vp, _vp, _vp, _sz, _st, _vp, _vp]),
    "nnhip_pages_assign": (_st, [_vp, _vp, _sz, _sz, _sz, _sz, _vp, _vp, _vp, _vp, _vp, _vp, _sz, _vp, _vp]),
    "nnhip_pages_slots": (_st, [_vp, _vp, _sz, _sz, _sz, _vp, _vp, _sz, _sz, _vp, _vp]),
    "nnhip_pages_release": (_st, [_vp, _vp, _sz, _sz, _sz, _sz, _vp, _vp, _vp, _vp]),
    "nnhip_attention_pages_workspace_bytes": (_sz, [_vp, _sz, _sz, _sz, _sz, _sz]),
    "nnhip_logits_workspace_bytes": (_sz, [_vp, _sz, _sz]),
    "nnhip_logits_adjust_rows": (_st, [_vp, _vp, _sz, _sz, _vp, _vp, _vp, _vp]),
    "nnhip_token_counts_add": (_st, [_vp, _vp, _sz, _vp, _sz, _sz, _vp]),
}

ACT_SWIGLU, ACT_RELU2GLU = 0, 1
# prefill GEMM block tiles (nnhip_ctx_set_gemm_tile)
GEMM_TILE_AUTO, GEMM_TILE_256x128, GEMM_TILE_128x128, GEMM_TILE_64x64 = 0, 1, 2, 3

_lib = None


def lib() -> ctypes.CDLL:
    """Load libnn-hip.so (raises if it has not been built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise NNHipError(-1, f"{LIB_PATH} is missing: run __graft_entry__.build() "
                                 "(make -C neuralnet.cpp_amd)")
        L = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            f = getattr(L, name)
            f.restype = res
            f.argtypes = args
        _lib = L
    return _lib


def _check(status: int, fn: str) -> None:
    if status != 0:
        msg = lib().nnhip_last_error().decode(errors="replace")
        raise NNHipError(status, msg or fn)


def fnv1a64(t) -> str:
    """FNV-1a 64 of a tensor's bytes (a device tensor is copied to the host first), as hex: the
    reference layer_bench --hash of an output."""
    import numpy as np
    a = np.ascontiguousarray(t.detach().cpu().numpy() if hasattr(t, "detach") else t)
    return "%016x" % lib().nnhip_fnv1a64(_vp(a.ctypes.data), a.nbytes)


def repacked_bytes(N: int, K: int) -> int:
    return int(lib().nnhip_repacked_bytes(N, K))


def act_i8_bytes(K: int, M: int) -> int:
    return int(lib().nnhip_act_i8_bytes(K, M))


def glu_rows(F: int) -> int:
    return int(lib().nnhip_glu_rows(F))


def rope_table(dk: int, max_len: int):
    """Host RoPE tables (cos, sin), each (max_len, dk/2) float32 numpy (nnhip_rope_table)."""
    import numpy as np
    c = np.empty((max_len, dk // 2), np.float32)
    s = np.empty((max_len, dk // 2), np.float32)
    _check(lib().nnhip_rope_table(dk, max_len, _vp(c.ctypes.data), _vp(s.ctypes.data)), "nnhip_rope_table")
    return c, s


def attention_workspace_bytes(B: int, H: int, Hkv: int, dk: int, len_bound: int) -> int:
    return int(lib().nnhip_attention_workspace_bytes(B, H, Hkv, dk, len_bound))


def device_info(device: int = 0) -> dict:
    """HIP's compute-unit count, peak engine clock, memory clock (kHz) and bus width (bits)."""
    v = [ctypes.c_int(0) for _ in range(4)]
    _check(lib().nnhip_device_info(device, *[ctypes.byref(x) for x in v]), "nnhip_device_info")
    return {"cus": v[0].value, "clock_khz": v[1].value, "mem_clock_khz": v[2].value, "bus_bits": v[3].value}


def device_name(device: int = 0) -> str:
    """HIP's name and architecture of a device (nnhip_device_name)."""
    buf = ctypes.create_string_buffer(256)
    _check(lib().nnhip_device_name(device, buf, 256), "nnhip_device_name")
    return buf.value.decode(errors="replace")


def kp(K: int) -> int:
    return (K + TILE_K - 1) // TILE_K * TILE_K


def _device_args(named):
    """Checks (name, tensor or None, dtypes, shape or None) tuples: device, contiguity, type and shape, all
    on one device."""
    dev = None
    for name, t, dtypes, shape in named:
        if t is None:
            continue
        if not t.is_cuda:
            raise NNHipError(1, f"{name} must be a device tensor")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise NNHipError(1, f"{name} is on {t.device}, other operands on {dev}")
        if not t.is_contiguous():
            raise NNHipError(1, f"{name} must be contiguous")
        if t.dtype not in dtypes:
            raise NNHipError(1, f"{name} has dtype {t.dtype}, expected {' or '.join(str(d) for d in dtypes)}")
        if shape is not None and tuple(t.shape) != shape:
            raise NNHipError(1, f"{name} has shape {tuple(t.shape)}, expected {shape}")
    return dev


class KVPages:
    """One layer's paged KV cache (nnhip_kv_pages): pools k, v (num_pages, Hkv, page_size, dk), float32 or
    float16, and the page table (B, pages per sequence) int32, whose rows the sequences of a call are. The
    tensors' contents may change between calls (the table's too); the tensors themselves stay."""

    def __init__(self, k, v, table):
        import torch
        if k.dim() != 4 or table.dim() != 2:
            raise NNHipError(1, "pools must be (num_pages, Hkv, page_size, dk), the table (B, pages)")
        self.device = _device_args([("k", k, (torch.float32, torch.float16), None), ("v", v, (k.dtype,), tuple(k.shape)),
                                    ("table", table, (torch.int32,), None)])
        self.k, self.v, self.table = k, v, table
        self.num_pages, self.Hkv, self.page_size, self.dk = k.shape
        self.rows, self.max_pages = table.shape
        self.desc = _KVPagesDesc(k.data_ptr(), v.data_ptr(), table.data_ptr(), self.num_pages, self.page_size,
                                 self.max_pages, self.Hkv, self.dk, int(k.dtype == torch.float16))
        self.ref = ctypes.addressof(self.desc)


class KVPagesI8:
    """One layer's paged KV cache in 8 bits (nnhip_kv_pages_i8): codes k (num_pages, Hkv, page_size/16, dk/16, 16, 16) and v
    (num_pages, Hkv, page_size/16, dk, 16) int8, keys by (16 positions, 16 dimensions) and values by (dimension, 16 positions);
    scales k_scale, v_scale (num_pages, Hkv, page_size/block) float32, one for every `block` positions of a head; and
    the page table as KVPages'. It is taken wherever KVPages is. empty() makes the tensors of a new cache."""

    def __init__(self, k, v, k_scale, v_scale, table):
        import torch
        if k.dim() != 6 or tuple(k.shape[4:]) != (16, 16) or k_scale.dim() != 3 or table.dim() != 2:
            raise NNHipError(1, "codes must be (num_pages, Hkv, page_size/16, dk/16, 16, 16) and (num_pages, Hkv, "
                                "page_size/16, dk, 16), scales (num_pages, Hkv, page_size/block), the table (B, pages)")
        pages, Hkv, groups, chunks = k.shape[:4]
        i8, f32 = (torch.int8,), (torch.float32,)
        self.device = _device_args([("k", k, i8, None), ("v", v, i8, (pages, Hkv, groups, 16 * chunks, 16)),
                                    ("k_scale", k_scale, f32, (pages, Hkv, k_scale.shape[2])),
                                    ("v_scale", v_scale, f32, tuple(k_scale.shape)), ("table", table, (torch.int32,), None)])
        self.k, self.v, self.k_scale, self.v_scale, self.table = k, v, k_scale, v_scale, table
        self.num_pages, self.Hkv, self.page_size, self.dk = pages, Hkv, 16 * groups, 16 * chunks
        if k_scale.shape[2] < 1 or self.page_size % k_scale.shape[2]:
            raise NNHipError(1, f"{k_scale.shape[2]} scales do not divide a page of {self.page_size} positions")
        self.block = self.page_size // k_scale.shape[2]
        self.rows, self.max_pages = table.shape
        self.desc = _KVPagesI8Desc(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), table.data_ptr(),
                                   pages, self.page_size, self.block, self.max_pages, Hkv, self.dk)
        self.ref = ctypes.addressof(self.desc)

    @classmethod
    def empty(cls, num_pages: int, Hkv: int, page_size: int, dk: int, block: int, table):
        """A new cache on the table's device."""
        import torch
        if page_size < 16 or page_size % 16 or dk % 16 or block < 1 or page_size % block:
            raise NNHipError(1, "page_size and dk must be multiples of 16, block a divisor of page_size")
        new = lambda dt, *s: torch.zeros((num_pages, Hkv) + s, dtype=dt, device=table.device)  # noqa: E731
        scales = [new(torch.float32, page_size // block) for _ in range(2)]
        return cls(new(torch.int8, page_size // 16, dk // 16, 16, 16), new(torch.int8, page_size // 16, dk, 16), *scales, table)


class LogitRules:
    """What nnhip_logits_adjust_rows does to a batch's logits over a vocabulary of V (nnhip_logit_rules): counts
    (B, V) int32, repeat / presence / frequency (B) float32, bias (B, V) or (1, V) float32, allowed
    (B, ceil(V/32)) or (1, ceil(V/32)) int32 words of a bit per token; each may be None. With count_choice the
    chosen tokens are counted. The tensors' contents may change between calls."""

    def __init__(self, V: int, counts=None, repeat=None, presence=None, frequency=None, bias=None, allowed=None,
                 count_choice: bool = False):
        import torch
        f32, i32, words = (torch.float32,), (torch.int32,), (V + 31) // 32
        rows = [t.shape[0] for t in (counts, repeat, presence, frequency) if t is not None]
        rows += [t.shape[0] for t in (bias, allowed) if t is not None and t.shape[0] != 1]
        if any(r != rows[0] for r in rows):
            raise NNHipError(1, f"the rules' rows differ: {rows}")
        self.rows, self.V = rows[0] if rows else None, V  # rows: None fits any batch
        self.device = _device_args(
            [("counts", counts, i32, (self.rows, V)), ("repeat", repeat, f32, (self.rows,)),
             ("presence", presence, f32, (self.rows,)), ("frequency", frequency, f32, (self.rows,)),
             ("bias", bias, f32, None if bias is None else (bias.shape[0], V)),
             ("allowed", allowed, i32, None if allowed is None else (allowed.shape[0], words))])
        self.tensors = (counts, repeat, presence, frequency, bias, allowed)
        self.masks = allowed is not None  # the choice may be -1
        self.counts_choice = bool(count_choice)
        p = [None if t is None else t.data_ptr() for t in self.tensors]
        self.desc = _LogitRulesDesc(p[0], p[1], p[2], p[3], p[4], V if bias is not None and bias.shape[0] > 1 else 0,
                                    p[5], words if allowed is not None and allowed.shape[0] > 1 else 0,
                                    int(count_choice))
        self.ref = ctypes.addressof(self.desc)


class Context:
    """One nnhip context (device + stream). Arguments are torch CUDA tensors."""

    def __init__(self, device: int = 0):
        import torch

        self._torch = torch
        if not torch.cuda.is_available():
            raise NNHipError(4, "no GPU visible to torch")
        self.device = device
        self._device = torch.device("cuda", device)
        # the current stream's handle without a Stream object around it (0.1 instead of 1.1 us; a
        # call's Python side is on the critical path of a decode-size kernel)
        self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
            (lambda d: torch.cuda.current_stream(d).cuda_stream)
        h = _vp()
        _check(lib().nnhip_ctx_create(device, ctypes.byref(h)), "nnhip_ctx_create")
        self.h = h

    def close(self) -> None:
        if getattr(self, "h", None):
            lib().nnhip_ctx_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # -- helpers
    def _bind_stream(self) -> None:
        st = lib().nnhip_ctx_set_stream(self.h, self._raw_stream(self.device))
        if st != 0:
            _check(st, "nnhip_ctx_set_stream")

    def _dev(self, t, dtype=None, name="tensor"):
        """The device address of t (None: null), after its checks."""
        if t is None:
            return None
        if not t.is_cuda:
            raise NNHipError(1, f"{name} must be a device tensor")
        if not t.is_contiguous():
            raise NNHipError(1, f"{name} must be contiguous")
        if dtype is not None and t.dtype is not dtype and t.dtype not in (dtype if isinstance(dtype, tuple) else (dtype,)):
            raise NNHipError(1, f"{name} has dtype {t.dtype}, expected {dtype}")
        return t.data_ptr()

    def _empty(self, shape, dtype):
        return self._torch.empty(shape, dtype=dtype, device=self._device)

    def sync(self) -> None:
        self._bind_stream()
        _check(lib().nnhip_sync(self.h), "nnhip_sync")

    def set_gemm_tile(self, tile: int) -> None:
        """Force the prefill GEMM block tile (GEMM_TILE_*); GEMM_TILE_AUTO picks per call."""
        _check(lib().nnhip_ctx_set_gemm_tile(self.h, tile), "nnhip_ctx_set_gemm_tile")

    def prefetch_next(self, tensors) -> None:
        """Device tensors (up to 4) that the next per-token quantizer call (act_quant_i8 /
        rmsnorm_quant_i8 at M <= 64, rmsnorm_quant_i8_tokens, partial_residual_quant_i8) also
        reads, so that the kernel after it finds them in the memory-side cache. Results are
        unaffected; an empty list clears them."""
        ts = [t for t in tensors if t is not None]
        if len(ts) > 4:
            raise NNHipError(1, "at most 4 ranges")
        ptrs = (_vp * max(1, len(ts)))(*[self._dev(t, None, "range") for t in ts])
        nb = (_sz * max(1, len(ts)))(*[t.numel() * t.element_size() for t in ts])
        _check(lib().nnhip_ctx_prefetch_next(self.h, len(ts), ptrs, nb), "nnhip_ctx_prefetch_next")

    # -- reference-layout primitives
    def row_absmean(self, W):
        torch = self._torch
        N, K = W.shape
        tau = self._empty((N,), torch.float32)
        self._bind_stream()
        _check(lib().nnhip_row_absmean(self.h, self._dev(W, torch.float32, "W"), N, K,
                                       self._dev(tau)), "nnhip_row_absmean")
        return tau

    def trit_pack(self, W, tau):
        torch = self._torch
        N, K = W.shape
        wq = self._empty((N, (K + 15) // 16), torch.int32)
        self._bind_stream()
        _check(lib().nnhip_trit_pack(self.h, self._dev(W, torch.float32, "W"),
                                     self._dev(tau, torch.float32, "tau"), N, K, self._dev(wq)),
               "nnhip_trit_pack")
        return wq

    def col_reduce_max(self, x):
        torch = self._torch
        rows, cols = x.shape
        out = self._empty((cols,), torch.float32)
        self._bind_stream()
        _check(lib().nnhip_col_reduce_max(self.h, self._dev(x, torch.float32, "x"), rows, cols,
                                          self._dev(out)), "nnhip_col_reduce_max")
        return out

    def abs(self, x, out=None):
        torch = self._torch
        out = self._empty(x.shape, torch.float32) if out is None else out
        self._bind_stream()
        _check(lib().nnhip_abs(self.h, self._dev(x, torch.float32, "x"), x.numel(), self._dev(out)),
               "nnhip_abs")
        return out

    def scale_inplace(self, x, alpha: float):
        self._bind_stream()
        _check(lib().nnhip_scale_inplace(self.h, self._dev(x, self._torch.float32, "x"), x.numel(),
                                         alpha), "nnhip_scale_inplace")
        return x

    def act_scale(self, X):
        torch = self._torch
        K, M = X.shape
        s = self._empty((M,), torch.float32)
        self._bind_stream()
        _check(lib().nnhip_act_scale(self.h, self._dev(X, torch.float32, "X"), K, M, self._dev(s)),
               "nnhip_act_scale")
        return s

    def quantize_i8(self, x, scale, col_scale: bool = True):
        torch = self._torch
        rows, cols = x.shape
        out = self._empty((rows, (cols + 3) // 4), torch.int32)
        self._bind_stream()
        _check(lib().nnhip_quantize_i8(self.h, self._dev(x, torch.float32, "x"),
                                       self._dev(scale, torch.float32, "scale"), rows, cols,
                                       int(col_scale), self._dev(out)), "nnhip_quantize_i8")
        return out

    def unpack_i8(self, packed, cols: int):
        torch = self._torch
        rows = packed.shape[0]
        out = self._empty((rows, cols), torch.float32)
        self._bind_stream()
        _check(lib().nnhip_unpack_i8(self.h, self._dev(packed, torch.int32, "packed"), rows, cols,
                                     self._dev(out)), "nnhip_unpack_i8")
        return out

    def matmul_q_i8(self, wq, tau, xq, s, K: int, M: int):
        torch = self._torch
        N = wq.shape[0]
        Y = self._empty((N, M), torch.float32)
        self._bind_stream()
        _check(lib().nnhip_matmul_q_i8(self.h, self._dev(wq, torch.int32, "wq"),
                                       self._dev(tau, torch.float32, "tau"),
                                       self._dev(xq, torch.int32, "xq"),
                                       self._dev(s, torch.float32, "s"), N, K, M, self._dev(Y)),
               "nnhip_matmul_q_i8")
        return Y

    def matmul_q_i8_noalloc(self, wq, tau, xq, s, K: int, M: int, out):
        """nnhip_matmul_q_i8 with the library's static per-GPU scratch (no device allocation);
        `out` (N, M) float32 is required, so the call allocates nothing on the device."""
        torch = self._torch
        N = wq.shape[0]
        if tuple(out.shape) != (N, M):
            raise NNHipError(1, f"out has shape {tuple(out.shape)}, expected {(N, M)}")
        self._bind_stream()
        _check(lib().nnhip_matmul_q_i8_noalloc(self.h, self._dev(wq, torch.int32, "wq"),
                                               self._dev(tau, torch.float32, "tau"),
                                               self._dev(xq, torch.int32, "xq"),
                                               self._dev(s, torch.float32, "s"), N, K, M,
                                               self._dev(out, torch.float32, "out")),
               "nnhip_matmul_q_i8_noalloc")
        return out

    def matmul_q(self, wq, tau, B, K: int, out_f16: bool = False, out=None):
        """Y (N, M) = (tau o trit(wq)) . B; B f32 or f16 (K, M); Y f32, or f16 if out_f16."""
        torch = self._torch
        N, M = wq.shape[0], B.shape[1]
        if B.shape[0] != K:
            raise NNHipError(1, f"B has {B.shape[0]} rows, expected K={K}")
        ydt = torch.float16 if out_f16 else torch.float32
        Y = self._empty((N, M), ydt) if out is None else out
        self._dev(Y, ydt, "out")
        if tuple(Y.shape) != (N, M):
            raise NNHipError(1, f"out has shape {tuple(Y.shape)}, expected {(N, M)}")
        self._bind_stream()
        _check(lib().nnhip_matmul_q(self.h, self._dev(wq, torch.int32, "wq"), self._dev(tau, torch.float32, "tau"),
                                    self._dev(B, (torch.float32, torch.float16), "B"),
                                    1 if B.dtype == torch.float16 else 0, N, K, M, self._dev(Y),
                                    1 if out_f16 else 0), "nnhip_matmul_q")
        return Y

    def matmul_q_t(self, A, tau, B, M: int, out_f16: bool = False, out=None):
        """Y (M, N) = (tau o trit(A))^T . B, A (K, ceil(M/16)) packed with tau per stored row."""
        torch = self._torch
        K, N = A.shape[0], B.shape[1]
        if B.shape[0] != K:
            raise NNHipError(1, f"B has {B.shape[0]} rows, expected K={K}")
        ydt = torch.float16 if out_f16 else torch.float32
        Y = self._empty((M, N), ydt) if out is None else out
        self._dev(Y, ydt, "out")
        if tuple(Y.shape) != (M, N):
            raise NNHipError(1, f"out has shape {tuple(Y.shape)}, expected {(M, N)}")
        self._bind_stream()
        _check(lib().nnhip_matmul_q_t(self.h, self._dev(A, torch.int32, "A"), self._dev(tau, torch.float32, "tau"),
                                      self._dev(B, (torch.float32, torch.float16), "B"),
                                      1 if B.dtype == torch.float16 else 0, K, M, N, self._dev(Y),
                                      1 if out_f16 else 0), "nnhip_matmul_q_t")
        return Y

    def add_row_broadcast(self, Y, b):
        torch = self._torch
        N, M = Y.shape
        self._bind_stream()
        _check(lib().nnhip_add_row_broadcast(self.h, self._dev(Y, torch.float32, "Y"),
                                             self._dev(b, torch.float32, "b"), N, M),
               "nnhip_add_row_broadcast")
        return Y

    def rmsnorm(self, X, gamma, eps: float):
        torch = self._torch
        F, M = X.shape
        out = self._empty((F, M), torch.float32)
        self._bind_stream()
        _check(lib().nnhip_rmsnorm(self.h, self._dev(X, torch.float32, "X"),
                                   self._dev(gamma, torch.float32, "gamma"), eps, F, M,
                                   self._dev(out)), "nnhip_rmsnorm")
        return out

    def layernorm(self, X, gamma, beta, eps: float = 1e-5):
        """LayerNorm of each token (column) of X (F, M) with gain gamma (F) and shift beta (F):
        LayerNorm::forward (include/neuralnet.cpp/compute_layer_mlp.hpp:529-545), the SubLN norm type
        FeedForward takes by default. Returns (F, M) float32."""
        torch = self._torch
        F, M = X.shape
        if gamma.numel() != F or beta.numel() != F:
            raise NNHipError(1, f"layernorm: gamma and beta must hold F={F} values "
                                f"(got {gamma.numel()}, {beta.numel()})")
        out = self._empty((F, M), torch.float32)
        self._bind_stream()
        _check(lib().nnhip_layernorm(self.h, self._dev(X, torch.float32, "X"),
                                     self._dev(gamma, torch.float32, "gamma"),
                                     self._dev(beta, torch.float32, "beta"), eps, F, M,
                                     self._dev(out)), "nnhip_layernorm")
        return out

    # -- fast path
    def repack(self, wq, K: int):
        torch = self._torch
        N = wq.shape[0]
        rp = self._empty((repacked_bytes(N, K) // 4,), torch.int32)
        self._bind_stream()
        _check(lib().nnhip_repack_ternary(self.h, self._dev(wq, torch.int32, "wq"), N, K,
                                          self._dev(rp)), "nnhip_repack_ternary")
        return rp

    def unrepack(self, rp, N: int, K: int):
        torch = self._torch
        wq = self._empty((N, (K + 15) // 16), torch.int32)
        self._bind_stream()
        _check(lib().nnhip_unrepack_ternary(self.h, self._dev(rp, torch.int32, "rp"), N, K,
                                            self._dev(wq)), "nnhip_unrepack_ternary")
        return wq

    def _act_out(self, K: int, M: int):
        torch = self._torch
        xi = self._empty((M, kp(K)), torch.int8)
        s = self._empty((M,), torch.float32)
        rs = self._empty((M,), torch.int32)
        return xi, s, rs

    def act_quant_i8(self, X, want_container: bool = False, outs=None):
        """outs: optional preallocated (xi, s, rowsum) to write into."""
        torch = self._torch
        K, M = X.shape
        xi, s, rs = self._act_out(K, M) if outs is None else outs
        xq = self._empty((K, (M + 3) // 4), torch.int32) if want_container else None
        self._bind_stream()
        _check(lib().nnhip_act_quant_i8(self.h, self._dev(X, torch.float32, "X"), K, M,
                                        self._dev(xi), self._dev(s), self._dev(rs),
                                        self._dev(xq) if xq is not None else None),
               "nnhip_act_quant_i8")
        return (xi, s, rs, xq) if want_container else (xi, s, rs)

    def rmsnorm_quant_i8(self, X, gamma, eps: float, want_container: bool = False, outs=None):
        """outs: optional preallocated (xi, s, rowsum) to write into."""
        torch = self._torch
        F, M = X.shape
        xi, s, rs = self._act_out(F, M) if outs is None else outs
        xq = self._empty((F, (M + 3) // 4), torch.int32) if want_container else None
        self._bind_stream()
        _check(lib().nnhip_rmsnorm_quant_i8(self.h, self._dev(X, torch.float32, "X"),
                                            self._dev(gamma, torch.float32, "gamma"), eps, F, M,
                                            self._dev(xi), self._dev(s), self._dev(rs),
                                            self._dev(xq) if xq is not None else None),
               "nnhip_rmsnorm_quant_i8")
        return (xi, s, rs, xq) if want_container else (xi, s, rs)

    def act_from_container(self, xq, K: int, M: int):
        torch = self._torch
        xi, _, rs = self._act_out(K, M)
        self._bind_stream()
        _check(lib().nnhip_act_i8_from_container(self.h, self._dev(xq, torch.int32, "xq"), K, M,
                                                 self._dev(xi), self._dev(rs)),
               "nnhip_act_i8_from_container")
        return xi, rs

    def act_to_container(self, xi, K: int, M: int):
        torch = self._torch
        xq = self._empty((K, (M + 3) // 4), torch.int32)
        self._bind_stream()
        _check(lib().nnhip_act_i8_to_container(self.h, self._dev(xi, torch.int8, "xi"), K, M,
                                               self._dev(xq)), "nnhip_act_i8_to_container")
        return xq

    def ternary_matmul(self, rp, tau, xi, s, rowsum, N: int, K: int, M: int, bias=None, out=None):
        torch = self._torch
        Y = self._empty((N, M), torch.float32) if out is None else out
        self._bind_stream()
        _check(lib().nnhip_ternary_matmul(self.h, self._dev(rp, torch.int32, "rp"),
                                          self._dev(tau, torch.float32, "tau"),
                                          self._dev(xi, torch.int8, "xi"),
                                          self._dev(s, torch.float32, "s"),
                                          self._dev(rowsum, torch.int32, "rowsum"),
                                          self._dev(bias, torch.float32, "bias"), N, K, M,
                                          self._dev(Y, torch.float32, "Y")),
               "nnhip_ternary_matmul")
        return Y

    def ternary_matmul_f(self, rp, tau, B, N: int, K: int, out_f16: bool = False, out=None):
        """Float-activation product on repacked weights: (tau o trit) . B, B (K, M) f32 or f16."""
        torch = self._torch
        M = B.shape[1]
        Y = self._empty((N, M), torch.float16 if out_f16 else torch.float32) if out is None else out
        self._bind_stream()
        _check(lib().nnhip_ternary_matmul_f(self.h, self._dev(rp, torch.int32, "rp"), self._dev(tau, torch.float32, "tau"),
                                            self._dev(B, (torch.float32, torch.float16), "B"),
                                            int(B.dtype == torch.float16), N, K, M,
                                            self._dev(Y, (torch.float32, torch.float16), "Y"), int(out_f16)),
               "nnhip_ternary_matmul_f")
        return Y

    def stream_xor(self, src, out):
        """out (1 int32 word on the device) ^= xor of src's 32-bit words."""
        torch = self._torch
        self._bind_stream()
        _check(lib().nnhip_stream_xor(self.h, self._dev(src), src.numel() * src.element_size(),
                                      self._dev(out, torch.int32, "out")), "nnhip_stream_xor")
        return out

    def trit_transpose(self, A, M: int):
        """A (K, ceil(M/16)) packed -> At (M, ceil(K/16))."""
        torch = self._torch
        K = A.shape[0]
        At = self._empty((M, (K + 15) // 16), torch.int32)
        self._bind_stream()
        _check(lib().nnhip_trit_transpose(self.h, self._dev(A, torch.int32, "A"), K, M, self._dev(At)),
               "nnhip_trit_transpose")
        return At

    def ternary_matmul_t_f(self, rpT, tau, B, M: int, out_f16: bool = False, out=None):
        """(tau o trit(A))^T . B on rpT = repack(transpose(A)); B (K, N); returns (M, N)."""
        torch = self._torch
        K, N = B.shape
        Y = self._empty((M, N), torch.float16 if out_f16 else torch.float32) if out is None else out
        self._bind_stream()
        _check(lib().nnhip_ternary_matmul_t_f(self.h, self._dev(rpT, torch.int32, "rpT"),
                                              self._dev(tau, torch.float32, "tau"),
                                              self._dev(B, (torch.float32, torch.float16), "B"),
                                              int(B.dtype == torch.float16), K, M, N,
                                              self._dev(Y, (torch.float32, torch.float16), "Y"), int(out_f16)),
               "nnhip_ternary_matmul_t_f")
        return Y

    def ternary_matmul_add(self, rp, tau, xi, s, rowsum, N: int, K: int, M: int, res, bias=None, out=None,
                           tokens: bool = False):
        """Y = ternary_matmul(...) + res (res must not alias Y); with tokens, res and Y are (M, N)
        (nnhip_ternary_matmul_add_tokens, decode sizes)."""
        torch = self._torch
        Y = self._empty((M, N) if tokens else (N, M), torch.float32) if out is None else out
        self._bind_stream()
        entry = lib().nnhip_ternary_matmul_add_tokens if tokens else lib().nnhip_ternary_matmul_add
        _check(entry(self.h, self._dev(rp, torch.int32, "rp"),
                                              self._dev(tau, torch.float32, "tau"), self._dev(xi, torch.int8, "xi"),
                                              self._dev(s, torch.float32, "s"),
                                              self._dev(rowsum, torch.int32, "rowsum"),
                                              self._dev(bias, torch.float32, "bias"),
                                              self._dev(res, torch.float32, "res"), N, K, M,
                                              self._dev(Y, torch.float32, "Y")),
               "nnhip_ternary_matmul_add_tokens" if tokens else "nnhip_ternary_matmul_add")
        return Y

    def ternary_matmul_partial(self, rp, xi, N: int, K: int, M: int, slices: int, out=None):
        """Split-k integer partial sums part (slices, M, N) int32 of the ternary GEMV (no epilogue)."""
        torch = self._torch
        part = self._empty((slices, M, N), torch.int32) if out is None else out
        self._bind_stream()
        _check(lib().nnhip_ternary_matmul_partial(self.h, self._dev(rp, torch.int32, "rp"),
                                                  self._dev(xi, torch.int8, "xi"), N, K, M, slices,
                                                  self._dev(part, torch.int32, "part")),
               "nnhip_ternary_matmul_partial")
        return part

    def partial_residual_quant_i8(self, part, tau, s_in, rowsum_in, N: int, M: int, x_out, res=None, bias=None,
                                  gamma=None, eps: float = 0.0, outs=None, tokens: bool = False):
        """x_out = epilogue(sum of part) [+ bias] [+ res], then [RMSNorm(gamma) ->] int8: returns (xi, s, rowsum).
        With tokens, res and x_out are token-major (M, N)."""
        torch = self._torch
        xi, s, rs = self._act_out(N, M) if outs is None else outs
        self._bind_stream()
        entry = lib().nnhip_partial_residual_quant_i8_tokens if tokens else lib().nnhip_partial_residual_quant_i8
        _check(entry(self.h, self._dev(part, torch.int32, "part"), part.shape[0],
                                                     self._dev(tau, torch.float32, "tau"),
                                                     self._dev(s_in, torch.float32, "s_in"),
                                                     self._dev(rowsum_in, torch.int32, "rowsum_in"),
                                                     self._dev(bias, torch.float32, "bias"),
                                                     self._dev(res, torch.float32, "res"), N, M,
                                                     self._dev(x_out, torch.float32, "x_out"),
                                                     self._dev(gamma, torch.float32, "gamma"), eps,
                                                     self._dev(xi), self._dev(s), self._dev(rs)),
               "nnhip_partial_residual_quant_i8_tokens" if tokens else "nnhip_partial_residual_quant_i8")
        return xi, s, rs

    def ternary_matmul_n(self, problems, xi, s, rowsum, K: int, M: int, tokens: bool = False):
        """problems: list of (rp, tau, bias or None, N, out or None) sharing the input; returns the outputs
        ((N, M) each, or token-major (M, N) with tokens: nnhip_ternary_matmul_n_tokens)."""
        torch = self._torch
        n = len(problems)
        outs = [p[4] if p[4] is not None else self._empty((M, p[3]) if tokens else (p[3], M), torch.float32)
                for p in problems]
        rp = (_vp * n)(*[self._dev(p[0], torch.int32, "rp") for p in problems])
        tau = (_vp * n)(*[self._dev(p[1], torch.float32, "tau") for p in problems])
        bias = (_vp * n)(*[self._dev(p[2], torch.float32, "bias") for p in problems])
        Ns = (_sz * n)(*[p[3] for p in problems])
        Ys = (_vp * n)(*[self._dev(o, torch.float32, "Y") for o in outs])
        self._bind_stream()
        entry = lib().nnhip_ternary_matmul_n_tokens if tokens else lib().nnhip_ternary_matmul_n
        _check(entry(self.h, n, rp, tau, bias, Ns, Ys, self._dev(xi, torch.int8, "xi"),
                     self._dev(s, torch.float32, "s"), self._dev(rowsum, torch.int32, "rowsum"), K, M),
               "nnhip_ternary_matmul_n_tokens" if tokens else "nnhip_ternary_matmul_n")
        return outs

    def ffn_glu_i8_add(self, X, gamma, eps: float, F: int, rp1, tau1, b1, rp2, tau2, b2, res, act: int = ACT_SWIGLU,
                       out=None, gamma_sub=None, eps_sub: float = 1e-5):
        """res + ffn_glu_i8(X, ...) (res must not alias the output)."""
        torch = self._torch
        d, M = X.shape
        Y = self._empty((d, M), torch.float32) if out is None else out
        self._bind_stream()
        _check(lib().nnhip_ffn_glu_i8_add(self.h, self._dev(X, torch.float32, "X"),
                                          self._dev(gamma, torch.float32, "gamma"), eps, d, F, M, act,
                                          self._dev(rp1, torch.int32, "rp1"), self._dev(tau1, torch.float32, "tau1"),
                                          self._dev(b1, torch.float32, "b1"),
                                          self._dev(gamma_sub, torch.float32, "gamma_sub"), eps_sub,
                                          self._dev(rp2, torch.int32, "rp2"), self._dev(tau2, torch.float32, "tau2"),
                                          self._dev(b2, torch.float32, "b2"), self._dev(res, torch.float32, "res"),
                                          self._dev(Y, torch.float32, "Y")), "nnhip_ffn_glu_i8_add")
        return Y

    # -- batched decode step
    def attention_decode(self, q, k, v, H: int, Hkv: int, dk: int, pos, len_bound: int, k_cache, v_cache,
                         scale: float, cos=None, sin=None, out=None, tokens: bool = False):
        """q (H*dk, B), k/v (Hkv*dk, B), pos (B) int32 device, caches (B, max_len, Hkv*dk) updated in
        place (row pos[b]); cos/sin (max_len, dk/2) device tables or None. Returns out (H*dk, B).
        With tokens, q (B, H*dk), k/v (B, Hkv*dk) and out (B, H*dk) (nnhip_attention_decode_tokens).
        float16 caches (compute = F16) run the _h entry points; both caches have one dtype."""
        torch = self._torch
        B = q.shape[0] if tokens else q.shape[1]
        max_len = k_cache.shape[1]
        ct = self._cache_dtype(k_cache, v_cache)
        if out is None:
            out = self._empty((B, H * dk) if tokens else (H * dk, B), torch.float32)
        self._bind_stream()
        name = ("nnhip_attention_decode_tokens" if tokens else "nnhip_attention_decode") + \
            ("_h" if ct == torch.float16 else "")
        _check(getattr(lib(), name)(
            self.h, self._dev(q, torch.float32, "q"), self._dev(k, torch.float32, "k"),
            self._dev(v, torch.float32, "v"), B, H, Hkv, dk, self._dev(pos, torch.int32, "pos"), len_bound,
            self._dev(cos, torch.float32, "cos"), self._dev(sin, torch.float32, "sin"),
            self._dev(k_cache, ct, "k_cache"), self._dev(v_cache, ct, "v_cache"), max_len,
            scale, self._dev(out, torch.float32, "out")), name)
        return out

    def _cache_dtype(self, k_cache, v_cache):
        """The caches' element type: float32, or float16 under compute = F16 (both alike)."""
        torch = self._torch
        if k_cache.dtype != v_cache.dtype or k_cache.dtype not in (torch.float32, torch.float16):
            raise NNHipError(1, f"caches must both be float32 or both float16 (got {k_cache.dtype}, {v_cache.dtype})")
        return k_cache.dtype

    def kv_cache_fill(self, k, v, B: int, T: int, Hkv: int, dk: int, pos0: int, k_cache, v_cache, cos=None, sin=None):
        """Append T tokens of each of B sequences (k / v (Hkv*dk, B*T)) to the caches at rows pos0 + t
        (float16 caches: nnhip_kv_cache_fill_h)."""
        torch = self._torch
        ct = self._cache_dtype(k_cache, v_cache)
        name = "nnhip_kv_cache_fill" + ("_h" if ct == torch.float16 else "")
        self._bind_stream()
        _check(getattr(lib(), name)(self.h, self._dev(k, torch.float32, "k"), self._dev(v, torch.float32, "v"),
                                    B, T, Hkv, dk, pos0, self._dev(cos, torch.float32, "cos"),
                                    self._dev(sin, torch.float32, "sin"), self._dev(k_cache, ct, "k_cache"),
                                    self._dev(v_cache, ct, "v_cache"), k_cache.shape[1]), name)

    def attention_prefill(self, q, k_cache, v_cache, B: int, T: int, H: int, Hkv: int, dk: int, pos0: int,
                          scale: float, cos=None, sin=None, out=None):
        """Causal attention of T tokens per sequence (q (H*dk, B*T)) over caches holding rows [0, pos0 + T)."""
        torch = self._torch
        ct = self._cache_dtype(k_cache, v_cache)
        name = "nnhip_attention_prefill" + ("_h" if ct == torch.float16 else "")
        Y = out if out is not None else self._empty((H * dk, B * T), torch.float32)
        self._bind_stream()
        _check(getattr(lib(), name)(self.h, self._dev(q, torch.float32, "q"), self._dev(k_cache, ct, "k_cache"),
                                    self._dev(v_cache, ct, "v_cache"), B, T, H, Hkv, dk, pos0,
                                    self._dev(cos, torch.float32, "cos"), self._dev(sin, torch.float32, "sin"),
                                    k_cache.shape[1], scale, self._dev(Y, torch.float32, "out")), name)
        return Y

    def copy_columns(self, src, col0: int, stride: int, n: int, out=None):
        """dst (rows, n): column j = src column col0 + j * stride."""
        torch = self._torch
        rows, cols = src.shape
        Y = out if out is not None else self._empty((rows, n), torch.float32)
        self._bind_stream()
        _check(lib().nnhip_copy_columns(self.h, self._dev(src, torch.float32, "src"), rows, cols, col0, stride, n,
                                        self._dev(Y, torch.float32, "dst")), "nnhip_copy_columns")
        return Y

    def to_f16(self, x, out=None):
        """f32 -> binary16 (round to nearest even), as a torch.float16 tensor."""
        torch = self._torch
        Y = out if out is not None else self._empty(tuple(x.shape), torch.float16)
        self._bind_stream()
        _check(lib().nnhip_convert_f32_f16(self.h, self._dev(x, torch.float32, "x"), x.numel(),
                                           self._dev(Y, torch.float16, "out")), "nnhip_convert_f32_f16")
        return Y

    def to_f32(self, x, out=None):
        """binary16 -> f32 (exact)."""
        torch = self._torch
        Y = out if out is not None else self._empty(tuple(x.shape), torch.float32)
        self._bind_stream()
        _check(lib().nnhip_convert_f16_f32(self.h, self._dev(x, torch.float16, "x"), x.numel(),
                                           self._dev(Y, torch.float32, "out")), "nnhip_convert_f16_f32")
        return Y

    def add(self, x, y, out=None):
        torch = self._torch
        if out is None:
            out = self._empty(tuple(x.shape), torch.float32)
        self._bind_stream()
        _check(lib().nnhip_add(self.h, self._dev(x, torch.float32, "x"), self._dev(y, torch.float32, "y"),
                               x.numel(), self._dev(out, torch.float32, "out")), "nnhip_add")
        return out

    def embedding_gather(self, table, ids, out=None, tokens: bool = False):
        """table (V, d), ids (B) int32 device -> (d, B), or (B, d) with tokens."""
        torch = self._torch
        V, d = table.shape
        B = ids.shape[0]
        if out is None:
            out = self._empty((B, d) if tokens else (d, B), torch.float32)
        self._bind_stream()
        entry = lib().nnhip_embedding_gather_tokens if tokens else lib().nnhip_embedding_gather
        _check(entry(self.h, self._dev(table, torch.float32, "table"),
                                            self._dev(ids, torch.int32, "ids"), V, d, B,
                                            self._dev(out, torch.float32, "out")),
               "nnhip_embedding_gather_tokens" if tokens else "nnhip_embedding_gather")
        return out

    def argmax_cols(self, logits, out=None):
        """logits (V, B) -> (B) int32 greedy token ids."""
        torch = self._torch
        V, B = logits.shape
        if out is None:
            out = self._empty((B,), torch.int32)
        self._bind_stream()
        _check(lib().nnhip_argmax_cols(self.h, self._dev(logits, torch.float32, "logits"), V, B,
                                       self._dev(out, torch.int32, "out")), "nnhip_argmax_cols")
        return out

    def argmax_rows(self, logits, out=None, pos=None):
        """token-major logits (B, V) -> (B) int32 greedy token ids; pos (B) int32, when given, is
        advanced by one in the same launch."""
        torch = self._torch
        B, V = logits.shape
        if out is None:
            out = self._empty((B,), torch.int32)
        if pos is not None and tuple(pos.shape) != (B,):
            raise NNHipError(1, f"pos must have shape ({B},)")
        self._bind_stream()
        _check(lib().nnhip_argmax_rows(self.h, self._dev(logits, torch.float32, "logits"), V, B,
                                       self._dev(out, torch.int32, "out"), self._dev(pos, torch.int32, "pos")),
               "nnhip_argmax_rows")
        return out

    # -- paged KV cache, adjusted logits
    def _arg(self, t, dtype, shape, name):
        """The device address of t (None: null) after its checks: this context's device, contiguous, type, shape."""
        if t is None:
            return None
        if t.get_device() == self.device and t.dtype is dtype and t.shape == shape and t.is_contiguous():
            return t.data_ptr()
        if t.get_device() != self.device:
            raise NNHipError(1, f"{name} is on {t.device}, the context on {self._device}")
        if t.dtype is not dtype:
            raise NNHipError(1, f"{name} has dtype {t.dtype}, expected {dtype}")
        if t.shape != shape:
            raise NNHipError(1, f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
        raise NNHipError(1, f"{name} must be contiguous")

    def _rope(self, cos, sin, dk: int, limit: int = 0):
        """Addresses and rows of the rope tables (None, None, limit without)."""
        if cos is None and sin is None:
            if limit < 0:
                raise NNHipError(1, "limit must be at least 0")
            return None, None, limit
        if limit:
            raise NNHipError(1, "limit goes without tables, whose rows bound the positions")
        if cos is None or sin is None:
            raise NNHipError(1, "cos and sin go together")
        shape = (cos.shape[0], dk // 2)
        f32 = self._torch.float32
        return self._arg(cos, f32, shape, "cos"), self._arg(sin, f32, shape, "sin"), shape[0]

    def _packed(self, cache, cu, pos0):
        """The sequences of a packed call (cu (B + 1), pos0 (B) or None): B and both addresses."""
        if cache.device != self._device:
            raise NNHipError(1, f"the cache is on {cache.device}, the context on {self._device}")
        B, i32 = cu.shape[0] - 1, self._torch.int32
        if B < 0 or B > cache.rows:
            raise NNHipError(1, f"cu must hold B + 1 offsets, B at most the page table's {cache.rows} rows")
        return B, self._arg(cu, i32, (B + 1,), "cu"), self._arg(pos0, i32, (B,), "pos0")

    def kv_pages_fill(self, cache, k, v, cu, pos0=None, cos=None, sin=None, limit: int = 0) -> None:
        """The keys and values k / v (Hkv*dk, M) of packed prompts (sequence b: columns cu[b] .. cu[b+1] - 1,
        positions pos0[b] on) rotated into the pages of cache, a KVPages or a KVPagesI8 (which holds them quantized).
        Not written: positions at or past the tables' rows, or without tables at or past limit (0: the page table's end)."""
        B, cu_p, pos0_p = self._packed(cache, cu, pos0)
        f32, M = self._torch.float32, k.shape[-1]
        cs, sn, rows = self._rope(cos, sin, cache.dk, limit)
        shape = (cache.Hkv * cache.dk, M)
        self._bind_stream()
        fn = "nnhip_kv_pages_fill_i8" if isinstance(cache, KVPagesI8) else "nnhip_kv_pages_fill"
        _check(getattr(lib(), fn)(self.h, cache.ref, self._arg(k, f32, shape, "k"), self._arg(v, f32, shape, "v"),
                                  M, cu_p, pos0_p, B, cs, sn, rows), fn)

    def kv_pages_read(self, cache, cu, M: int, pos0=None, k=None, v=None):
        """The values that cache, a KVPagesI8, holds: k, v (Hkv*dk, M) get in columns cu[b] .. cu[b+1] - 1 those of sequence
        b's positions pos0[b] on. Returns k, v."""
        if not isinstance(cache, KVPagesI8):
            raise NNHipError(1, "kv_pages_read takes a KVPagesI8 (the pools of a KVPages are its values)")
        B, cu_p, pos0_p = self._packed(cache, cu, pos0)
        f32, shape = self._torch.float32, (cache.Hkv * cache.dk, M)
        k = self._empty(shape, f32) if k is None else k
        v = self._empty(shape, f32) if v is None else v
        self._bind_stream()
        _check(lib().nnhip_kv_pages_read_i8(self.h, cache.ref, M, cu_p, pos0_p, B, self._arg(k, f32, shape, "k"),
                                            self._arg(v, f32, shape, "v")), "nnhip_kv_pages_read_i8")
        return k, v

    def attention_pages_decode(self, cache, q, k, v, H: int, pos, len_bound: int, scale: float, cos=None, sin=None,
                               softcap: float = 0.0, slopes=None, out=None, tokens: bool = False):
        """Attention of one new token per sequence over the pages of cache (a KVPages or KVPagesI8, whose table has B rows),
        which also get its key and value (k and v None, over a KVPagesI8: it holds position pos already): q (H*dk, B), k / v (Hkv*dk, B), or token-major (B, ...) with tokens;
        pos (B) int32 device, below 0 for an empty slot. softcap > 0 caps the scores, slopes (H) bias them by
        distance. Returns out like q."""
        if cache.device != self._device:
            raise NNHipError(1, f"the cache is on {cache.device}, the context on {self._device}")
        f32, dk, B = self._torch.float32, cache.dk, pos.shape[0]
        if B > cache.rows:
            raise NNHipError(1, f"{B} sequences, the page table has {cache.rows} rows")
        qs, ks = ((B, H * dk), (B, cache.Hkv * dk)) if tokens else ((H * dk, B), (cache.Hkv * dk, B))
        if out is None:
            out = self._empty(qs, f32)
        cs, sn, rows = self._rope(cos, sin, dk)
        self._bind_stream()
        fn = "nnhip_attention_pages_decode_i8" if isinstance(cache, KVPagesI8) else "nnhip_attention_pages_decode"
        _check(getattr(lib(), fn)(
            self.h, cache.ref, self._arg(q, f32, qs, "q"), self._arg(k, f32, ks, "k"), self._arg(v, f32, ks, "v"), B, H,
            self._arg(pos, self._torch.int32, (B,), "pos"), len_bound, cs, sn, rows, scale, softcap,
            self._arg(slopes, f32, (H,), "slopes"), int(tokens), self._arg(out, f32, qs, "out")), fn)
        return out

    def attention_pages_prefill(self, cache, q, cu, t_bound: int, H: int, scale: float, pos0=None, cos=None, sin=None,
                                softcap: float = 0.0, slopes=None, prefix=None, out=None, distance: bool = False,
                                limit: int = 0):
        """Attention of packed prompts q (H*dk, M) (sequence b: columns cu[b] .. cu[b+1] - 1, at most t_bound <= M of
        them, positions pos0[b] on) over the pages of cache, which hold all their positions: causal, and bidirectional
        over the first prefix[b] positions (prefix (B) int32, or None). slopes (H) bias the scores by
        slopes[h] * (j - i), or with distance by -slopes[h] * |j - i|: for keys ahead of the query, inside a prefix,
        these differ. A sequence with positions at or past the tables' rows, or without tables at or past limit (0: the
        page table's end), gets NaN. Returns out (H*dk, M)."""
        B, cu_p, pos0_p = self._packed(cache, cu, pos0)
        f32, M = self._torch.float32, q.shape[-1]
        shape = (H * cache.dk, M)
        if out is None:
            out = self._empty(shape, f32)
        cs, sn, rows = self._rope(cos, sin, cache.dk, limit)
        self._bind_stream()
        more = ()
        if isinstance(cache, KVPagesI8):
            fn, more = "nnhip_attention_pages_prefill_i8", (int(distance),)
        else:
            fn = "nnhip_attention_pages_prefill_distance" if distance else "nnhip_attention_pages_prefill"
        _check(getattr(lib(), fn)(
            self.h, cache.ref, self._arg(q, f32, shape, "q"), M, cu_p, pos0_p, B, t_bound, H, cs, sn, rows, scale,
            softcap, self._arg(slopes, f32, (H,), "slopes"), self._arg(prefix, self._torch.int32, (B,), "prefix"),
            *more, self._arg(out, f32, shape, "out")), fn)
        return out

    def qk_norm_rope(self, q, k, dk: int, eps: float, gamma_q=None, gamma_k=None, pos=None, cos=None, sin=None,
                     q_out=None, k_out=None, tokens: bool = False):
        """RMSNorm of every head (dk elements, gains gamma_q, gamma_k (dk) or None) of q (H*dk, M) and k (Hkv*dk, M), or
        token-major with tokens, and their rotation at pos (M) int32 device (a token below 0 stays). q or k may be
        None; q_out and k_out, made when not given, may be q and k. Returns them."""
        torch = self._torch
        f32 = torch.float32
        if q is None and k is None:
            raise NNHipError(1, "q or k must be given")
        M = (k if q is None else q).shape[0 if tokens else 1]

        def one(x, out, name):
            if x is None:
                if out is not None:
                    raise NNHipError(1, f"{name}_out without {name}")
                return 0, None, None, None
            rows = x.shape[1 if tokens else 0]
            if rows % dk:
                raise NNHipError(1, f"{name} has {rows} features, heads of {dk}")
            shape = (M, rows) if tokens else (rows, M)
            if out is None:
                out = self._empty(shape, f32)
            return rows // dk, self._arg(x, f32, shape, name), self._arg(out, f32, shape, name + "_out"), out

        H, q_p, qo_p, q_out = one(q, q_out, "q")
        Hkv, k_p, ko_p, k_out = one(k, k_out, "k")
        cs, sn, rows = self._rope(cos, sin, dk)
        if cos is not None and rows == 0:
            raise NNHipError(1, "the rope tables are empty")
        self._bind_stream()
        _check(lib().nnhip_qk_norm_rope(
            self.h, q_p, k_p, M, H, Hkv, dk, self._arg(gamma_q, f32, (dk,), "gamma_q"),
            self._arg(gamma_k, f32, (dk,), "gamma_k"), eps, self._arg(pos, torch.int32, (M,), "pos"), cs, sn, rows,
            int(tokens), qo_p, ko_p), "nnhip_qk_norm_rope")
        return q_out, k_out

    def _table(self, table):
        """The address and shape of a page table."""
        if table.dim() != 2:
            raise NNHipError(1, f"the page table must be (B, pages), not {tuple(table.shape)}")
        return self._arg(table, self._torch.int32, table.shape, "table"), table.shape

    def _places(self, pos, slots):
        """The capacity M of per-token outputs and their addresses."""
        i32 = self._torch.int32
        M = 0 if pos is None and slots is None else (slots if pos is None else pos).shape[0]
        return M, self._arg(pos, i32, (M,), "pos"), self._arg(slots, i32, (M,), "slots")

    def pages_assign(self, table, page_size: int, free_pages, free_count, lens, add, cu=None, pos0=None, pos=None, slots=None):
        """Pages for add[b] new tokens of each sequence from the list free_pages (num_pages) with free_count (1) entries, into
        its row of table (B, pages), behind the pages of its lens[b] positions; lens moves on (all int32 device tensors). cu
        (B + 1): offsets of the tokens that got their places; pos0 (B): the first one's position, -1 for none; pos, slots
        (M), when given: every token's position and slot, -1 behind the last. Returns cu, pos0."""
        i32, (table_p, (B, width)) = self._torch.int32, self._table(table)
        cu = self._empty((B + 1,), i32) if cu is None else cu
        pos0 = self._empty((B,), i32) if pos0 is None else pos0
        num_pages = free_pages.shape[0]
        M, pos_p, slots_p = self._places(pos, slots)
        self._bind_stream()
        _check(lib().nnhip_pages_assign(
            self.h, table_p, width, page_size, num_pages, B,
            self._arg(free_pages, i32, (num_pages,), "free_pages"), self._arg(free_count, i32, (1,), "free_count"),
            self._arg(lens, i32, (B,), "lens"), self._arg(add, i32, (B,), "add"), self._arg(cu, i32, (B + 1,), "cu"),
            self._arg(pos0, i32, (B,), "pos0"), M, pos_p, slots_p), "nnhip_pages_assign")
        return cu, pos0

    def pages_slots(self, table, page_size: int, num_pages: int, cu, pos0=None, pos=None, slots=None):
        """Positions pos (M) and slots (M) of packed tokens (cu (B + 1), pos0 (B) or None), either of which may be None."""
        i32, B, (table_p, (table_rows, width)) = self._torch.int32, cu.shape[0] - 1, self._table(table)
        if B < 0 or B > table_rows:
            raise NNHipError(1, f"cu must hold B + 1 offsets, B at most the page table's {table_rows} rows")
        M, pos_p, slots_p = self._places(pos, slots)
        self._bind_stream()
        _check(lib().nnhip_pages_slots(
            self.h, table_p, width, page_size, num_pages,
            self._arg(cu, i32, (B + 1,), "cu"), self._arg(pos0, i32, (B,), "pos0"), B, M, pos_p, slots_p),
            "nnhip_pages_slots")
        return pos, slots

    def pages_release(self, table, page_size: int, free_pages, free_count, lens, keep) -> None:
        """Sequence b keeps its first keep[b] positions (0: none): lens[b] becomes that, and the pages behind go back to
        the list, so that a release of what pages_assign has just given leaves the list as it was."""
        i32, (table_p, (B, width)) = self._torch.int32, self._table(table)
        num_pages = free_pages.shape[0]
        self._bind_stream()
        _check(lib().nnhip_pages_release(
            self.h, table_p, width, page_size, num_pages, B,
            self._arg(free_pages, i32, (num_pages,), "free_pages"), self._arg(free_count, i32, (1,), "free_count"),
            self._arg(lens, i32, (B,), "lens"), self._arg(keep, i32, (B,), "keep")), "nnhip_pages_release")

    def attention_pages_workspace_bytes(self, B: int, H: int, Hkv: int, dk: int, len_bound: int) -> int:
        return int(lib().nnhip_attention_pages_workspace_bytes(self.h, B, H, Hkv, dk, len_bound))

    def logits_workspace_bytes(self, V: int, B: int) -> int:
        return int(lib().nnhip_logits_workspace_bytes(self.h, V, B))

    def logits_adjust_rows(self, logits, rules=None, ids=None, out=None, pos=None):
        """Token-major logits (B, V) adjusted by rules (a LogitRules, or None) and the greedy choice among the
        allowed tokens into ids (B) int32 (-1: nothing is allowed), made when neither ids nor out is given. out
        (B, V), when given, gets the adjusted logits (it may be logits itself); pos (B) int32 is advanced by one
        after a choice. Returns ids."""
        B, V = logits.shape
        f32, i32 = self._torch.float32, self._torch.int32
        if rules is not None:
            if rules.V != V or rules.rows not in (None, B):
                raise NNHipError(1, f"rules for {(rules.rows, rules.V)}, logits of {(B, V)}")
            if rules.device not in (None, self._device):
                raise NNHipError(1, f"the rules are on {rules.device}, the context on {self._device}")
        if ids is None and out is None:
            ids = self._empty((B,), i32)
        self._bind_stream()
        _check(lib().nnhip_logits_adjust_rows(
            self.h, self._arg(logits, f32, (B, V), "logits"), V, B, None if rules is None else rules.ref,
            self._arg(out, f32, (B, V), "out"), self._arg(ids, i32, (B,), "ids"), self._arg(pos, i32, (B,), "pos")),
            "nnhip_logits_adjust_rows")
        return ids

    def token_counts_add(self, ids, cu, counts):
        """counts (B, V) int32 [b, ids[m]] += 1 for the tokens m of each packed sequence (cu (B + 1))."""
        i32 = self._torch.int32
        B, V = counts.shape
        M = ids.shape[0]
        self._bind_stream()
        _check(lib().nnhip_token_counts_add(self.h, self._arg(ids, i32, (M,), "ids"), M,
                                            self._arg(cu, i32, (B + 1,), "cu"), B, V,
                                            self._arg(counts, i32, (B, V), "counts")), "nnhip_token_counts_add")
        return counts

    # -- gated feed-forward block
    def glu(self, Y1, act: int = ACT_SWIGLU):
        """Y1 (2F, M): gate rows then up rows -> h (F, M)."""
        torch = self._torch
        F, M = Y1.shape[0] // 2, Y1.shape[1]
        h = self._empty((F, M), torch.float32)
        self._bind_stream()
        _check(lib().nnhip_glu(self.h, self._dev(Y1, torch.float32, "Y1"), F, M, act, self._dev(h)), "nnhip_glu")
        return h

    def glu_interleave(self, wq, tau, bias, F: int, K: int):
        """fc1 container (2F, ceil(K/16)) + tau/bias (2F) -> interleaved (wq, tau, bias)."""
        torch = self._torch
        rows = glu_rows(F)
        wo = self._empty((rows, (K + 15) // 16), torch.int32)
        to = self._empty((rows,), torch.float32)
        bo = self._empty((rows,), torch.float32) if bias is not None else None
        self._bind_stream()
        _check(lib().nnhip_glu_interleave(self.h, self._dev(wq, torch.int32, "wq"), self._dev(tau, torch.float32, "tau"),
                                          self._dev(bias, torch.float32, "bias"), F, K, self._dev(wo), self._dev(to),
                                          self._dev(bo) if bo is not None else None), "nnhip_glu_interleave")
        return wo, to, bo

    def ternary_matmul_glu_tokens(self, rp, tau, xi, s, rowsum, F: int, K: int, M: int, act: int = ACT_SWIGLU,
                                  bias=None, out=None):
        """ternary_matmul_glu with h token-major (M, F) (decode sizes)."""
        torch = self._torch
        h = self._empty((M, F), torch.float32) if out is None else out
        self._bind_stream()
        _check(lib().nnhip_ternary_matmul_glu_tokens(self.h, self._dev(rp, torch.int32, "rp"),
                                                     self._dev(tau, torch.float32, "tau"),
                                                     self._dev(xi, torch.int8, "xi"), self._dev(s, torch.float32, "s"),
                                                     self._dev(rowsum, torch.int32, "rowsum"),
                                                     self._dev(bias, torch.float32, "bias"), F, K, M, act,
                                                     self._dev(h, torch.float32, "h")),
               "nnhip_ternary_matmul_glu_tokens")
        return h

    def rmsnorm_quant_i8_tokens(self, X, gamma, eps: float, outs=None):
        """[RMSNorm (gamma, or None) ->] absmax -> int8 of a token-major X (M, K); returns (xi, s, rowsum)."""
        torch = self._torch
        M, K = X.shape
        if outs is None:
            outs = (self._empty((M, kp(K)), torch.int8), self._empty((M,), torch.float32),
                    self._empty((M,), torch.int32))
        xi, s, rs = outs
        self._bind_stream()
        _check(lib().nnhip_rmsnorm_quant_i8_tokens(self.h, self._dev(X, torch.float32, "X"),
                                                   self._dev(gamma, torch.float32, "gamma"), eps, K, M,
                                                   self._dev(xi, torch.int8, "xi"), self._dev(s, torch.float32, "s"),
                                                   self._dev(rs, torch.int32, "rowsum")),
               "nnhip_rmsnorm_quant_i8_tokens")
        return outs

    def embedding_rmsnorm_quant_i8_tokens(self, table, ids, gamma, eps: float, out=None, outs=None):
        """Rows ids[b] of table (V, d) into out (B, d) and their [RMSNorm (gamma, or None) ->] absmax
        -> int8 in the same launch; returns (out, (xi, s, rowsum))."""
        torch = self._torch
        V, d = table.shape
        B = ids.shape[0]
        if out is None:
            out = self._empty((B, d), torch.float32)
        if outs is None:
            outs = (self._empty((B, kp(d)), torch.int8), self._empty((B,), torch.float32),
                    self._empty((B,), torch.int32))
        xi, s, rs = outs
        self._bind_stream()
        _check(lib().nnhip_embedding_rmsnorm_quant_i8_tokens(
            self.h, self._dev(table, torch.float32, "table"), self._dev(ids, torch.int32, "ids"), V, d, B,
            self._dev(gamma, torch.float32, "gamma"), eps, self._dev(out, torch.float32, "out"),
            self._dev(xi, torch.int8, "xi"), self._dev(s, torch.float32, "s"), self._dev(rs, torch.int32, "rowsum")),
            "nnhip_embedding_rmsnorm_quant_i8_tokens")
        return out, outs

    def ternary_matmul_glu(self, rp, tau, xi, s, rowsum, F: int, K: int, M: int, act: int = ACT_SWIGLU,
                           bias=None, out=None):
        torch = self._torch
        h = self._empty((F, M), torch.float32) if out is None else out
        self._bind_stream()
        _check(lib().nnhip_ternary_matmul_glu(self.h, self._dev(rp, torch.int32, "rp"),
                                              self._dev(tau, torch.float32, "tau"), self._dev(xi, torch.int8, "xi"),
                                              self._dev(s, torch.float32, "s"),
                                              self._dev(rowsum, torch.int32, "rowsum"),
                                              self._dev(bias, torch.float32, "bias"), F, K, M, act,
                                              self._dev(h, torch.float32, "h")), "nnhip_ternary_matmul_glu")
        return h

    def ffn_glu_i8(self, X, gamma, eps: float, F: int, rp1, tau1, b1, rp2, tau2, b2, act: int = ACT_SWIGLU,
                   out=None, gamma_sub=None, eps_sub: float = 1e-5):
        """Gated FFN block on X (d, M): [RMSNorm] -> int8 -> fc1 (interleaved) -> act -> [SubLN RMSNorm
        (gamma_sub, eps_sub)] -> int8 -> fc2."""
        torch = self._torch
        d, M = X.shape
        Y = self._empty((d, M), torch.float32) if out is None else out
        self._bind_stream()
        _check(lib().nnhip_ffn_glu_i8(self.h, self._dev(X, torch.float32, "X"), self._dev(gamma, torch.float32, "gamma"),
                                      eps, d, F, M, act, self._dev(rp1, torch.int32, "rp1"),
                                      self._dev(tau1, torch.float32, "tau1"), self._dev(b1, torch.float32, "b1"),
                                      self._dev(gamma_sub, torch.float32, "gamma_sub"), eps_sub,
                                      self._dev(rp2, torch.int32, "rp2"), self._dev(tau2, torch.float32, "tau2"),
                                      self._dev(b2, torch.float32, "b2"), self._dev(Y, torch.float32, "Y")),
               "nnhip_ffn_glu_i8")
        return Y

    def group_create(self, problems):
        """problems: list of dicts with rp, tau, xi, s, rowsum, bias (or None), y, N, K, M."""
        arr = (GemvDesc * len(problems))()
        for i, p in enumerate(problems):
            arr[i] = GemvDesc(p["rp"].data_ptr(), p["tau"].data_ptr(), p["xi"].data_ptr(),
                              p["s"].data_ptr(), p["rowsum"].data_ptr(),
                              p["bias"].data_ptr() if p.get("bias") is not None else None,
                              p["y"].data_ptr(), p["N"], p["K"], p["M"])
        h = _vp()
        self._bind_stream()
        _check(lib().nnhip_group_create(self.h, arr, len(problems), ctypes.byref(h)),
               "nnhip_group_create")
        return h

    def group_run(self, h) -> None:
        self._bind_stream()
        _check(lib().nnhip_group_run(self.h, h), "nnhip_group_run")

    def group_destroy(self, h) -> None:
        self._bind_stream()
        _check(lib().nnhip_group_destroy(self.h, h), "nnhip_group_destroy")

    def group_info(self, h) -> dict:
        """What nnhip_group_create chose: {"lds": True (every launch stages its activations in LDS),
        False (register variant only) or "mixed", "waves": int, "lds_bytes": int}."""
        v, w, b = ctypes.c_int(0), _sz(0), _sz(0)
        _check(lib().nnhip_group_info(h, ctypes.byref(v), ctypes.byref(w), ctypes.byref(b)), "nnhip_group_info")
        lds = {0: False, 1: True}.get(v.value, "mixed")
        return {"lds": lds, "waves": int(w.value), "lds_bytes": int(b.value)}

    def gemv_grid_waves(self, items: int) -> int:
        return int(lib().nnhip_gemv_grid_waves(self.h, items))
