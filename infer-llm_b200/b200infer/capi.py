"""ctypes binding of the single-op C ABI (include/b200_infer.h).

Tensor arguments are torch tensors on the current CUDA device (contiguous,
float32 / int32); the functions pass their data pointers and the current
torch stream to the library. Shapes follow the reference's node semantics:
``mul_mat(w (N,K), x (M,K)) -> (M,N)`` is OpFactory::mul_mat(w, x).
"""
from __future__ import annotations

import ctypes as C
import functools
import os
import struct
import subprocess

PKG_DIR = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))  # infer-llm_b200/
REPO_DIR = os.path.dirname(PKG_DIR)
lib_path = os.path.join(PKG_DIR, "lib", "libb200infer.so")
HEADER = os.path.join(REPO_DIR, "include", "b200_infer.h")

PREC_FFMA, PREC_TF32 = 0, 1
STATUS = {0: "ok", 1: "invalid argument", 2: "not supported", 3: "out of range", 4: "CUDA error",
          5: "out of memory", 6: "device-side check failed", 7: "device wait timed out",
          8: "NaN or +inf logits"}


class B200Error(RuntimeError):
    def __init__(self, fn: str, status: int):
        super().__init__(f"{fn} failed: {STATUS.get(status, status)} ({status})")
        self.status = status


def build(jobs: int = 8) -> str:
    """Compile libb200infer.so in-tree for sm_100a (nvcc cross-compiles without a GPU)."""
    subprocess.run(["make", "-s", "-C", PKG_DIR, f"-j{jobs}"], check=True)
    return lib_path


_lib = None
_vp, _i64, _i32, _f32, _sz = C.c_void_p, C.c_int64, C.c_int32, C.c_float, C.c_size_t

_SIGS = {
    "b200_status_string": ([C.c_int], C.c_char_p),
    "b200_device_supported": ([C.c_int], C.c_int),
    "b200_mul_mat": ([_vp, _vp, _vp, _i64, _i64, _i64, C.c_int, _vp], C.c_int),
    "b200_mul_mat_ws": ([_vp, _vp, _vp, _i64, _i64, _i64, _i32, _vp, _sz, _vp], C.c_int),
    "b200_mul_mat_workspace_bytes": ([_i64, _i64, _i64, _i32], _sz),
    "b200_rms_norm": ([_vp, _vp, _vp, _i64, _i64, _f32, _vp], C.c_int),
    "b200_rope": ([_vp, _vp, _vp, _i64, _vp, _i64, _i64, _i64, _vp, _vp], C.c_int),
    "b200_qk_norm_rope": ([_vp, _i64, _vp, _i64, _vp, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _vp, _i64,
                           _i64, _i64, _i64, _i64, _i64, _f32, _vp, _vp], C.c_int),
    "b200_rope_freqs": ([_f32, _i64, _vp], None),
    "b200_flash_attn": ([_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _f32, _i64, _i64, _i64,
                         _i64, _vp, _sz, _vp], C.c_int),
    "b200_flash_attn_ex": ([_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _f32, _i64, _i64, _i64,
                            _i64, _vp, _sz, _vp, _i32], C.c_int),
    "b200_flash_attn_workspace_bytes": ([_i64, _i64, _i64, _i64, _i64], _sz),
    "b200_silu": ([_vp, _vp, _i64, _vp], C.c_int),
    "b200_mul": ([_vp, _vp, _vp, _i64, _vp], C.c_int),
    "b200_add": ([_vp, _vp, _vp, _i64, _vp], C.c_int),
    "b200_swiglu": ([_vp, _vp, _vp, _i64, _vp], C.c_int),
    "b200_get_rows": ([_vp, _vp, _vp, _i64, _i64, _i64, _vp, _vp], C.c_int),
    "b200_copy": ([_vp, _vp, _sz, _vp], C.c_int),
    "b200_argmax": ([_vp, _i64, _vp, _vp, _sz, _vp, _vp], C.c_int),
    "b200_argmax_workspace_bytes": ([_i64], _sz),
    "b200_argmax_noalloc": ([_vp, _i64, _vp, _vp, _vp], C.c_int),
    "b200_engine_create": ([_vp, C.c_int, _vp], C.c_int),
    "b200_engine_destroy": ([_vp], None),
    "b200_engine_memory": ([_vp, _vp, _vp, _vp], C.c_int),
    "b200_engine_set_weight": ([_vp, C.c_char_p, _vp, _i64], C.c_int),
    "b200_engine_init_random": ([_vp, C.c_uint64, _f32], C.c_int),
    "b200_engine_finalize": ([_vp], C.c_int),
    "b200_engine_reset": ([_vp], C.c_int),
    "b200_engine_n_past": ([_vp], _i64),
    "b200_engine_set_precision": ([_vp, C.c_int32], C.c_int),
    "b200_engine_decode_launches": ([_vp], C.c_int),
    "b200_engine_eval": ([_vp, _vp, _i64, _vp, _vp], C.c_int),
    "b200_engine_generate": ([_vp, _i64, _vp], C.c_int),
    "b200_engine_profile_step": ([_vp, _vp, C.c_int, _vp, C.c_int], C.c_int),
    "b200_engine_trace_step": ([_vp, _vp, C.c_int], C.c_int),
    "b200_engine_stream": ([_vp], _vp),
    "b200_engine_read_status": ([_vp, _vp], C.c_int),
    "b200_engine_load_gguf": ([_vp, C.c_char_p, C.c_int64], C.c_int),
    "b200_engine_get_weight": ([_vp, C.c_char_p, _vp, C.c_int64], C.c_int),
    "b200_engine_eval_device": ([_vp, _vp, C.c_int64, _vp, _vp], C.c_int),
    "b200_engine_set_n_past": ([_vp, C.c_int64], C.c_int),
    "b200_engine_set_rope_freqs": ([_vp, _vp], C.c_int),
    "b200_engine_bind_kv": ([_vp, C.c_int32, _vp, _vp], C.c_int),
    "b200_engine_tp_peer_exchange": ([_vp], C.c_int),
    "b200_paged_kv_write": ([_vp, _vp, C.c_int64, _vp, _vp, C.c_int64, C.c_int64, C.c_int64, C.c_int64, C.c_int64,
                             C.c_int64, _vp, _vp], C.c_int),
    "b200_flash_attn_paged": ([_vp, _vp, _vp, C.c_int64, C.c_int64, _vp, C.c_int64, C.c_int64, C.c_int64, C.c_int64,
                               C.c_int64, C.c_int64, C.c_float, _vp, _sz, _vp, _vp], C.c_int),
    "b200_flash_attn_paged_workspace_bytes": ([C.c_int64] * 5, _sz),
    "b200_flash_attn_packed": ([_vp, _i64, _i64, _vp, _i64, _i64, _vp, _i64, _i64, _vp, _i64, _i64, _vp, _vp, _i64,
                                _i64, _i64, _i64, _i64, _i64, _f32, _i32, _vp, _sz, _vp, _vp], C.c_int),
    "b200_flash_attn_packed_workspace_bytes": ([_i64] * 6 + [_i32], _sz),
    "b200_paged_kv_append": ([_vp, _i64, _i64, _vp, _i64, _i64, _vp, _vp, _i64, _i64, _vp, _vp, _i64, _i64, _vp, _vp],
                             C.c_int),
    "b200_flash_attn_paged_batch": ([_vp, _i64, _i64, _vp, _i64, _i64, _vp, _vp, _i64, _i64, _vp, _i64, _i64, _f32,
                                     _vp, _sz, _vp, _vp], C.c_int),
    "b200_flash_attn_paged_batch_workspace_bytes": ([_i64] * 5 + [_i32], _sz),
    "b200_paged_kv_append_q8": ([_vp, _i64, _i64, _vp, _i64, _i64, _i32, _vp, _vp, _i64, _i64, _vp, _vp, _i64, _i64, _vp, _vp],
                                C.c_int),
    "b200_paged_kv_read_q8": ([_vp, _vp, _i64, _i64, _vp, _vp, _i64, _i64, _vp, _i64, _i64, _vp, _i64, _i64, _i32, _vp, _vp],
                              C.c_int),
    "b200_flash_attn_paged_batch_q8": ([_vp, _i64, _i64, _vp, _i64, _i64, _i32, _vp, _vp, _i64, _i64, _vp, _i64, _i64, _f32,
                                        _vp, _sz, _vp, _vp], C.c_int),
    "b200_flash_attn_paged_batch_q8_workspace_bytes": ([_i64] * 5, _sz),
    "b200_flash_attn_paged_shared": ([_vp, _i64, _i64, _vp, _i64, _i64, _vp, _vp, _i64, _i64, _vp, _vp, _i64, _vp, _i64, _i64,
                                      _vp, _i64, _i64, _f32, _vp, _sz, _vp, _vp], C.c_int),
    "b200_flash_attn_paged_shared_workspace_bytes": ([_i64] * 7 + [_i32], _sz),
    "b200_adjust_logits": ([_vp, _i64, _vp, _i64, _i64, _i64, _i32, _vp, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _vp,
                            _vp, _i64, _vp, _vp], C.c_int),
    "b200_sample": ([_vp, _i64, _i64, _i64, _i32, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp], C.c_int),
    "b200_engine_inject_withhold": ([_vp, C.c_int32, C.c_int32], C.c_int),
    "b200_engine_set_decode_launch_counter": ([_vp, C.c_uint64], C.c_int),
    "b200_tp_unique_id": ([_vp], C.c_int),
    "b200_engine_tp_init": ([_vp, _vp], C.c_int),
}


def lib() -> C.CDLL:
    """The loaded library (raises FileNotFoundError if it has not been built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(lib_path):
            raise FileNotFoundError(f"{lib_path} is missing: run b200infer.build() (make -C infer-llm_b200)")
        L = C.CDLL(lib_path)
        for name, (args, res) in _SIGS.items():
            f = getattr(L, name)
            f.argtypes = args
            f.restype = res
        _lib = L
    return _lib


def _chk(name: str, rc: int):
    if rc != 0:
        raise B200Error(name, rc)


def _p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _stream():
    import torch
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _dev_check(*ts):
    for t in ts:
        if t is not None:
            assert t.is_cuda and t.is_contiguous(), "expected contiguous CUDA tensors"


def mul_mat(w, x, precision=PREC_FFMA, out=None, workspace=None):
    """y = x . w^T; w (N, K), x (M, K) -> (M, N) float32.

    workspace: a uint8 tensor of b200_mul_mat_workspace_bytes bytes for the split-K
    partials (None: one is allocated when the shape splits K; an empty tensor: no
    split)."""
    import torch
    _dev_check(w, x)
    N, K = w.shape
    M = x.shape[0]
    out = out if out is not None else torch.empty((M, N), device=x.device, dtype=torch.float32)
    if workspace is None:
        nbytes = lib().b200_mul_mat_workspace_bytes(K, N, M, precision)
        workspace = torch.empty(nbytes, device=x.device, dtype=torch.uint8)
    _chk("b200_mul_mat_ws", lib().b200_mul_mat_ws(_p(w), _p(x), _p(out), K, N, M, precision,
                                                  _p(workspace) if workspace.numel() else None,
                                                  workspace.numel(), _stream()))
    return out


def rms_norm(x, gamma, eps, out=None):
    import torch
    _dev_check(x, gamma)
    D = gamma.numel()
    out = out if out is not None else torch.empty_like(x)
    _chk("b200_rms_norm", lib().b200_rms_norm(_p(x), _p(gamma), _p(out), D, x.numel() // D, eps, _stream()))
    return out


def rope(x, pos, table, status=None, out=None):
    """x (T, H, D); pos int32 (T,); table (n_ctx, D/2) device angles."""
    import torch
    _dev_check(x, pos, table)
    T, H, D = x.shape
    out = out if out is not None else torch.empty_like(x)
    _chk("b200_rope", lib().b200_rope(_p(x), _p(pos), _p(table), table.shape[0], _p(out), D, H, T,
                                       _p(status), _stream()))
    return out


def rope_freqs(theta: float, D: int):
    import numpy as np
    f = np.empty(D // 2, np.float32)
    lib().b200_rope_freqs(theta, D, C.c_void_p(f.ctypes.data))
    return f


def qk_norm_rope(q, k, q_gamma, k_gamma, freq, pos, eps, n_ctx, v=None, k_out=None, v_out=None,
                 status=None):
    """q (T, Hq, D), k/v (T, Hkv, D) -> (q_rot, k_rot[, v copy]) (fresh tensors unless given)."""
    import torch
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    q_out = torch.empty_like(q)
    k_out = k_out if k_out is not None else torch.empty_like(k)
    if v is not None and v_out is None:
        v_out = torch.empty_like(v)
    _chk("b200_qk_norm_rope", lib().b200_qk_norm_rope(
        _p(q), Hq * D, _p(k), Hkv * D, _p(v), Hkv * D, _p(q_gamma), _p(k_gamma), _p(freq), _p(pos),
        _p(q_out), _p(k_out), Hkv * D, _p(v_out), Hkv * D, D, Hq, Hkv, T, n_ctx, eps, _p(status), _stream()))
    return q_out, k_out, v_out


def flash_attn(q, k, v, n_past, scale=0.0, out=None, workspace=None, precision=0):
    """q (Tq, Hq, D); k, v (Tkv, Hkv, D) token-major; returns (Tq, Hq, D).

    workspace: a zero-filled uint8 tensor of b200_flash_attn_workspace_bytes bytes
    (reusable across calls), or None for a fresh one; pass an empty tensor to run
    decode without one (the cluster-merged path). precision: PREC_FFMA (exact F32)
    or PREC_TF32 (prefill on the tensor cores, head_dim 128)."""
    import torch
    _dev_check(q, k, v)
    Tq, Hq, D = q.shape
    Tkv, Hkv, _ = k.shape
    out = out if out is not None else torch.empty_like(q)
    nbytes = lib().b200_flash_attn_workspace_bytes(D, Hq, Hkv, Tq, Tkv)
    if workspace is None:  # zero-filled: the decode split counters start at zero
        workspace = torch.zeros(nbytes, device=q.device, dtype=torch.uint8)
    _chk("b200_flash_attn_ex", lib().b200_flash_attn_ex(
        _p(q), _p(k), _p(v), _p(out), D, Hq, Hkv, Tq, Tkv, n_past, scale, Hkv * D, D, Hkv * D, D,
        _p(workspace), workspace.numel(), _stream(), precision))
    return out


def _elt(fn, *ts, out=None):
    import torch
    out = out if out is not None else torch.empty_like(ts[0])
    args = [_p(t) for t in ts] + [_p(out), ts[0].numel(), _stream()]
    _chk(fn, getattr(lib(), fn)(*args))
    return out


def silu(x, out=None):
    return _elt("b200_silu", x, out=out)


def mul(a, b, out=None):
    return _elt("b200_mul", a, b, out=out)


def add(a, b, out=None):
    return _elt("b200_add", a, b, out=out)


def swiglu(gate, up, out=None):
    return _elt("b200_swiglu", gate, up, out=out)


def get_rows(table, ids, status=None, out=None):
    import torch
    n_rows, D = table.shape
    out = out if out is not None else torch.zeros((ids.numel(), D), device=table.device, dtype=torch.float32)
    _chk("b200_get_rows", lib().b200_get_rows(_p(table), _p(ids), _p(out), D, ids.numel(), n_rows,
                                               _p(status), _stream()))
    return out


def copy(dst, src):
    _chk("b200_copy", lib().b200_copy(_p(dst), _p(src), src.numel() * src.element_size(), _stream()))
    return dst


def argmax(logits, status=None):
    import torch
    n = logits.numel()
    ws = torch.empty(lib().b200_argmax_workspace_bytes(n), device=logits.device, dtype=torch.uint8)
    out = torch.empty(1, device=logits.device, dtype=torch.int32)
    _chk("b200_argmax", lib().b200_argmax(_p(logits), n, _p(out), _p(ws), ws.numel(), _p(status), _stream()))
    return out


class PagedKV:
    """A paged K/V cache on the device for tests and benchmarks: n_blocks blocks of
    block_tokens tokens each (one torch tensor per pool; the block tables list the
    blocks in `order`, so logical block i is pool block order[i])."""

    def __init__(self, n_blocks, block_tokens, Hkv, D, device, order=None):
        import torch
        self.bt, self.Hkv, self.D = block_tokens, Hkv, D
        self.kpool = torch.zeros((n_blocks, block_tokens, Hkv, D), device=device)
        self.vpool = torch.zeros_like(self.kpool)
        order = list(range(n_blocks)) if order is None else list(order)
        bytes_per = block_tokens * Hkv * D * 4
        self.ktab = torch.tensor([self.kpool.data_ptr() + i * bytes_per for i in order], dtype=torch.int64, device=device)
        self.vtab = torch.tensor([self.vpool.data_ptr() + i * bytes_per for i in order], dtype=torch.int64, device=device)
        self.n_blocks = len(order)

    def write(self, k, v, pos0, status=None):
        """k, v (T, Hkv, D) contiguous -> positions pos0..pos0+T-1."""
        T = k.shape[0]
        _chk("b200_paged_kv_write", lib().b200_paged_kv_write(
            _p(k), _p(v), self.Hkv * self.D, _p(self.ktab), _p(self.vtab), self.n_blocks, self.bt, pos0, T,
            self.Hkv, self.D, _p(status), _stream()))

    def attn(self, q, n_past, scale=0.0, out=None, workspace=None, status=None):
        """q (Tq, Hq, D) against positions [0, n_past + Tq)."""
        import torch
        Tq, Hq, D = q.shape
        Tkv = n_past + Tq
        out = out if out is not None else torch.empty_like(q)
        nbytes = lib().b200_flash_attn_paged_workspace_bytes(D, Hq, self.Hkv, Tq, Tkv)
        if workspace is None:
            workspace = torch.zeros(nbytes, device=q.device, dtype=torch.uint8)
        _chk("b200_flash_attn_paged", lib().b200_flash_attn_paged(
            _p(q), _p(self.ktab), _p(self.vtab), self.n_blocks, self.bt, _p(out), D, Hq, self.Hkv, Tq, Tkv, n_past,
            scale, _p(workspace), workspace.numel(), _p(status), _stream()))
        return out


# ---------------------------------------------------------------------------
# Batched serving: packed prompts, paged caches of many sequences, sampling. Tensors
# are float32, float16 or bfloat16, on one device, with a contiguous last axis; calls
# go to the current torch stream of that device.

class _KVPool(C.Structure):
    """b200_kv_pool."""
    _fields_ = [("k", _vp), ("v", _vp), ("n_blocks", _i64), ("block_tokens", _i64), ("block_stride", _i64),
                ("tok_stride", _i64), ("head_stride", _i64), ("n_head_kv", _i64), ("head_dim", _i64),
                ("dtype", C.c_int32)]


_POOL = struct.Struct("@PPqqqqqqqi4x")  # the same, packed (a call of its own per decode step and layer)


class _KVPoolQ8(C.Structure):
    """b200_kv_pool_q8."""
    _fields_ = [("k", _vp), ("v", _vp), ("k_scale", _vp), ("v_scale", _vp), ("n_blocks", _i64), ("block_tokens", _i64),
                ("block_stride", _i64), ("tok_stride", _i64), ("head_stride", _i64), ("scale_block_stride", _i64),
                ("scale_tok_stride", _i64), ("scale_head_stride", _i64), ("n_head_kv", _i64), ("head_dim", _i64)]


_POOL_Q8 = struct.Struct("@PPPPqqqqqqqqqq")


class _Host:
    """What the batched calls take from torch, looked up once: a decode step makes several of
    these calls per layer, and each is only microseconds on the device."""

    def __init__(self):
        import torch
        self.torch = torch
        self.empty_like = torch.empty_like
        self.empty, self.i32, self.f32, self.u8 = torch.empty, torch.int32, torch.float32, torch.uint8
        self.dtypes = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
        self.current = torch._C._cuda_getDevice
        self.stream = torch._C._cuda_getCurrentRawStream
        L = lib()
        self.packed, self.packed_bytes = L.b200_flash_attn_packed, L.b200_flash_attn_packed_workspace_bytes
        self.batch, self.batch_bytes = L.b200_flash_attn_paged_batch, _by_sizes(L.b200_flash_attn_paged_batch_workspace_bytes)
        self.append, self.sample = L.b200_paged_kv_append, L.b200_sample
        self.e4m3, self.e8m0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
        self.append_q8, self.read_q8 = L.b200_paged_kv_append_q8, L.b200_paged_kv_read_q8
        self.batch_q8 = L.b200_flash_attn_paged_batch_q8
        self.batch_q8_bytes = _by_sizes(L.b200_flash_attn_paged_batch_q8_workspace_bytes)
        self.shared, self.shared_bytes = L.b200_flash_attn_paged_shared, _by_sizes(L.b200_flash_attn_paged_shared_workspace_bytes)
        self.adjust = L.b200_adjust_logits


_host = None


def _start(t):
    """(host, device index) for a call whose first tensor is t."""
    global _host
    dev = t.get_device()
    if dev < 0:
        raise ValueError("expected CUDA tensors")
    if _host is None:
        _host = _Host()
    return _host, dev


def _elsewhere(fn, dev, *args, **kw):
    """The call with its tensors' device made current."""
    with _host.torch.cuda.device(dev):
        return fn(*args, **kw)


def _dtype(t):
    d = _host.dtypes.get(t.dtype)
    if d is None:
        raise TypeError(f"expected float32, float16 or bfloat16, got {t.dtype}")
    return d


def _rows(t, name, dtype, dev):
    """Checks a (rows, heads, D) tensor with a contiguous last axis; its shape and strides."""
    st = t.stride()
    if len(st) != 3 or t.dtype is not dtype or t.get_device() != dev or (st[2] != 1 and t.shape[2] != 1):
        raise ValueError(f"{name}: expected (rows, heads, D) of {dtype} on cuda:{dev}, last axis contiguous")
    return st


def _vector(t, name, n, dtype, dev):
    if t.dtype is not dtype or t.get_device() != dev or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name}: expected {n} contiguous {dtype} on cuda:{dev}")
    return t.data_ptr()


def _status_word(status, dev):
    if status is None:
        return None
    if status.dtype != _host.i32 or status.get_device() != dev or status.numel() < 1:
        raise ValueError(f"status: expected int32 on cuda:{dev}")
    return status.data_ptr()


def _by_sizes(fn):
    """A function of a device and sizes that decode steps repeat: their workspaces' bytes, 1 us less once known."""
    return functools.lru_cache(maxsize=1024)(lambda dev, *sizes: fn(*sizes))


def _scratch(workspace, nbytes, like, dev):
    if workspace is None:
        return like.new_empty(nbytes, dtype=_host.u8) if nbytes else None
    if not workspace.is_contiguous() or workspace.get_device() != dev or workspace.nbytes < nbytes:
        raise ValueError(f"workspace: expected {nbytes} bytes on cuda:{dev}")
    return workspace


def _out_rows(out, q, dev):
    if out is None:
        return _host.empty_like(q)
    if out.shape != q.shape:
        raise ValueError("out: expected q's shape")
    _rows(out, "out", q.dtype, dev)
    return out


def flash_attn_packed(q, k, v, cu_q, cu_k=None, scale=0.0, out=None, workspace=None, status=None):
    """Causal attention of packed sequences: q (Tq, Hq, D); k, v (Tk, Hkv, D); cu_q, cu_k int32
    (n + 1,) offsets of the n sequences (cu_k None: as cu_q). Row i of a sequence with nq
    queries and nk keys sees its keys 0 .. nk - nq + i. Returns (Tq, Hq, D). Rows outside every
    sequence are not written; offsets out of range leave zeros, and set `status`."""
    h, dev = _start(q)
    if h.current() != dev:
        return _elsewhere(flash_attn_packed, dev, q, k, v, cu_q, cu_k, scale, out, workspace, status)
    kind, dt = q.dtype, _dtype(q)
    qs, ks, vs = _rows(q, "q", kind, dev), _rows(k, "k", kind, dev), _rows(v, "v", kind, dev)
    Tq, Hq, D = q.shape
    Tk, Hkv, Dk = k.shape
    if v.shape != k.shape or Dk != D or Hkv <= 0 or Hq % Hkv:
        raise ValueError("k, v: shapes do not go with q")
    n = cu_q.shape[0] - 1
    pq = _vector(cu_q, "cu_q", n + 1, h.i32, dev)
    pk = pq if cu_k is None else _vector(cu_k, "cu_k", n + 1, h.i32, dev)
    out = _out_rows(out, q, dev)
    os = out.stride()
    nbytes = h.packed_bytes(n, Tq, Tk, D, Hq, Hkv, dt)
    ws = _scratch(workspace, nbytes, q, dev)
    _chk("b200_flash_attn_packed", h.packed(
        q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], out.data_ptr(), os[0], os[1],
        pq, pk, n, Tq, Tk, D, Hq, Hkv, scale, dt, None if ws is None else ws.data_ptr(), nbytes, _status_word(status, dev),
        h.stream(dev)))
    return out


def _pool(k_pool, v_pool):
    s = k_pool.stride()
    if len(s) != 4 or k_pool.shape != v_pool.shape or s != v_pool.stride() or k_pool.dtype != v_pool.dtype or \
            k_pool.get_device() != v_pool.get_device() or s[3] != 1:
        raise ValueError("k_pool, v_pool: expected two (blocks, block_tokens, Hkv, D) tensors alike, last axis contiguous")
    n, bt, Hkv, D = k_pool.shape
    return _POOL.pack(k_pool.data_ptr(), v_pool.data_ptr(), n, bt, s[0], s[1], s[2], Hkv, D, _dtype(k_pool)), bt, Hkv, D


def _table(t, n, dev, name="block_table"):
    st, shape = t.stride(), t.shape
    if len(st) != 2 or shape[0] != n or t.dtype is not _host.i32 or t.get_device() != dev or (st[1] != 1 and shape[1] != 1):
        raise ValueError(f"{name}: expected int32 ({n}, blocks) on cuda:{dev}")
    # a table of one row may report any stride; the rows must not overlap
    return t.data_ptr(), st[0] if n > 1 else shape[1], shape[1]


def paged_kv_append(k, v, cu_new, seq_lens, k_pool, v_pool, block_table, status=None):
    """The rows k, v (T, Hkv, D) of new tokens into the pools (blocks, block_tokens, Hkv, D):
    sequence s owns rows [cu_new[s], cu_new[s + 1]), which become its last positions;
    seq_lens (n,) counts them in, block_table (n, max blocks) names its blocks; all int32."""
    h, dev = _start(k)
    if h.current() != dev:
        return _elsewhere(paged_kv_append, dev, k, v, cu_new, seq_lens, k_pool, v_pool, block_table, status)
    kind = k.dtype
    if k_pool.get_device() != dev or k_pool.dtype != kind:
        raise ValueError(f"k_pool: expected {kind} on cuda:{dev}")
    pool, _, Hkv, D = _pool(k_pool, v_pool)
    ks, vs = _rows(k, "k", kind, dev), _rows(v, "v", kind, dev)
    T = k.shape[0]
    if k.shape != v.shape or k.shape[1] != Hkv or k.shape[2] != D:
        raise ValueError("k, v: expected (T, Hkv, D)")
    n = seq_lens.shape[0]
    table, stride, blocks = _table(block_table, n, dev)
    _chk("b200_paged_kv_append", h.append(
        k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], _vector(cu_new, "cu_new", n + 1, h.i32, dev),
        _vector(seq_lens, "seq_lens", n, h.i32, dev), n, T, pool, table, stride, blocks, _status_word(status, dev),
        h.stream(dev)))


def flash_attn_paged_batch(q, k_pool, v_pool, block_table, seq_lens, scale=0.0, out=None, workspace=None, status=None):
    """One new token of each sequence, q (n, Hq, D), against its seq_lens[s] cached positions
    in the pools (arguments as for paged_kv_append). Returns (n, Hq, D)."""
    h, dev = _start(q)
    if h.current() != dev:
        return _elsewhere(flash_attn_paged_batch, dev, q, k_pool, v_pool, block_table, seq_lens, scale, out, workspace,
                          status)
    kind, dt = q.dtype, _dtype(q)
    if k_pool.get_device() != dev or k_pool.dtype != kind:
        raise ValueError(f"k_pool: expected {kind} on cuda:{dev}")
    pool, bt, Hkv, Dk = _pool(k_pool, v_pool)
    qs = _rows(q, "q", kind, dev)
    n, Hq, D = q.shape
    if D != Dk or Hkv <= 0 or Hq % Hkv:
        raise ValueError("q: shape does not go with the pools")
    table, stride, blocks = _table(block_table, n, dev)
    out = _out_rows(out, q, dev)
    os = out.stride()
    nbytes = h.batch_bytes(dev, n, blocks * bt, D, Hq, Hkv, dt)
    ws = _scratch(workspace, nbytes, q, dev)
    _chk("b200_flash_attn_paged_batch", h.batch(
        q.data_ptr(), qs[0], qs[1], out.data_ptr(), os[0], os[1], pool, table, stride, blocks,
        _vector(seq_lens, "seq_lens", n, h.i32, dev), n, Hq, scale, None if ws is None else ws.data_ptr(), nbytes,
        _status_word(status, dev), h.stream(dev)))
    return out


def _pool_q8(k_pool, v_pool, k_scale, v_scale, dev):
    e4m3, e8m0 = _host.e4m3, _host.e8m0
    s, e, shape = k_pool.stride(), k_scale.stride(), k_pool.shape
    if len(s) != 4 or s[3] != 1 or k_pool.dtype is not e4m3 or v_pool.dtype is not e4m3 or v_pool.shape != shape or \
            v_pool.stride() != s or k_pool.get_device() != dev or v_pool.get_device() != dev:
        raise ValueError("k_pool, v_pool: expected two (blocks, block_tokens, Hkv, D) float8_e4m3fn tensors alike, last axis "
                         f"contiguous, on cuda:{dev}")
    n, bt, Hkv, D = shape
    shape = (n, Hkv, bt)
    if k_scale.dtype is not e8m0 or v_scale.dtype is not e8m0 or k_scale.shape != shape or v_scale.shape != shape or \
            v_scale.stride() != e or k_scale.get_device() != dev or v_scale.get_device() != dev:
        raise ValueError(f"k_scale, v_scale: expected two (blocks, Hkv, block_tokens) float8_e8m0fnu tensors alike on cuda:{dev}")
    return _POOL_Q8.pack(k_pool.data_ptr(), v_pool.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), n, bt, s[0], s[1], s[2],
                         e[0], e[2], e[1], Hkv, D), bt, Hkv, D


def paged_kv_append_q8(k, v, cu_new, seq_lens, k_pool, v_pool, k_scale, v_scale, block_table, status=None):
    """paged_kv_append into an 8-bit cache: k_pool, v_pool (blocks, block_tokens, Hkv, D) float8_e4m3fn and k_scale,
    v_scale (blocks, Hkv, block_tokens) float8_e8m0fnu, one scale a row of D elements. Each row gets the least power of
    two with which its largest element is at most 448; a row that holds an infinity or a NaN reads as NaN."""
    h, dev = _start(k)
    if h.current() != dev:
        return _elsewhere(paged_kv_append_q8, dev, k, v, cu_new, seq_lens, k_pool, v_pool, k_scale, v_scale, block_table, status)
    kind, dt = k.dtype, _dtype(k)
    pool, _, Hkv, D = _pool_q8(k_pool, v_pool, k_scale, v_scale, dev)
    ks, vs = _rows(k, "k", kind, dev), _rows(v, "v", kind, dev)
    T, heads, dim = shape = k.shape
    if v.shape != shape or heads != Hkv or dim != D:
        raise ValueError("k, v: expected (T, Hkv, D)")
    n = seq_lens.shape[0]
    table, stride, blocks = _table(block_table, n, dev)
    _chk("b200_paged_kv_append_q8", h.append_q8(
        k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], dt, _vector(cu_new, "cu_new", n + 1, h.i32, dev),
        _vector(seq_lens, "seq_lens", n, h.i32, dev), n, T, pool, table, stride, blocks, _status_word(status, dev),
        h.stream(dev)))


def paged_kv_read_q8(cu_rows, seq_lens, n_rows, k_pool, v_pool, k_scale, v_scale, block_table, dtype=None, k=None, v=None,
                     status=None):
    """Rows of an 8-bit cache as packed rows (n_rows, Hkv, D), k and v: sequence s gets the rows [cu_rows[s],
    cu_rows[s + 1]), its last positions of the seq_lens[s] cached. `dtype` (None: bfloat16) is that of new tensors, else
    they go to the given `k` and `v`, whose rows outside every sequence stay as they are (of new tensors: undefined).
    For flash_attn_packed, where a prompt goes on behind a cached head."""
    h, dev = _start(k_pool)
    if h.current() != dev:
        return _elsewhere(paged_kv_read_q8, dev, cu_rows, seq_lens, n_rows, k_pool, v_pool, k_scale, v_scale, block_table, dtype,
                          k, v, status)
    pool, _, Hkv, D = _pool_q8(k_pool, v_pool, k_scale, v_scale, dev)
    if k is None and v is None:
        k = k_pool.new_empty((n_rows, Hkv, D), dtype=dtype or h.torch.bfloat16)
        v = h.empty_like(k)
        dt = _dtype(k)
        ks = vs = (Hkv * D, D)
    elif k is None or v is None or k.shape != v.shape or k.shape != (n_rows, Hkv, D) or (dtype or k.dtype) != k.dtype:
        raise ValueError("k, v: expected both (n_rows, Hkv, D), of `dtype`")
    else:
        kind, dt = k.dtype, _dtype(k)
        ks, vs = _rows(k, "k", kind, dev), _rows(v, "v", kind, dev)
    n = seq_lens.shape[0]
    table, stride, blocks = _table(block_table, n, dev)
    _chk("b200_paged_kv_read_q8", h.read_q8(
        pool, table, stride, blocks, _vector(cu_rows, "cu_rows", n + 1, h.i32, dev), _vector(seq_lens, "seq_lens", n, h.i32, dev),
        n, n_rows, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], dt, _status_word(status, dev), h.stream(dev)))
    return k, v


def flash_attn_paged_batch_q8(q, k_pool, v_pool, k_scale, v_scale, block_table, seq_lens, scale=0.0, out=None, workspace=None,
                              status=None):
    """flash_attn_paged_batch over an 8-bit cache (arguments as for paged_kv_append_q8): q (n, Hq, D) of float32,
    float16 or bfloat16 against the values that the cache stands for. Returns (n, Hq, D)."""
    h, dev = _start(q)
    if h.current() != dev:
        return _elsewhere(flash_attn_paged_batch_q8, dev, q, k_pool, v_pool, k_scale, v_scale, block_table, seq_lens, scale, out,
                          workspace, status)
    kind, dt = q.dtype, _dtype(q)
    pool, bt, Hkv, Dk = _pool_q8(k_pool, v_pool, k_scale, v_scale, dev)
    qs = _rows(q, "q", kind, dev)
    n, Hq, D = q.shape
    if D != Dk or Hkv <= 0 or Hq % Hkv:
        raise ValueError("q: shape does not go with the pools")
    table, stride, blocks = _table(block_table, n, dev)
    out = _out_rows(out, q, dev)
    os = out.stride()
    nbytes = h.batch_q8_bytes(dev, n, blocks * bt, D, Hq, Hkv)
    ws = _scratch(workspace, nbytes, q, dev)
    _chk("b200_flash_attn_paged_batch_q8", h.batch_q8(
        q.data_ptr(), qs[0], qs[1], out.data_ptr(), os[0], os[1], dt, pool, table, stride, blocks,
        _vector(seq_lens, "seq_lens", n, h.i32, dev), n, Hq, scale, None if ws is None else ws.data_ptr(), nbytes,
        _status_word(status, dev), h.stream(dev)))
    return out


def flash_attn_paged_shared(q, k_pool, v_pool, prefix_table, prefix_lens, cu_seqs, block_table, seq_lens, scale=0.0, out=None,
                            workspace=None, status=None):
    """flash_attn_paged_batch of sequences that share prefixes: group g, the sequences [cu_seqs[g], cu_seqs[g + 1]),
    sees the prefix_lens[g] positions of row g of prefix_table first, then each its seq_lens[s] own positions
    of block_table (int32; both name blocks of the pools). Returns (n, Hq, D)."""
    h, dev = _start(q)
    if h.current() != dev:
        return _elsewhere(flash_attn_paged_shared, dev, q, k_pool, v_pool, prefix_table, prefix_lens, cu_seqs, block_table,
                          seq_lens, scale, out, workspace, status)
    kind, dt = q.dtype, _dtype(q)
    if k_pool.get_device() != dev or k_pool.dtype != kind:
        raise ValueError(f"k_pool: expected {kind} on cuda:{dev}")
    pool, bt, Hkv, Dk = _pool(k_pool, v_pool)
    qs = _rows(q, "q", kind, dev)
    n, Hq, D = q.shape
    if D != Dk or Hkv <= 0 or Hq % Hkv:
        raise ValueError("q: shape does not go with the pools")
    groups = prefix_lens.shape[0]
    table, stride, blocks = _table(block_table, n, dev)
    ptable, pstride, pblocks = _table(prefix_table, groups, dev, "prefix_table")
    out = _out_rows(out, q, dev)
    os = out.stride()
    nbytes = h.shared_bytes(dev, n, blocks * bt, groups, pblocks * bt, D, Hq, Hkv, dt)
    ws = _scratch(workspace, nbytes, q, dev)
    _chk("b200_flash_attn_paged_shared", h.shared(
        q.data_ptr(), qs[0], qs[1], out.data_ptr(), os[0], os[1], pool, ptable, pstride, pblocks,
        _vector(prefix_lens, "prefix_lens", groups, h.i32, dev), _vector(cu_seqs, "cu_seqs", groups + 1, h.i32, dev), groups,
        table, stride, blocks, _vector(seq_lens, "seq_lens", n, h.i32, dev), n, Hq, scale,
        None if ws is None else ws.data_ptr(), nbytes, _status_word(status, dev), h.stream(dev)))
    return out


def adjust_logits(logits, tokens=None, cu_tokens=None, prompt_lens=None, repetition=None, frequency=None, presence=None,
                  bias_ids=None, bias_values=None, cu_bias=None, mask=None, out=None, status=None):
    """Logits (n, vocab) as their rows' requests want them before `sample`. Row s has the history `tokens`
    [cu_tokens[s], cu_tokens[s + 1]) (int32), of which the first prompt_lens[s] are its prompt. In this order: a
    token of the history is divided by (where positive, else multiplied by) repetition[s]; one drawn c > 0 times
    after the prompt loses c frequency[s] + presence[s]; token bias_ids[i] gains bias_values[i], i in [cu_bias[s],
    cu_bias[s + 1]) (the last of several for one token); tokens whose bit is 0 in mask (n, ceil(vocab / 32)) int32, bit t %
    32 of word t / 32, become -inf. What is None is off. `out` (None: a new tensor) may be `logits`. Returns out."""
    h, dev = _start(logits)
    if h.current() != dev:
        return _elsewhere(adjust_logits, dev, logits, tokens, cu_tokens, prompt_lens, repetition, frequency, presence, bias_ids,
                          bias_values, cu_bias, mask, out, status)
    st = logits.stride()
    dt = _dtype(logits)
    if len(st) != 2 or (st[1] != 1 and logits.shape[1] != 1):
        raise ValueError("logits: expected (n, vocab), last axis contiguous")
    n, vocab = logits.shape
    if out is None:
        out = h.empty_like(logits) if st[0] == vocab else logits.new_empty((n, vocab))
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.get_device() != dev or \
            (out.stride(1) != 1 and vocab != 1):
        raise ValueError("out: expected logits' shape and type, last axis contiguous")

    def row(t, name, kind, m=n):
        return None if t is None else _vector(t, name, m, kind, dev)

    if (tokens is None) != (cu_tokens is None) or (bias_ids is None) != (bias_values is None) or \
            (bias_ids is None) != (cu_bias is None):
        raise ValueError("tokens and cu_tokens go together, and bias_ids, bias_values and cu_bias")
    T, m = 0 if tokens is None else tokens.shape[0], 0 if bias_ids is None else bias_ids.shape[0]
    words, word_stride = None, 0
    if mask is not None:
        ms = mask.stride()
        if len(ms) != 2 or mask.shape[0] != n or mask.shape[1] * 32 < vocab or mask.dtype != h.i32 or \
                mask.get_device() != dev or (ms[1] != 1 and mask.shape[1] != 1):
            raise ValueError(f"mask: expected int32 (n, ceil(vocab / 32)) on cuda:{dev}, last axis contiguous")
        words, word_stride = mask.data_ptr(), ms[0]
    _chk("b200_adjust_logits", h.adjust(
        logits.data_ptr(), st[0], out.data_ptr(), out.stride(0), n, vocab, dt, row(tokens, "tokens", h.i32, T), T,
        row(cu_tokens, "cu_tokens", h.i32, n + 1), row(prompt_lens, "prompt_lens", h.i32), row(repetition, "repetition", h.f32),
        row(frequency, "frequency", h.f32), row(presence, "presence", h.f32), row(bias_ids, "bias_ids", h.i32, m),
        row(bias_values, "bias_values", h.f32, m), m, row(cu_bias, "cu_bias", h.i32, n + 1), words, word_stride,
        _status_word(status, dev), h.stream(dev)))
    return out


def sample(logits, u, temperature, top_k=None, top_p=None, min_p=None, out=None, status=None):
    """One token id per row of logits (n, vocab), drawn with u (n,) uniform in [0, 1);
    temperature, top_p, min_p float32 (n,), top_k int32 (n,) (None: that filter is off).
    Returns int32 (n,); -1 for a row that cannot be sampled."""
    h, dev = _start(logits)
    if h.current() != dev:
        return _elsewhere(sample, dev, logits, u, temperature, top_k, top_p, min_p, out, status)
    st = logits.stride()
    dt = _dtype(logits)
    if len(st) != 2 or (st[1] != 1 and logits.shape[1] != 1):
        raise ValueError("logits: expected (n, vocab), last axis contiguous")
    n, vocab = logits.shape
    if out is None:
        out = h.empty(n, device=logits.device, dtype=h.i32)
    _chk("b200_sample", h.sample(
        logits.data_ptr(), st[0], n, vocab, dt, _vector(u, "u", n, h.f32, dev),
        _vector(temperature, "temperature", n, h.f32, dev),
        None if top_k is None else _vector(top_k, "top_k", n, h.i32, dev),
        None if top_p is None else _vector(top_p, "top_p", n, h.f32, dev),
        None if min_p is None else _vector(min_p, "min_p", n, h.f32, dev), _vector(out, "out", n, h.i32, dev),
        _status_word(status, dev), h.stream(dev)))
    return out
