"""ctypes binding of the single-op C ABI (include/b200_infer.h).

Tensor arguments are torch tensors on the current CUDA device (contiguous,
float32 / int32); the functions pass their data pointers and the current
torch stream to the library. Shapes follow the reference's node semantics:
``mul_mat(w (N,K), x (M,K)) -> (M,N)`` is OpFactory::mul_mat(w, x).
"""
from __future__ import annotations

import ctypes as C
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
        self.batch, self.batch_bytes = L.b200_flash_attn_paged_batch, L.b200_flash_attn_paged_batch_workspace_bytes
        self.append, self.sample = L.b200_paged_kv_append, L.b200_sample


_host = None


def _start(t):
    """(host, device index) for a call whose first tensor is t."""
    global _host
    if not t.is_cuda:
        raise ValueError("expected CUDA tensors")
    if _host is None:
        _host = _Host()
    return _host, t.get_device()


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
    if len(st) != 3 or t.dtype != dtype or t.get_device() != dev or (st[2] != 1 and t.shape[2] != 1):
        raise ValueError(f"{name}: expected (rows, heads, D) of {dtype} on cuda:{dev}, last axis contiguous")
    return st


def _vector(t, name, n, dtype, dev):
    if t.dtype != dtype or t.get_device() != dev or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name}: expected {n} contiguous {dtype} on cuda:{dev}")
    return t.data_ptr()


def _status_word(status, dev):
    if status is None:
        return None
    if status.dtype != _host.i32 or status.get_device() != dev or status.numel() < 1:
        raise ValueError(f"status: expected int32 on cuda:{dev}")
    return status.data_ptr()


def _scratch(workspace, nbytes, like, dev):
    if workspace is None:
        return _host.empty(nbytes, device=like.device, dtype=_host.u8) if nbytes else None
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


def _table(t, n, dev):
    if t.dim() != 2 or t.shape[0] != n or t.dtype != _host.i32 or t.get_device() != dev or \
            (t.stride(1) != 1 and t.shape[1] != 1):
        raise ValueError(f"block_table: expected int32 ({n}, blocks) on cuda:{dev}")
    # a table of one row may report any stride; the rows must not overlap
    return t.data_ptr(), t.stride(0) if n > 1 else t.shape[1], t.shape[1]


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
    nbytes = h.batch_bytes(n, blocks * bt, D, Hq, Hkv, dt)
    ws = _scratch(workspace, nbytes, q, dev)
    _chk("b200_flash_attn_paged_batch", h.batch(
        q.data_ptr(), qs[0], qs[1], out.data_ptr(), os[0], os[1], pool, table, stride, blocks,
        _vector(seq_lens, "seq_lens", n, h.i32, dev), n, Hq, scale, None if ws is None else ws.data_ptr(), nbytes,
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
