"""memvanta_b200 -- B200 (sm_100a) implementation of MemVanta's GGUF
block-quantized matmul hot path, behind a C ABI (include/memvanta_b200.h).

This module is the Python host side over that ABI.  Its names mirror the
reference's C++ API so tests read like the reference's own:

* ``tensor_matvec``, ``tensor_matmul_batch``, ``tensor_matmul_batch_v06``,
  ``tensor_read_row_f32`` -- include/memvanta/gguf_kernels.hpp:25-30, with the
  reference's host-pointer contract (numpy in, numpy out);
* ``LlamaModel`` with ``forward`` / ``prefill`` / ``generate`` / ``reset`` /
  ``position`` / ``kv_bytes_allocated`` -- include/memvanta/llama_model.hpp:100-113.

Device-pointer entry points (``gemv``, ``gemm``, ``quantize_q8``, ...) take
torch CUDA tensors and run asynchronously on the given (or current) stream;
torch only provides device memory and streams here.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from ._lib import (F32, F16, BF16, Q4_0, Q8_0, Q6_K, ACT_F32, ACT_Q8, KV_F32, KV_F16, KV_Q8, KV_Q8_0,  # noqa: F401
                   KV_Q4_0, MV_ERR_TIMEOUT, ROPE_HALF, ROPE_INTERLEAVED, ROPE_SCALE_BANDS, ROPE_SCALE_LINEAR,
                   ROPE_SCALE_NONE, ROPE_SCALE_YARN, MemVantaError, check, load)

__all__ = [
    "init", "Weight", "tensor_matvec", "tensor_matmul_batch", "tensor_matmul_batch_v06", "tensor_read_row_f32",
    "gemv", "gemm", "quantize_q8", "q4_0_block_dots", "read_rows", "rmsnorm", "rope", "silu_mul", "add_inplace",
    "fp32_to_fp16", "kv_row_bytes", "kv_row_scales", "kv_append", "paged_attn_decode", "paged_attn_prefill",
    "rope_table", "rope_apply", "kv_pools", "rope_kv_append", "kv_read", "paged_attn_q4", "paged_attn_q4_prefill",
    "LlamaModel", "SequenceSet",
    "MemVantaError",
]


def init(device: int = 0) -> None:
    check(load().mv_init(device))


def _np_ptr(a: np.ndarray):
    return a.ctypes.data_as(C.c_void_p)


def _t_ptr(t):
    return None if t is None else t.data_ptr()


_torch_module = _current = _device = None


def _torch():
    """torch, imported with the first call that takes its tensors."""
    global _torch_module
    if _torch_module is None:
        import torch
        _torch_module = torch
    return _torch_module


def _current_device() -> int:
    """Index of the current GPU (torch.cuda.current_device() without its checks)."""
    global _device
    if _device is None:
        import torch
        torch.cuda.init()
        _device = torch._C._cuda_getDevice
    return _device()


def _current_stream():
    """Handle of the current device's current stream (torch.cuda.current_stream()
    builds an object around it: 3 us of a call that takes 10)."""
    global _current
    if _current is None:
        import torch
        torch.cuda.init()
        device, raw = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
        _current = lambda: raw(device())  # noqa: E731
    return _current()


def _stream(stream):
    if stream is None:
        return _current_stream()
    if isinstance(stream, int):
        return C.c_void_p(stream)
    return C.c_void_p(stream.cuda_stream)


class Weight:
    """One GGUF tensor resident in HBM (planar repack of its blocks)."""

    def __init__(self, handle, ggml_type: int, rows: int, cols: int):
        self._h = handle
        self.type, self.rows, self.cols = ggml_type, rows, cols

    @classmethod
    def upload(cls, blocks, ggml_type: int, rows: int, cols: int, stream=None) -> "Weight":
        """blocks: the tensor's raw GGML bytes (numpy uint8 / bytes / memoryview)."""
        buf = np.ascontiguousarray(np.frombuffer(blocks, dtype=np.uint8) if not isinstance(blocks, np.ndarray)
                                   else blocks.view(np.uint8).reshape(-1))
        h = C.c_void_p()
        s = C.c_void_p(0) if stream is None else _stream(stream)
        check(load().mv_weight_upload(_np_ptr(buf), buf.nbytes, ggml_type, rows, cols, s, C.byref(h)))
        return cls(h, ggml_type, rows, cols)

    @property
    def handle(self):
        return self._h

    def info(self) -> dict:
        t, r, c, b = C.c_int(), C.c_uint64(), C.c_uint64(), C.c_uint64()
        check(load().mv_weight_info(self._h, C.byref(t), C.byref(r), C.byref(c), C.byref(b)))
        return {"type": t.value, "rows": r.value, "cols": c.value, "device_bytes": b.value}

    def download(self) -> np.ndarray:
        from .gguf import tensor_nbytes
        n = tensor_nbytes(self.type, self.rows * self.cols)
        out = np.empty(n, np.uint8)
        check(load().mv_weight_download(self._h, _np_ptr(out), n))
        return out

    def free(self) -> None:
        if self._h:
            check(load().mv_weight_free(self._h))
            self._h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


# ------------------------------------------------ reference host contract

def tensor_matvec(w: Weight, x: np.ndarray) -> np.ndarray:
    """memvanta::tensor_matvec (src/gguf_kernels.cpp:244-253): host x -> host y."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    if x.size != w.cols:
        raise ValueError(f"x has {x.size} elements, tensor has {w.cols} columns")
    y = np.empty(w.rows, np.float32)
    check(load().mv_tensor_matvec_host(w.handle, _np_ptr(x), _np_ptr(y)))
    return y


def tensor_matmul_batch_v06(w: Weight, x: np.ndarray, force_q8: bool = False) -> np.ndarray:
    """memvanta::tensor_matmul_batch_v06 (src/gguf_kernels.cpp:261-271);
    force_q8 selects the MEMVANTA_FORCE_Q8_ACT=1 path."""
    x = np.ascontiguousarray(x, dtype=np.float32).reshape(-1, w.cols)
    y = np.empty((x.shape[0], w.rows), np.float32)
    check(load().mv_tensor_matmul_batch_host(w.handle, _np_ptr(x), _np_ptr(y), x.shape[0],
                                             ACT_Q8 if force_q8 else ACT_F32))
    return y


def tensor_matmul_batch(w: Weight, x: np.ndarray) -> np.ndarray:
    """memvanta::tensor_matmul_batch (src/gguf_kernels.cpp:255-259): fp32 activations."""
    return tensor_matmul_batch_v06(w, x, force_q8=False)


def tensor_read_row_f32(w: Weight, row: int) -> np.ndarray:
    """memvanta::tensor_read_row_f32 (src/gguf_kernels.cpp:226)."""
    out = np.empty(w.cols, np.float32)
    check(load().mv_tensor_read_row_host(w.handle, row, _np_ptr(out)))
    return out


# ------------------------------------------- device-pointer entry points

def gemv(w: Weight, x, y, stream=None) -> None:
    check(load().mv_gemv(w.handle, _t_ptr(x), _t_ptr(y), _stream(stream)))


def gemm(w: Weight, x, y, act_mode: int = ACT_Q8, stream=None) -> None:
    check(load().mv_gemm(w.handle, _t_ptr(x), x.shape[0] if x.dim() > 1 else 1, _t_ptr(y), act_mode,
                         _stream(stream)))


def stream_status(stream=None) -> None:
    """Synchronise the stream; raise MV_ERR_TIMEOUT if a tensor-core kernel
    gave up a bounded device-side wait since the last check."""
    check(load().mv_stream_status(_stream(stream)))


def test_gemm_stall(skip_commit_stage: int, wait_limit_us: int = 0) -> None:
    """Test hook: the next fp16 tensor-core GEMM launch leaves out one MMA
    commit and bounds its waits by wait_limit_us (mv_test_gemm_stall)."""
    check(load().mv_test_gemm_stall(skip_commit_stage, wait_limit_us))


def quantize_q8(x, stream=None):
    import torch
    rows, cols = (1, x.numel()) if x.dim() == 1 else tuple(x.shape)
    q = torch.empty((rows, cols), dtype=torch.int8, device=x.device)
    d = torch.empty((rows, cols // 32), dtype=torch.float32, device=x.device)
    check(load().mv_quantize_q8(_t_ptr(x), rows, cols, _t_ptr(q), _t_ptr(d), _stream(stream)))
    return q, d


# ---- internal (non-GGUF) block formats: device twins of quant.hpp / matmul.hpp
# Tensors are torch CUDA tensors; blocks are uint8 tensors of 20 (Q4_0) or 36
# (Q8_0) bytes per 32 elements.

def int_quantize_q8_0(x, stream=None):
    """quantize_q8_0 (src/quant.cpp:44-62) -> uint8[n/32*36]."""
    import torch
    out = torch.empty(x.numel() // 32 * 36, dtype=torch.uint8, device=x.device)
    check(load().mv_int_quantize_q8_0(_t_ptr(x), x.numel(), _t_ptr(out), _stream(stream)))
    return out


def int_quantize_q4_0(x, stream=None):
    """quantize_q4_0 (src/quant.cpp:64-85) -> uint8[n/32*20]."""
    import torch
    out = torch.empty(x.numel() // 32 * 20, dtype=torch.uint8, device=x.device)
    check(load().mv_int_quantize_q4_0(_t_ptr(x), x.numel(), _t_ptr(out), _stream(stream)))
    return out


def int_matvec_q4_q8(A20, x36, rows: int, cols: int, stream=None):
    import torch
    y = torch.empty(rows, dtype=torch.float32, device=A20.device)
    check(load().mv_int_matvec_q4_q8(_t_ptr(A20), _t_ptr(x36), _t_ptr(y), rows, cols, _stream(stream)))
    return y


def int_matvec_q4_0(A20, x, rows: int, cols: int, stream=None):
    import torch
    y = torch.empty(rows, dtype=torch.float32, device=A20.device)
    check(load().mv_int_matvec_q4_0(_t_ptr(A20), _t_ptr(x), _t_ptr(y), rows, cols, _stream(stream)))
    return y


def int_matvec_q8_0(A36, x, rows: int, cols: int, stream=None):
    import torch
    y = torch.empty(rows, dtype=torch.float32, device=A36.device)
    check(load().mv_int_matvec_q8_0(_t_ptr(A36), _t_ptr(x), _t_ptr(y), rows, cols, _stream(stream)))
    return y


def int_matmul_q4_0_batch(A20, x, rows: int, cols: int, batch: int, stream=None):
    import torch
    y = torch.empty((batch, rows), dtype=torch.float32, device=A20.device)
    check(load().mv_int_matmul_q4_0_batch(_t_ptr(A20), _t_ptr(x), _t_ptr(y), rows, cols, batch, _stream(stream)))
    return y


def matvec_f32(A, x, stream=None):
    import torch
    rows, cols = A.shape
    y = torch.empty(rows, dtype=torch.float32, device=A.device)
    check(load().mv_matvec_f32(_t_ptr(A), _t_ptr(x), _t_ptr(y), rows, cols, _stream(stream)))
    return y


def q4_0_block_dots(w: Weight, x, stream=None):
    import torch
    isum = torch.empty((w.rows, w.cols // 32), dtype=torch.int32, device=x.device)
    check(load().mv_q4_0_block_dots(w.handle, _t_ptr(x), _t_ptr(isum), _stream(stream)))
    return isum


def read_rows(w: Weight, rows, stream=None):
    import torch
    out = torch.empty((rows.numel(), w.cols), dtype=torch.float32, device=rows.device)
    check(load().mv_read_rows(w.handle, _t_ptr(rows), rows.numel(), _t_ptr(out), _stream(stream)))
    return out


def rmsnorm(x, w, eps: float, stream=None):
    import torch
    out = torch.empty_like(x)
    rows = 1 if x.dim() == 1 else x.shape[0]
    check(load().mv_rmsnorm(_t_ptr(x), _t_ptr(w), rows, x.shape[-1], eps, _t_ptr(out), _stream(stream)))
    return out


def rope(q, n_head: int, k, n_head_kv: int, head_dim: int, cos_t, sin_t, pos, stream=None) -> None:
    """In place on q [rows, n_head*hd] and k [rows, n_head_kv*hd]."""
    check(load().mv_rope(_t_ptr(q), n_head, _t_ptr(k), n_head_kv, head_dim, pos.numel(), _t_ptr(cos_t),
                         _t_ptr(sin_t), _t_ptr(pos), _stream(stream)))


def silu_mul(g, u, stream=None):
    import torch
    out = torch.empty_like(g)
    check(load().mv_silu_mul(_t_ptr(g), _t_ptr(u), _t_ptr(out), g.numel(), _stream(stream)))
    return out


def add_inplace(x, y, stream=None) -> None:
    check(load().mv_add_inplace(_t_ptr(x), _t_ptr(y), x.numel(), _stream(stream)))


def fp32_to_fp16(x, stream=None):
    import torch
    h = torch.empty(x.shape, dtype=torch.int16, device=x.device)
    check(load().mv_fp32_to_fp16(_t_ptr(x), _t_ptr(h), x.numel(), _stream(stream)))
    return h


def kv_row_bytes(kv_type: int, kv_dim: int) -> int:
    return load().mv_kv_row_bytes(kv_type, kv_dim)


def kv_row_scales(kv_type: int, kv_dim: int) -> int:
    return load().mv_kv_row_scales(kv_type, kv_dim)


def kv_append(kv_type, k, v, pos, block_table, max_pages, page, k_pages, v_pages, k_scales=None, v_scales=None,
              seq=None, stream=None) -> None:
    rows, kv_dim = k.shape
    check(load().mv_kv_append(kv_type, _t_ptr(k), _t_ptr(v), rows, kv_dim, _t_ptr(seq), _t_ptr(pos),
                              _t_ptr(block_table), max_pages, page, _t_ptr(k_pages), _t_ptr(v_pages),
                              _t_ptr(k_scales), _t_ptr(v_scales), _stream(stream)))


def paged_attn_decode(kv_type, q, n_head, n_head_kv, head_dim, k_pages, v_pages, block_table, max_pages, page,
                      ctx_len, max_ctx, k_scales=None, v_scales=None, out=None, stream=None):
    import torch
    n_seq = q.shape[0]
    if out is None:
        out = torch.empty((n_seq, n_head * head_dim), dtype=torch.float32, device=q.device)
    check(load().mv_paged_attn_decode(kv_type, _t_ptr(q), n_seq, n_head, n_head_kv, head_dim, _t_ptr(k_pages),
                                      _t_ptr(v_pages), _t_ptr(k_scales), _t_ptr(v_scales), _t_ptr(block_table),
                                      max_pages, page, _t_ptr(ctx_len), max_ctx, _t_ptr(out), _stream(stream)))
    return out


def paged_attn_decode_split(kv_type, q, n_head, n_head_kv, head_dim, k_pages, v_pages, block_table, max_pages,
                            page, ctx_len, max_ctx, k_scales=None, v_scales=None, out=None, stream=None):
    """paged_attn_decode split over the context (not bit-exact: ~1e-6)."""
    import torch
    n_seq = q.shape[0]
    if out is None:
        out = torch.empty((n_seq, n_head * head_dim), dtype=torch.float32, device=q.device)
    check(load().mv_paged_attn_decode_split(kv_type, _t_ptr(q), n_seq, n_head, n_head_kv, head_dim, _t_ptr(k_pages),
                                            _t_ptr(v_pages), _t_ptr(k_scales), _t_ptr(v_scales),
                                            _t_ptr(block_table), max_pages, page, _t_ptr(ctx_len), max_ctx,
                                            _t_ptr(out), _stream(stream)))
    return out


def paged_attn_prefill(kv_type, q, n_head, n_head_kv, head_dim, k_pages, v_pages, block_table, max_pages, page,
                       ctx_len, max_ctx, k_scales=None, v_scales=None, out=None, stream=None):
    """Attention of the query rows of one sequence (a prefill chunk): every
    row reads block-table row 0; row i sees ctx_len[i] tokens."""
    import torch
    n_q = q.shape[0]
    if out is None:
        out = torch.empty((n_q, n_head * head_dim), dtype=torch.float32, device=q.device)
    check(load().mv_paged_attn_prefill(kv_type, _t_ptr(q), n_q, n_head, n_head_kv, head_dim, _t_ptr(k_pages),
                                       _t_ptr(v_pages), _t_ptr(k_scales), _t_ptr(v_scales), _t_ptr(block_table),
                                       max_pages, page, _t_ptr(ctx_len), max_ctx, _t_ptr(out), _stream(stream)))
    return out


# ---- rotary positions and the 4-bit cache.  Activations are [rows, heads,
# head_dim] CUDA tensors (float32, float16 or bfloat16) whose heads may lie
# anywhere as long as a head's dimensions are next to one another.

_ACT = {}


def _act_type(t) -> int:
    if not _ACT:
        import torch
        _ACT.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16})
    try:
        return _ACT[t.dtype]
    except KeyError:
        raise MemVantaError(_lib.MV_ERR_UNSUPPORTED, f"activations must be float32, float16 or bfloat16, not {t.dtype}")


def _bad(msg: str):
    raise MemVantaError(_lib.MV_ERR_INVALID, msg)


def _on_gpu(x, *tensors):
    """Refuses tensors that are not all on the current GPU: the kernels would
    read and write addresses that are none of its memory.  (0.07 us a tensor.)"""
    at = x.get_device()
    for t in tensors:
        if t is not None and t.get_device() != at:
            _bad("tensors must be CUDA tensors, all of them on the current GPU")
    if at < 0 or at != _current_device():
        _bad("tensors must be CUDA tensors, all of them on the current GPU")


def _heads(name: str, t, rows: int | None = None, hd: int | None = None):
    """Row and head stride of an activation tensor, checked."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or (stride[2] != 1 and shape[2] > 1):
        _bad(f"{name} must be [rows, heads, head_dim] with a head's dimensions next to one another")
    if rows is not None and shape[0] != rows or hd is not None and shape[2] != hd:
        _bad(f"{name} is {tuple(shape)}: rows or head_dim differ from the other tensors'")
    return stride


def _i32(name: str, t, n: int | None = None):
    if t is None:
        return None
    if t.dtype is not _torch().int32 or not t.is_contiguous() or (n is not None and t.numel() != n):
        _bad(f"{name} must be a contiguous int32 tensor" + ("" if n is None else f" of {n} elements"))
    return t.data_ptr()


def _rope_tables(cos_t, sin_t, rot_dim, head_dim):
    """(rot_dim, rows of the tables); without tables nothing is rotated."""
    if cos_t is None and sin_t is None and not rot_dim:
        return 0, 0
    shape = () if cos_t is None else cos_t.shape
    if sin_t is None or len(shape) != 2 or sin_t.shape != shape or \
            not (cos_t.is_contiguous() and sin_t.is_contiguous()) or cos_t.dtype is not _torch().float32 or \
            sin_t.dtype is not cos_t.dtype:
        _bad("cos and sin must be contiguous float32 tables [n_pos, rot_dim / 2]")
    n_pos, half = shape
    if rot_dim is None:
        rot_dim = 2 * half
    if 2 * half != rot_dim or rot_dim > head_dim:
        _bad(f"the tables hold {half} angles per position: rot_dim {rot_dim}, head_dim {head_dim}")
    return rot_dim, n_pos


def rope_table(rot_dim: int, n_pos: int, theta: float = 10000.0, scaling: int = ROPE_SCALE_NONE, factor: float = 1.0,
               orig_ctx: float = 0.0, beta_fast: float = 32.0, beta_slow: float = 1.0, attn_factor: float = 0.0,
               freq_factors=None, device=None, stream=None):
    """cos and sin tables [n_pos, rot_dim / 2] (mv_rope_table)."""
    import torch
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    cos_t = torch.empty((n_pos, rot_dim // 2), dtype=torch.float32, device=dev)
    sin_t = torch.empty_like(cos_t)
    if freq_factors is not None and (freq_factors.dtype != torch.float32 or not freq_factors.is_contiguous()
                                     or freq_factors.numel() != rot_dim // 2):
        _bad("freq_factors must be a contiguous float32 tensor of rot_dim / 2 elements")
    _on_gpu(cos_t, freq_factors)
    check(load().mv_rope_table(rot_dim, n_pos, theta, scaling, factor, orig_ctx, beta_fast, beta_slow, attn_factor,
                               _t_ptr(freq_factors), _t_ptr(cos_t), _t_ptr(sin_t), _stream(stream)))
    return cos_t, sin_t


def rope_apply(x, cos_t, sin_t, pos, layout: int = ROPE_HALF, rot_dim: int | None = None, out=None, stream=None):
    """x [rows, heads, head_dim] with the first rot_dim (default: the tables'
    width) dimensions of each head rotated by its row's position; out may be x."""
    rows, n_head, hd = x.shape
    _on_gpu(x, cos_t, sin_t, pos, out)
    if out is None:
        import torch
        out = torch.empty((rows, n_head, hd), dtype=x.dtype, device=x.device)
    elif out.dtype != x.dtype or out.shape != x.shape:
        _bad("out must have x's shape and type")
    xs, os_ = _heads("x", x), _heads("out", out)
    rot_dim, n_pos = _rope_tables(cos_t, sin_t, rot_dim, hd)
    check(load().mv_rope_apply(_act_type(x), x.data_ptr(), xs[0], xs[1], out.data_ptr(), os_[0], os_[1], rows, n_head,
                               hd, rot_dim, layout, _t_ptr(cos_t), _t_ptr(sin_t), n_pos, _i32("pos", pos, rows),
                               _stream(stream)))
    return out


def kv_pools(kv_type: int, n_pages: int, page: int, n_head_kv: int, head_dim: int, device=None):
    """Empty (zeroed) pools (k_pages, v_pages, k_scales, v_scales) of a paged
    cache; the scales are None for the types that have none."""
    import torch
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    kv_dim, slots = n_head_kv * head_dim, n_pages * page
    shape, dtype = {KV_F32: ((n_pages, page, n_head_kv, head_dim), torch.float32),
                    KV_F16: ((n_pages, page, n_head_kv, head_dim), torch.float16),
                    KV_Q8: ((n_pages, page, n_head_kv, head_dim), torch.int8),
                    KV_Q8_0: ((n_pages, page, n_head_kv, head_dim), torch.int8),
                    KV_Q4_0: ((n_pages, n_head_kv, page, head_dim // 2), torch.uint8)}[kv_type]
    pages = [torch.zeros(shape, dtype=dtype, device=dev) for _ in range(2)]
    if kv_type == KV_Q4_0:
        scales = [torch.zeros((n_pages, n_head_kv, page, head_dim // 32), dtype=torch.bfloat16, device=dev)
                  for _ in range(2)]
    elif kv_type in (KV_Q8, KV_Q8_0):
        scales = [torch.zeros((slots, kv_row_scales(kv_type, kv_dim)), dtype=torch.float32, device=dev)
                  for _ in range(2)]
    else:
        scales = [None, None]
    return pages[0], pages[1], scales[0], scales[1]


_KV_ELEMENT = {KV_F32: 4, KV_F16: 2, KV_Q8: 1, KV_Q8_0: 1}


def _pool_pages(kv_type: int, pages, scales, page: int, n_head_kv: int, head_dim: int) -> int:
    """Pages that a pool's tensor holds, its scales checked against it."""
    if kv_type != KV_Q4_0 and kv_type not in _KV_ELEMENT:
        raise MemVantaError(_lib.MV_ERR_UNSUPPORTED, "unknown KV cache type")
    kv_dim = n_head_kv * head_dim
    if not pages.is_contiguous() or (scales is not None and not scales.is_contiguous()):
        _bad("cache pages and scales must be contiguous")
    per = page * kv_dim // 2 if kv_type == KV_Q4_0 else page * kv_dim * _KV_ELEMENT[kv_type]
    n = pages.nbytes // per if per else 0
    if kv_type >= KV_Q8 and scales is not None:
        need = n * page * (1 if kv_type == KV_Q8 else kv_dim // 32)
        if scales.numel() < need or scales.element_size() != (2 if kv_type == KV_Q4_0 else 4):
            _bad("the scale array does not fit the pages")
    return n


def _table(block_table):
    if block_table.dim() != 2:
        _bad("block_table must be [n_seq, max_pages]")
    return _i32("block_table", block_table), block_table.shape[0], block_table.shape[1]


def rope_kv_append(kv_type: int, q, k, v, cos_t, sin_t, pos, block_table, page: int, k_pages, v_pages, k_scales=None,
                   v_scales=None, seq=None, layout: int = ROPE_HALF, rot_dim: int | None = None, q_out=None,
                   stream=None):
    """Rotates q (may be None) into q_out and k into the paged cache, and stores
    v (mv_rope_kv_append); returns q_out.  Without tables nothing is rotated."""
    rows, n_head_kv, hd = k.shape
    _on_gpu(k, q, v, cos_t, sin_t, pos, block_table, k_pages, v_pages, k_scales, v_scales, seq, q_out)
    ks, vs = _heads("k", k), _heads("v", v, rows, hd)
    if v.shape[1] != n_head_kv or v.dtype != k.dtype or (q is not None and q.dtype != k.dtype):
        _bad("q, k and v must have one type, k and v the same heads")
    n_head, qs, os_ = 0, (0, 0), (0, 0)
    if q is not None:
        qs, n_head = _heads("q", q, rows, hd), q.shape[1]
        if q_out is None:
            import torch
            q_out = torch.empty((rows, n_head, hd), dtype=q.dtype, device=q.device)
        elif q_out.dtype != q.dtype or q_out.shape != q.shape:
            _bad("q_out must have q's shape and type")
        os_ = _heads("q_out", q_out)
    rot_dim, n_pos = _rope_tables(cos_t, sin_t, rot_dim, hd)
    n_pages = min(_pool_pages(kv_type, k_pages, k_scales, page, n_head_kv, hd),
                  _pool_pages(kv_type, v_pages, v_scales, page, n_head_kv, hd))
    table, n_seq, max_pages = _table(block_table)
    check(load().mv_rope_kv_append(
        kv_type, _act_type(k), None if q is None else q.data_ptr(), qs[0], qs[1],
        None if q is None else q_out.data_ptr(), os_[0], os_[1], n_head, k.data_ptr(), ks[0], ks[1], v.data_ptr(),
        vs[0], vs[1], n_head_kv, rows, hd, rot_dim, layout, _t_ptr(cos_t), _t_ptr(sin_t), n_pos,
        _i32("seq", seq, rows), _i32("pos", pos, rows), table, n_seq, max_pages, page, n_pages, k_pages.data_ptr(),
        v_pages.data_ptr(), _t_ptr(k_scales), _t_ptr(v_scales), _stream(stream)))
    return q_out


def kv_read(kv_type: int, pages, scales, pos, block_table, page: int, n_head_kv: int, head_dim: int, seq=None,
            dtype=None, out=None, stream=None):
    """Cached rows of one pool as the values they stand for: [rows, n_head_kv,
    head_dim] of dtype (default float32) (mv_kv_read)."""
    import torch
    rows = pos.numel()
    _on_gpu(pages, scales, pos, block_table, seq, out)
    if out is None:
        out = torch.empty((rows, n_head_kv, head_dim), dtype=dtype or torch.float32, device=pages.device)
    elif tuple(out.shape) != (rows, n_head_kv, head_dim) or not out.is_contiguous():
        _bad("out must be a contiguous [rows, n_head_kv, head_dim] tensor")
    n_pages = _pool_pages(kv_type, pages, scales, page, n_head_kv, head_dim)
    table, n_seq, max_pages = _table(block_table)
    check(load().mv_kv_read(kv_type, pages.data_ptr(), _t_ptr(scales), n_head_kv, head_dim, rows,
                            _i32("seq", seq, rows), _i32("pos", pos, rows), table, n_seq, max_pages, page, n_pages,
                            _act_type(out), out.data_ptr(), _stream(stream)))
    return out


def _q4_args(q, k_pages, v_pages, k_scales, v_scales, out, *arrays):
    """Checked (type, strides, sizes) of a 4-bit attention call; pools as kv_pools shapes them."""
    rows, n_head, hd = q.shape
    _on_gpu(q, k_pages, v_pages, k_scales, v_scales, out, *arrays)
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.shape[3] * 2 != hd:
        _bad("pools must be [n_pages, n_head_kv, page, head_dim / 2], the same for k and v")
    n_pages, n_head_kv, page, _ = k_pages.shape
    for p, s in ((k_pages, k_scales), (v_pages, v_scales)):
        if p.element_size() != 1 or s is None or _pool_pages(KV_Q4_0, p, s, page, n_head_kv, hd) != n_pages:
            _bad("pools must hold bytes, with their scales")
    if out is None:
        import torch
        out = torch.empty((rows, n_head, hd), dtype=q.dtype, device=q.device)
    elif out.dtype != q.dtype or out.shape != q.shape:
        _bad("out must have q's shape and type")
    qs, os_ = _heads("q", q), _heads("out", out)
    if n_head > 1 and (qs[1] != hd or os_[1] != hd):
        _bad("the heads of a query row must be next to one another")
    # a tensor of one row may carry any stride
    qr, orow = (n_head * hd, n_head * hd) if rows == 1 else (qs[0], os_[0])
    return out, _act_type(q), qr, orow, n_head, n_head_kv, hd, page, n_pages


def paged_attn_q4(q, k_pages, v_pages, k_scales, v_scales, block_table, ctx_len, max_ctx: int, scale: float = 0.0,
                  out=None, stream=None):
    """Attention over a 4-bit cache, one query row per sequence: q [n_seq,
    heads, head_dim], row i sees its first ctx_len[i] tokens (mv_paged_attn_q4)."""
    out, ty, qr, orow, n_head, n_head_kv, hd, page, n_pages = _q4_args(q, k_pages, v_pages, k_scales, v_scales, out,
                                                                       block_table, ctx_len)
    table, n_seq, max_pages = _table(block_table)
    if n_seq != q.shape[0]:
        _bad(f"the block table has {n_seq} sequences, q {q.shape[0]} rows")
    check(load().mv_paged_attn_q4(ty, q.data_ptr(), qr, n_seq, n_head, n_head_kv, hd, k_pages.data_ptr(),
                                  v_pages.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), table, max_pages, page,
                                  n_pages, _i32("ctx_len", ctx_len, n_seq), max_ctx, scale, out.data_ptr(), orow,
                                  _stream(stream)))
    return out


def paged_attn_q4_prefill(q, k_pages, v_pages, k_scales, v_scales, block_table, q_start, max_q: int, ctx_len,
                          max_ctx: int, scale: float = 0.0, out=None, stream=None):
    """The same for chunks of query rows: sequence s owns rows q_start[s] ..
    q_start[s + 1] of q, row r sees ctx_len[r] tokens (mv_paged_attn_q4_prefill)."""
    out, ty, qr, orow, n_head, n_head_kv, hd, page, n_pages = _q4_args(q, k_pages, v_pages, k_scales, v_scales, out,
                                                                       block_table, q_start, ctx_len)
    table, n_seq, max_pages = _table(block_table)
    check(load().mv_paged_attn_q4_prefill(ty, q.data_ptr(), qr, q.shape[0], n_head, n_head_kv, hd, k_pages.data_ptr(),
                                          v_pages.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), table, n_seq,
                                          max_pages, page, n_pages, _i32("q_start", q_start, n_seq + 1), max_q,
                                          _i32("ctx_len", ctx_len, q.shape[0]), max_ctx, scale, out.data_ptr(), orow,
                                          _stream(stream)))
    return out


from .model import LlamaModel, SequenceSet  # noqa: E402
