"""Host-side mirror of the xLLMs paged-attention operator interface.

Three layers, all calling the C ABI of libxpa.so (include/operator_api.h):

* :func:`nxt_paged_attention`, :func:`nxt_paged_attention_v2`,
  :func:`nxt_paged_attention_flash` — the reference's entry points
  (include/operator_api.h:63-115 of the xLLMs project) with the same
  argument names, order and meaning. Pointer arguments accept torch CUDA
  tensors or raw device addresses. Unlike the reference (which returns
  nothing and checks nothing), a rejected call raises :class:`PagedAttentionError`.
* :func:`paged_attention` — tensor-level convenience over the status-returning
  ``nxt_paged_attention_ex`` that derives sizes and strides from the tensors.
* :class:`CudaBackendPlugin` — the dlopen'd plugin path
  (backends/cuda_backend.c:35-120), driven the way the reference's backend
  manager drives it (src/core/backend_manager.c:264-344).

torch is used for device memory and streams only; all arithmetic happens in
the native kernels.
"""
from __future__ import annotations

import contextlib
import ctypes
import math
from typing import Optional, Union

from . import _native

Pointer = Union[int, None, "torch.Tensor"]  # noqa: F821


class PagedAttentionError(RuntimeError):
    def __init__(self, code: int, where: str):
        self.code = code
        super().__init__(f"{where}: {_native.strerror(code)} ({code})")


def _ptr(x: Pointer) -> Optional[int]:
    if x is None:
        return None
    if isinstance(x, int):
        return x
    return x.data_ptr()


def _stream_ptr(stream) -> Optional[int]:
    if stream is None:
        try:
            import torch
            if torch.cuda.is_available() and torch.cuda.is_initialized():
                return torch.cuda.current_stream().cuda_stream
        except ImportError:  # pragma: no cover
            pass
        return None
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def _dropin(name: str, out, query, key_cache, value_cache, block_tables, seq_lens,
            num_seqs, num_heads, head_size, num_kv_heads, scale, max_num_blocks_per_seq,
            block_size, dtype_size, kv_block_stride, kv_head_stride, stream=None) -> None:
    lib = _native.xpa()
    getattr(lib, name)(
        _ptr(out), _ptr(query), _ptr(key_cache), _ptr(value_cache), _ptr(block_tables),
        _ptr(seq_lens), int(num_seqs), int(num_heads), int(head_size), int(num_kv_heads),
        float(scale), int(max_num_blocks_per_seq), int(block_size), int(dtype_size),
        int(kv_block_stride), int(kv_head_stride), _stream_ptr(stream))
    rc = lib.nxt_paged_attention_last_error()
    if rc != _native.NXT_PA_OK:
        raise PagedAttentionError(rc, name)


def nxt_paged_attention(out, query, key_cache, value_cache, block_tables, seq_lens,
                        num_seqs, num_heads, head_size, num_kv_heads, scale,
                        max_num_blocks_per_seq, block_size, dtype_size, kv_block_stride,
                        kv_head_stride, stream=None) -> None:
    """Reference ``nxt_paged_attention`` (operators/page_attention.cu:170)."""
    _dropin("nxt_paged_attention", out, query, key_cache, value_cache, block_tables, seq_lens,
            num_seqs, num_heads, head_size, num_kv_heads, scale, max_num_blocks_per_seq,
            block_size, dtype_size, kv_block_stride, kv_head_stride, stream)


def nxt_paged_attention_v2(out, query, key_cache, value_cache, block_tables, seq_lens,
                           num_seqs, num_heads, head_size, num_kv_heads, scale,
                           max_num_blocks_per_seq, block_size, dtype_size, kv_block_stride,
                           kv_head_stride, stream=None) -> None:
    """Reference ``nxt_paged_attention_v2`` (operators/page_attention_v2.cu:262)."""
    _dropin("nxt_paged_attention_v2", out, query, key_cache, value_cache, block_tables,
            seq_lens, num_seqs, num_heads, head_size, num_kv_heads, scale,
            max_num_blocks_per_seq, block_size, dtype_size, kv_block_stride, kv_head_stride,
            stream)


def nxt_paged_attention_flash(out, query, key_cache, value_cache, block_tables, seq_lens,
                              num_seqs, num_heads, head_size, num_kv_heads, scale,
                              max_num_blocks_per_seq, block_size, dtype_size, kv_block_stride,
                              kv_head_stride, stream=None) -> None:
    """Reference ``nxt_paged_attention_flash`` (operators/flashinfer_adapter.cu:329)."""
    _dropin("nxt_paged_attention_flash", out, query, key_cache, value_cache, block_tables,
            seq_lens, num_seqs, num_heads, head_size, num_kv_heads, scale,
            max_num_blocks_per_seq, block_size, dtype_size, kv_block_stride, kv_head_stride,
            stream)


def _dtype_size(t) -> int:
    import torch
    if t.dtype == torch.float16:
        return 2
    if t.dtype == torch.float32:
        return 4
    raise PagedAttentionError(_native.NXT_PA_EINVAL, f"dtype {t.dtype}")


def _check_attention_inputs(where, query, key_cache, value_cache, block_tables, seq_lens, out,
                            one_byte=False):
    """Host checks before any pointer reaches the C ABI: ranks, shapes, dtypes,
    contiguity and device. The kernels read raw pointers in the reference
    layout, so a mismatch there would be misread, not reported."""
    import torch

    def bad(msg):
        raise PagedAttentionError(_native.NXT_PA_EINVAL, f"{where}: {msg}")
    if query.dim() != 3 or key_cache.dim() != 4:
        bad("query must be [B, Hq, D] and the pools [num_blocks, Hkv, block_size, D]")
    B, Hq, D = query.shape
    if key_cache.shape[3] != D or tuple(value_cache.shape) != tuple(key_cache.shape):
        bad("cache shapes")
    if one_byte:
        if query.dtype != torch.float16:
            bad("query must be fp16")
        if key_cache.element_size() != 1 or value_cache.element_size() != 1:
            bad("one-byte pools must be 1-byte tensors")
    else:
        _dtype_size(query)
        if key_cache.dtype != query.dtype or value_cache.dtype != query.dtype:
            bad("the K/V pools must have the query's dtype")
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or block_tables.shape[0] < B:
        bad("block_tables must be int32 [B, max_blocks]")
    if seq_lens.dtype != torch.int32 or seq_lens.numel() < B:
        bad("seq_lens must be int32 [B]")
    ts = [query, key_cache, value_cache, block_tables, seq_lens]
    if out is not None:
        if tuple(out.shape) != tuple(query.shape) or out.dtype != query.dtype:
            bad("out must have the query's shape and dtype")
        ts.append(out)
    if not all(t.is_contiguous() for t in ts):
        bad("non-contiguous input")
    if not all(t.is_cuda and t.device == query.device for t in ts):
        bad("every tensor must be on the query's CUDA device")


def paged_attention(query, key_cache, value_cache, block_tables, seq_lens, *,
                    scale: Optional[float] = None, out=None, num_blocks: Optional[int] = None,
                    workspace=None, device_status=None, stream=None):
    """Decode attention of one new token per sequence over a paged KV cache.

    query [B, Hq, D]; key_cache/value_cache [num_blocks, Hkv, block_size, D]
    (contiguous, the reference layout); block_tables [B, max_blocks] int32;
    seq_lens [B] int32; all on the same CUDA device. Returns out [B, Hq, D] in
    query's dtype. ``scale`` defaults to 1/sqrt(D). ``num_blocks`` defaults to
    key_cache.shape[0], which lets the kernels mask out-of-range pages.
    """
    import torch
    _check_attention_inputs("paged_attention", query, key_cache, value_cache, block_tables,
                            seq_lens, out)
    B, Hq, D = query.shape
    nb, Hkv, bs, _ = key_cache.shape
    if out is None:
        out = torch.empty_like(query)
    ds = _dtype_size(query)
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    ws_bytes = 0
    if workspace is not None:
        ws_bytes = workspace.numel() * workspace.element_size()
    rc = _native.xpa().nxt_paged_attention_ex(
        _ptr(out), _ptr(query), _ptr(key_cache), _ptr(value_cache), _ptr(block_tables),
        _ptr(seq_lens), B, Hq, D, Hkv, float(scale), block_tables.shape[1], bs, ds,
        Hkv * bs * D, bs * D, nb if num_blocks is None else int(num_blocks),
        _ptr(workspace), ws_bytes, _ptr(device_status), _stream_ptr(stream))
    if rc != _native.NXT_PA_OK:
        raise PagedAttentionError(rc, "nxt_paged_attention_ex")
    return out


def workspace_size(num_seqs, num_heads, head_size, num_kv_heads, max_num_blocks_per_seq,
                   block_size=16, dtype_size=2) -> int:
    return int(_native.xpa().nxt_paged_attention_workspace_size(
        num_seqs, num_heads, head_size, num_kv_heads, max_num_blocks_per_seq, block_size,
        dtype_size))


def kernel_path(key_cache, value_cache, num_heads, head_size, num_kv_heads, block_size,
                dtype_size, kv_block_stride, kv_head_stride) -> int:
    """NXT_PA_PATH_* the kernels take for these arguments."""
    return int(_native.xpa().nxt_paged_attention_path(
        _ptr(key_cache), _ptr(value_cache), num_heads, head_size, num_kv_heads, block_size,
        dtype_size, kv_block_stride, kv_head_stride))


def device_status(clear: bool = True) -> int:
    """NXT_PA_DEV_* bits of the current device's library status word."""
    rc = _native.xpa().nxt_paged_attention_device_status(1 if clear else 0)
    if rc < 0:
        raise PagedAttentionError(rc, "nxt_paged_attention_device_status")
    return rc


# ── plugin path ───────────────────────────────────────────────────────────
class NxtBackend(ctypes.Structure):
    """Layout of the reference's NxtBackend (include/backend.h:141-151)."""
    _fields_ = [
        ("name", ctypes.c_char_p),
        ("so_path", ctypes.c_char_p),
        ("dl_handle", ctypes.c_void_p),
        ("api", ctypes.c_void_p * 8),
        ("state", ctypes.c_int),
        ("priority", ctypes.c_int32),
        ("model_count", ctypes.c_uint32),
        ("models", ctypes.c_void_p),
        ("backend_state", ctypes.c_void_p),
    ]


class NxtPagedAttentionInput(ctypes.Structure):
    """Layout of the reference's NxtPagedAttentionInput (backends/cuda_backend.h:29-46)."""
    _fields_ = [
        ("query", ctypes.c_void_p),
        ("key_cache", ctypes.c_void_p),
        ("value_cache", ctypes.c_void_p),
        ("block_tables", ctypes.c_void_p),
        ("seq_lens", ctypes.c_void_p),
        ("num_seqs", ctypes.c_int),
        ("num_heads", ctypes.c_int),
        ("head_size", ctypes.c_int),
        ("num_kv_heads", ctypes.c_int),
        ("scale", ctypes.c_float),
        ("max_num_blocks_per_seq", ctypes.c_int),
        ("block_size", ctypes.c_int),
        ("dtype_size", ctypes.c_int),
        ("kv_block_stride", ctypes.c_int),
        ("kv_head_stride", ctypes.c_int),
        ("stream", ctypes.c_void_p),
    ]


NXT_BACKEND_STATE_UNINITIALIZED = 0
NXT_BACKEND_STATE_READY = 2


class CudaBackendPlugin:
    """libxllm_cuda_backend.so driven like the reference backend manager does:
    init on load, run(input descriptor, output), fini on unload."""

    def __init__(self, name: str = "cuda"):
        self.lib = _native.plugin()
        self.backend = NxtBackend()
        self.backend.name = name.encode()
        self.backend.so_path = _native.PLUGIN_PATH.encode()
        rc = self.lib.nxt_backend_init(ctypes.byref(self.backend))
        if rc != 0:
            raise PagedAttentionError(_native.NXT_PA_ECUDA, "nxt_backend_init")

    def run(self, pa: NxtPagedAttentionInput, output: Pointer) -> int:
        return int(self.lib.nxt_backend_run(ctypes.byref(self.backend), ctypes.byref(pa),
                                            _ptr(output)))

    def close(self) -> int:
        return int(self.lib.nxt_backend_fini(ctypes.byref(self.backend)))


def make_input(query, key_cache, value_cache, block_tables, seq_lens, scale=None,
               stream=None) -> NxtPagedAttentionInput:
    """Fills the plugin's input descriptor from tensors in the reference layout."""
    B, Hq, D = query.shape
    nb, Hkv, bs, _ = key_cache.shape
    pa = NxtPagedAttentionInput()
    pa.query = _ptr(query)
    pa.key_cache = _ptr(key_cache)
    pa.value_cache = _ptr(value_cache)
    pa.block_tables = _ptr(block_tables)
    pa.seq_lens = _ptr(seq_lens)
    pa.num_seqs, pa.num_heads, pa.head_size, pa.num_kv_heads = B, Hq, D, Hkv
    pa.scale = 1.0 / math.sqrt(D) if scale is None else scale
    pa.max_num_blocks_per_seq = block_tables.shape[1]
    pa.block_size = bs
    pa.dtype_size = _dtype_size(query)
    pa.kv_block_stride = Hkv * bs * D
    pa.kv_head_stride = bs * D
    pa.stream = _stream_ptr(stream)
    return pa


# ── KV append ─────────────────────────────────────────────────────────────
def _index_ok(slot_mapping, n, like) -> bool:
    """slot_mapping: contiguous int64 with >= n entries on `like`'s device."""
    import torch
    return (slot_mapping.dtype == torch.int64 and slot_mapping.is_contiguous()
            and slot_mapping.numel() >= n and slot_mapping.device == like.device)


def reshape_and_cache(key, value, key_cache, value_cache, slot_mapping, stream=None) -> None:
    """Scatter key/value [T, Hkv, D] into the pools [NB, Hkv, P, D] at
    slot_mapping[t] (int64; page = slot // P, slot % P; negative: skipped)."""
    T, Hkv, D = key.shape
    nb, hk, bs, dk = key_cache.shape
    if (hk != Hkv or dk != D or tuple(value.shape) != tuple(key.shape)
            or tuple(value_cache.shape) != tuple(key_cache.shape)
            or not (key_cache.is_contiguous() and value_cache.is_contiguous())
            or key.stride(2) != 1 or key.stride(1) != D or value.stride() != key.stride()
            or key.dtype != key_cache.dtype or value.dtype != key_cache.dtype
            or value_cache.dtype != key_cache.dtype
            or not _index_ok(slot_mapping, T, key) or not key.is_cuda
            or len({t.device for t in (key, value, key_cache, value_cache)}) != 1):
        raise PagedAttentionError(_native.NXT_PA_EINVAL, "reshape_and_cache: shapes")
    rc = _native.xpa().nxt_reshape_and_cache(
        _ptr(key), _ptr(value), _ptr(key_cache), _ptr(value_cache), _ptr(slot_mapping), T, Hkv, D,
        bs, _dtype_size(key), Hkv * bs * D, bs * D, key.stride(0), _stream_ptr(stream))
    if rc != _native.NXT_PA_OK:
        raise PagedAttentionError(rc, "nxt_reshape_and_cache")


def paged_attention_append(query, key_cache, value_cache, block_tables, seq_lens, new_key,
                           new_value, slot_mapping, *, scale=None, out=None, num_blocks=None,
                           device_status=None, stream=None):
    """One decode step with the KV append fused in: new_key/new_value
    [B, Hkv, D] are written at slot_mapping[b] and included in the attention
    (seq_lens count them)."""
    import torch
    _check_attention_inputs("paged_attention_append", query, key_cache, value_cache,
                            block_tables, seq_lens, out)
    B, Hq, D = query.shape
    nb, Hkv, bs, _ = key_cache.shape
    if (tuple(new_key.shape) != (B, Hkv, D) or tuple(new_value.shape) != (B, Hkv, D)
            or new_key.dtype != query.dtype or new_value.dtype != query.dtype
            or not (new_key.is_contiguous() and new_value.is_contiguous())
            or not _index_ok(slot_mapping, B, query) or new_key.device != query.device
            or new_value.device != query.device):
        raise PagedAttentionError(_native.NXT_PA_EINVAL, "paged_attention_append: shapes")
    if out is None:
        out = torch.empty_like(query)
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    rc = _native.xpa().nxt_paged_attention_append_ex(
        _ptr(out), _ptr(query), _ptr(key_cache), _ptr(value_cache), _ptr(block_tables),
        _ptr(seq_lens), _ptr(new_key), _ptr(new_value), _ptr(slot_mapping), B, Hq, D, Hkv,
        float(scale), block_tables.shape[1], bs, _dtype_size(query), Hkv * bs * D, bs * D,
        nb if num_blocks is None else int(num_blocks), _ptr(device_status), _stream_ptr(stream))
    if rc != _native.NXT_PA_OK:
        raise PagedAttentionError(rc, "nxt_paged_attention_append_ex")
    return out


# ── shared-prefix (cascade) attention ─────────────────────────────────────
class PrefixGroups:
    """Device arrays of nxt_paged_attention_prefix_ex, built once from a host
    list of (member sequence ids, shared prefix pages) pairs."""

    def __init__(self, groups, num_seqs, device=None, *, prefix_pages=None, offsets=None,
                 members=None, bounds=None):
        import torch
        if bounds is not None:  # (num_groups, max_group_size, max_prefix_pages)
            self.num_groups, self.max_group_size, self.max_prefix_pages = (int(x) for x in bounds)
        else:
            self.num_groups = len(groups)
            self.max_group_size = max((len(m) for m, _ in groups), default=0)
            self.max_prefix_pages = max((int(p) for _, p in groups), default=0)
        if prefix_pages is None:
            pp, off, mem = self.host_arrays(groups, num_seqs)
            t = lambda x: torch.from_numpy(x).to(device)
            prefix_pages, offsets, members = t(pp), t(off), t(mem)
        self.prefix_pages, self.offsets, self.members = prefix_pages, offsets, members

    @staticmethod
    def host_arrays(groups, num_seqs):
        """(prefix_pages [num_seqs], offsets [G+1], members [sum of sizes]) as int32."""
        import numpy as np
        pp = np.zeros(max(1, num_seqs), dtype=np.int32)
        off = [0]
        mem = []
        for seqs, pages in groups:
            for b in seqs:
                if not 0 <= int(b) < num_seqs:
                    raise ValueError(f"group member {b} outside the batch")
                if pp[int(b)]:
                    raise ValueError(f"sequence {b} is in two prefix groups")
                pp[int(b)] = int(pages)
            mem.extend(int(b) for b in seqs)
            off.append(len(mem))
        return (pp, np.asarray(off, dtype=np.int32),
                np.asarray(mem if mem else [0], dtype=np.int32))


def paged_attention_prefix(query, key_cache, value_cache, block_tables, seq_lens, groups, *,
                           scale=None, out=None, num_blocks=None, device_status=None,
                           stream=None):
    """Decode attention for a batch with shared prefixes. `groups` is a
    PrefixGroups or a host list of (member sequence ids, shared prefix pages);
    every member's seq_len covers its prefix and its block-table row starts
    with the group's shared pages. The result equals paged_attention's."""
    import torch
    _check_attention_inputs("paged_attention_prefix", query, key_cache, value_cache,
                            block_tables, seq_lens, out)
    B, Hq, D = query.shape
    nb, Hkv, bs, _ = key_cache.shape
    if not isinstance(groups, PrefixGroups):
        groups = PrefixGroups(groups, B, query.device)
    if out is None:
        out = torch.empty_like(query)
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    rc = _native.xpa().nxt_paged_attention_prefix_ex(
        _ptr(out), _ptr(query), _ptr(key_cache), _ptr(value_cache), _ptr(block_tables),
        _ptr(seq_lens), _ptr(groups.prefix_pages), _ptr(groups.offsets), _ptr(groups.members),
        groups.num_groups, groups.max_group_size, groups.max_prefix_pages, B, Hq, D, Hkv,
        float(scale), block_tables.shape[1], bs, _dtype_size(query), Hkv * bs * D, bs * D,
        nb if num_blocks is None else int(num_blocks), None, 0, _ptr(device_status),
        _stream_ptr(stream))
    if rc != _native.NXT_PA_OK:
        raise PagedAttentionError(rc, "nxt_paged_attention_prefix_ex")
    return out


# ── activations (operators/activation_kernels.cu of the reference) ─────────
ACTIVATIONS = {
    "silu_and_mul": _native.NXT_ACT_SILU_AND_MUL,
    "mul_and_silu": _native.NXT_ACT_MUL_AND_SILU,
    "gelu_and_mul": _native.NXT_ACT_GELU_AND_MUL,
    "gelu_tanh_and_mul": _native.NXT_ACT_GELU_TANH_AND_MUL,
    "gelu": _native.NXT_ACT_GELU,
    "silu": _native.NXT_ACT_SILU,
}


def activation(name, x, *, out=None, stream=None):
    """Gated ops take x [..., 2d] ([gate | up]) and return [..., d]; the
    element-wise ops (gelu, silu) keep x's shape. fp16 or fp32, contiguous."""
    import torch
    op = ACTIVATIONS[name]
    if not x.is_contiguous():
        raise ValueError("activation input must be contiguous")
    gated = op <= _native.NXT_ACT_GELU_TANH_AND_MUL
    width = x.shape[-1]
    if gated and width % 2:
        raise ValueError("gated activation input needs an even last dimension")
    d = width // 2 if gated else width
    rows = x.numel() // width if width else 0
    if out is None:
        out = torch.empty(tuple(x.shape[:-1]) + (d,), dtype=x.dtype, device=x.device)
    elif out.numel() != rows * d or out.dtype != x.dtype or not out.is_contiguous():
        raise ValueError("activation output does not match the input")
    rc = _native.xpa().nxt_activation_ex(op, _ptr(out), _ptr(x), rows, d, _dtype_size(x),
                                         _stream_ptr(stream))
    if rc != _native.NXT_PA_OK:
        raise PagedAttentionError(rc, "nxt_activation_ex")
    return out


# ── one-byte KV cache (fp8 E4M3 / E5M2, int8) ──────────────────────────────
FP8_FORMATS = {"e4m3": _native.NXT_KV_FP8_E4M3, "e5m2": _native.NXT_KV_FP8_E5M2,
               "int8": _native.NXT_KV_INT8}


def _fp8_code(fmt):
    return FP8_FORMATS[fmt] if isinstance(fmt, str) else int(fmt)


def paged_attention_fp8(query, key_cache, value_cache, block_tables, seq_lens, fmt, k_scale,
                        v_scale, *, scale=None, out=None, num_blocks=None, workspace=None,
                        device_status=None, stream=None):
    """Decode attention over one-byte pools (uint8 / int8 / float8 tensors
    [NB, Hkv, P, D] holding encode(x / scale) in format `fmt`: "e4m3", "e5m2"
    or "int8"); query and output fp16 [B, Hq, D]."""
    import torch
    _check_attention_inputs("paged_attention_fp8", query, key_cache, value_cache, block_tables,
                            seq_lens, out, one_byte=True)
    B, Hq, D = query.shape
    nb, Hkv, bs, _ = key_cache.shape
    if out is None:
        out = torch.empty_like(query)
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    ws_ptr, ws_bytes = (None, 0) if workspace is None else (_ptr(workspace),
                                                            workspace.numel() * workspace.element_size())
    rc = _native.xpa().nxt_paged_attention_fp8_ex(
        _ptr(out), _ptr(query), _ptr(key_cache), _ptr(value_cache), _ptr(block_tables),
        _ptr(seq_lens), B, Hq, D, Hkv, float(scale), block_tables.shape[1], bs, _fp8_code(fmt),
        float(k_scale), float(v_scale), Hkv * bs * D, bs * D,
        nb if num_blocks is None else int(num_blocks), ws_ptr, ws_bytes, _ptr(device_status),
        _stream_ptr(stream))
    if rc != _native.NXT_PA_OK:
        raise PagedAttentionError(rc, "nxt_paged_attention_fp8_ex")
    return out


def reshape_and_cache_fp8(key, value, key_cache, value_cache, slot_mapping, fmt, k_scale, v_scale,
                          stream=None) -> None:
    """Quantise fp16 key/value [T, Hkv, D] into the one-byte pools
    [NB, Hkv, P, D] (format `fmt`) at slot_mapping[t] (int64; negative:
    skipped)."""
    import torch
    T, Hkv, D = key.shape
    nb, hk, bs, dk = key_cache.shape
    if (hk != Hkv or dk != D or tuple(value.shape) != tuple(key.shape)
            or tuple(value_cache.shape) != tuple(key_cache.shape)
            or key_cache.element_size() != 1 or value_cache.element_size() != 1
            or not (key_cache.is_contiguous() and value_cache.is_contiguous())
            or key.stride(2) != 1 or key.stride(1) != D or value.stride() != key.stride()
            or key.dtype != torch.float16 or value.dtype != torch.float16
            or not _index_ok(slot_mapping, T, key) or not key.is_cuda
            or len({t.device for t in (key, value, key_cache, value_cache)}) != 1):
        raise PagedAttentionError(_native.NXT_PA_EINVAL, "reshape_and_cache_fp8: shapes")
    rc = _native.xpa().nxt_reshape_and_cache_fp8(
        _ptr(key), _ptr(value), _ptr(key_cache), _ptr(value_cache), _ptr(slot_mapping), T, Hkv, D,
        bs, _fp8_code(fmt), float(k_scale), float(v_scale), Hkv * bs * D, bs * D, key.stride(0),
        _stream_ptr(stream))
    if rc != _native.NXT_PA_OK:
        raise PagedAttentionError(rc, "nxt_reshape_and_cache_fp8")


def paged_attention_fp8_append(query, key_cache, value_cache, block_tables, seq_lens, new_key,
                               new_value, slot_mapping, fmt, k_scale, v_scale, *, scale=None,
                               out=None, num_blocks=None, device_status=None, stream=None):
    """One decode step on one-byte pools with the quantising append fused in:
    new_key/new_value (fp16 [B, Hkv, D]) are stored at slot_mapping[b] in
    format `fmt` and included in the attention (seq_lens count them)."""
    import torch
    _check_attention_inputs("paged_attention_fp8_append", query, key_cache, value_cache,
                            block_tables, seq_lens, out, one_byte=True)
    B, Hq, D = query.shape
    nb, Hkv, bs, _ = key_cache.shape
    if (tuple(new_key.shape) != (B, Hkv, D) or tuple(new_value.shape) != (B, Hkv, D)
            or new_key.dtype != torch.float16 or new_value.dtype != torch.float16
            or not (new_key.is_contiguous() and new_value.is_contiguous())
            or not _index_ok(slot_mapping, B, query) or new_key.device != query.device
            or new_value.device != query.device):
        raise PagedAttentionError(_native.NXT_PA_EINVAL, "paged_attention_fp8_append: shapes")
    if out is None:
        out = torch.empty_like(query)
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    rc = _native.xpa().nxt_paged_attention_fp8_append_ex(
        _ptr(out), _ptr(query), _ptr(key_cache), _ptr(value_cache), _ptr(block_tables),
        _ptr(seq_lens), _ptr(new_key), _ptr(new_value), _ptr(slot_mapping), B, Hq, D, Hkv,
        float(scale), block_tables.shape[1], bs, _fp8_code(fmt), float(k_scale), float(v_scale),
        Hkv * bs * D, bs * D, nb if num_blocks is None else int(num_blocks),
        _ptr(device_status), _stream_ptr(stream))
    if rc != _native.NXT_PA_OK:
        raise PagedAttentionError(rc, "nxt_paged_attention_fp8_append_ex")
    return out


# ── 4-bit KV cache ─────────────────────────────────────────────────────────
# The calls below take microseconds on the device for a decode step, so what the
# host does per call counts: native functions are looked up once, and devices
# are compared by index (-1: not CUDA).
_functions = {}


def _native_call(name, *args):
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(_native.xpa(), name)
    rc = fn(*args)
    if rc != _native.NXT_PA_OK:
        raise PagedAttentionError(rc, name)


def _launch_on(device, stream):
    """(stream pointer, what to close after the call or None): `device` is
    current until then, and tensors made until then belong to the stream, so
    that the allocator gives their memory to no one else while kernels run."""
    import torch
    if stream is None and torch._C._cuda_getDevice() == device:
        return torch._C._cuda_getCurrentRawStream(device), None
    leave = contextlib.ExitStack()
    leave.enter_context(torch.cuda.device(device))
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(device), leave
    if isinstance(stream, int):
        # a raw 0 is the legacy default stream, which torch calls its default
        stream = (torch.cuda.ExternalStream(stream, device=device) if stream
                  else torch.cuda.default_stream(device))
    leave.enter_context(torch.cuda.stream(stream))
    return stream.cuda_stream, leave


def _refuse(where, msg):
    raise PagedAttentionError(_native.NXT_PA_EINVAL, f"{where}: {msg}")


def _known_blocks(where, given, nb):
    """num_blocks of a call: the pools' own by default; <= 0: page ids are not checked."""
    if given is None:
        return nb
    if given > nb:
        _refuse(where, f"num_blocks {given} of pools with {nb}")
    return given


def _opt_ptr(t):
    return None if t is None else t.data_ptr()


def q4_pool_shape(num_blocks, num_kv_heads, block_size, head_size):
    """Shape of a 4-bit K or V pool (uint8): [num_blocks, Hkv, block_size / 16,
    9 * head_size], one row of bytes per 16 tokens (include/operator_api.h)."""
    if block_size <= 0 or block_size % 16 or head_size <= 0 or head_size % 16 or head_size > 256:
        _refuse("q4_pool_shape", "block_size and head_size must be multiples of 16, head_size at "
                "most 256")
    return (num_blocks, num_kv_heads, block_size // 16, 9 * head_size)


def _q4_dims(where, key_cache, value_cache, device):
    """(num_blocks, Hkv, block size, head size, page and head strides) of 4-bit pools."""
    import torch
    shape = key_cache.shape
    if (len(shape) != 4 or value_cache.shape != shape or key_cache.dtype != torch.uint8
            or value_cache.dtype != torch.uint8 or shape[3] % 144 or not 0 < shape[3] <= 2304
            or not key_cache.is_contiguous() or not value_cache.is_contiguous() or device < 0
            or key_cache.get_device() != device or value_cache.get_device() != device):
        _refuse(where, "4-bit pools must be contiguous uint8 [num_blocks, Hkv, block_size / 16, "
                "9 * head_size] on one CUDA device")
    nb, hkv, spp, tile = shape
    return nb, hkv, 16 * spp, tile // 9, hkv * spp * tile, spp * tile


def _row_stride(where, key, value, slots, heads, dim, device):
    """Token stride of key and value rows [T, Hkv, D]. Strides of a dimension of
    one element reach no address and may be anything."""
    import torch
    T = key.shape[0] if key.dim() == 3 else -1
    if (key.shape != (T, heads, dim) or value.shape != key.shape or key.dtype != torch.float16
            or value.dtype != torch.float16 or slots.dtype != torch.int64 or slots.numel() < T
            or not slots.is_contiguous() or device < 0 or key.get_device() != device
            or value.get_device() != device or slots.get_device() != device):
        _refuse(where, "rows must be fp16 [T, Hkv, D] and slot_mapping int64 [T], on the pools' "
                "CUDA device")
    ks, vs = key.stride(), value.stride()
    if T and (ks[2] != 1 or vs[2] != 1 or (heads > 1 and (ks[1] != dim or vs[1] != dim))
              or (T > 1 and (ks[0] != vs[0] or ks[0] < heads * dim))):
        _refuse(where, "rows must have dense heads, and key and value one token stride")
    return ks[0] if T > 1 else heads * dim


def reshape_and_cache_q4(key, value, key_cache, value_cache, slot_mapping, k_scale, v_scale,
                         stream=None) -> None:
    """Quantise fp16 key/value [T, Hkv, D] into 4-bit pools (q4_pool_shape) at
    slot_mapping[t] (int64; negative or past the pools: skipped; distinct)."""
    where = "reshape_and_cache_q4"
    device = key_cache.get_device()
    nb, hkv, bs, d, page, head = _q4_dims(where, key_cache, value_cache, device)
    ts = _row_stride(where, key, value, slot_mapping, hkv, d, device)
    st, leave = _launch_on(device, stream)
    try:
        _native_call("nxt_reshape_and_cache_q4", key.data_ptr(), value.data_ptr(),
                     key_cache.data_ptr(), value_cache.data_ptr(), slot_mapping.data_ptr(),
                     key.shape[0], hkv, d, bs, k_scale, v_scale, page, head, ts, nb, st)
    finally:
        if leave is not None:
            leave.close()


def read_cache_q4(key_cache, value_cache, slot_mapping, k_scale, v_scale, *, key=None, value=None,
                  stream=None):
    """The rows that 4-bit pools hold at slot_mapping[t], as fp16 key and value
    [T, Hkv, D] (in `key` and `value`, of equal strides, when given); rows of
    negative slots, or slots past the pools, are zero."""
    import torch
    where = "read_cache_q4"
    device = key_cache.get_device()
    nb, hkv, bs, d, page, head = _q4_dims(where, key_cache, value_cache, device)
    T = slot_mapping.numel()
    st, leave = _launch_on(device, stream)
    try:
        if key is None:
            if value is None:
                value = key_cache.new_empty((T, hkv, d), dtype=torch.float16)
            key = torch.empty_strided(value.shape, value.stride(), dtype=torch.float16,
                                      device=value.device)
        elif value is None:
            value = torch.empty_strided(key.shape, key.stride(), dtype=torch.float16,
                                        device=key.device)
        ts = _row_stride(where, key, value, slot_mapping, hkv, d, device)
        if key.shape[0] != T:
            _refuse(where, "one row per slot")
        _native_call("nxt_read_cache_q4", key.data_ptr(), value.data_ptr(), key_cache.data_ptr(),
                     value_cache.data_ptr(), slot_mapping.data_ptr(), T, hkv, d, bs, k_scale,
                     v_scale, page, head, ts, nb, st)
    finally:
        if leave is not None:
            leave.close()
    return key, value


def _check_step(where, query, block_tables, seq_lens, out, device):
    """What every attention call needs besides its pools; (B, Hq, D)."""
    import torch
    shape = query.shape
    if len(shape) != 3 or not query.is_contiguous() or device < 0:
        _refuse(where, "query must be a contiguous CUDA tensor [B, Hq, D]")
    B = shape[0]
    if (block_tables.dtype != torch.int32 or block_tables.dim() != 2 or block_tables.shape[0] < B
            or not block_tables.is_contiguous() or block_tables.get_device() != device):
        _refuse(where, "block_tables must be contiguous int32 [B, max_blocks] on the query's device")
    if (seq_lens.dtype != torch.int32 or seq_lens.numel() < B or not seq_lens.is_contiguous()
            or seq_lens.get_device() != device):
        _refuse(where, "seq_lens must be contiguous int32 [B] on the query's device")
    if out is not None and (out.shape != shape or out.dtype != query.dtype
                            or not out.is_contiguous() or out.get_device() != device):
        _refuse(where, "out must be a contiguous tensor like query")
    return shape


def _check_q4_step(where, query, key_cache, value_cache, block_tables, seq_lens, out, device):
    import torch
    B, Hq, D = _check_step(where, query, block_tables, seq_lens, out, device)
    dims = _q4_dims(where, key_cache, value_cache, device)
    if query.dtype != torch.float16 or D != dims[3]:
        _refuse(where, "query must be fp16 with the pools' head size")
    return B, Hq, dims


def _workspace(where, t, device):
    if t is None:
        return None, 0
    if not t.is_contiguous() or t.get_device() != device:
        _refuse(where, "workspace must be contiguous, on the query's device")
    return t.data_ptr(), t.numel() * t.element_size()


def _status(where, t, device):
    import torch
    if t is None:
        return None
    if t.dtype != torch.int32 or t.numel() < 1 or t.get_device() != device:
        _refuse(where, "device_status must be an int32 tensor on the call's device")
    return t.data_ptr()


def paged_attention_q4(query, key_cache, value_cache, block_tables, seq_lens, k_scale, v_scale, *,
                       scale=None, out=None, num_blocks=None, workspace=None, device_status=None,
                       stream=None):
    """Decode attention over 4-bit pools (q4_pool_shape); query and output fp16
    [B, Hq, D], any number of query heads per KV head."""
    import torch
    where = "paged_attention_q4"
    device = query.get_device()
    B, Hq, (nb, hkv, bs, d, page, head) = _check_q4_step(
        where, query, key_cache, value_cache, block_tables, seq_lens, out, device)
    st, leave = _launch_on(device, stream)
    try:
        if out is None:
            out = torch.empty_like(query)
        _native_call("nxt_paged_attention_q4_ex", out.data_ptr(), query.data_ptr(),
                     key_cache.data_ptr(), value_cache.data_ptr(), block_tables.data_ptr(),
                     seq_lens.data_ptr(), B, Hq, d, hkv, d ** -0.5 if scale is None else scale,
                     block_tables.shape[1], bs, k_scale, v_scale, page, head,
                     _known_blocks(where, num_blocks, nb), *_workspace(where, workspace, device),
                     _status(where, device_status, device), st)
    finally:
        if leave is not None:
            leave.close()
    return out


def q4_workspace_size(num_seqs, num_heads, head_size, num_kv_heads, max_num_blocks_per_seq,
                      block_size=16) -> int:
    """Workspace bytes of a paged_attention_q4 call on the current device."""
    return int(_native.xpa().nxt_paged_attention_q4_workspace_size(
        num_seqs, num_heads, head_size, num_kv_heads, max_num_blocks_per_seq, block_size))


def paged_attention_q4_append(query, key_cache, value_cache, block_tables, seq_lens, new_key,
                              new_value, slot_mapping, k_scale, v_scale, *, scale=None, out=None,
                              num_blocks=None, device_status=None, stream=None):
    """One decode step on 4-bit pools: new_key/new_value (fp16 [B, Hkv, D]) are
    stored at slot_mapping[b] and included in the attention (seq_lens count
    them)."""
    import torch
    where = "paged_attention_q4_append"
    device = query.get_device()
    B, Hq, (nb, hkv, bs, d, page, head) = _check_q4_step(
        where, query, key_cache, value_cache, block_tables, seq_lens, out, device)
    _row_stride(where, new_key, new_value, slot_mapping, hkv, d, device)
    if new_key.shape[0] != B or not new_key.is_contiguous() or not new_value.is_contiguous():
        _refuse(where, "new rows must be contiguous [B, Hkv, D]")
    st, leave = _launch_on(device, stream)
    try:
        if out is None:
            out = torch.empty_like(query)
        _native_call("nxt_paged_attention_q4_append_ex", out.data_ptr(), query.data_ptr(),
                     key_cache.data_ptr(), value_cache.data_ptr(), block_tables.data_ptr(),
                     seq_lens.data_ptr(), new_key.data_ptr(), new_value.data_ptr(),
                     slot_mapping.data_ptr(), B, Hq, d, hkv, d ** -0.5 if scale is None else scale,
                     block_tables.shape[1], bs, k_scale, v_scale, page, head,
                     _known_blocks(where, num_blocks, nb), _status(where, device_status, device),
                     st)
    finally:
        if leave is not None:
            leave.close()
    return out


# ── page bounds and sparse attention ───────────────────────────────────────
def _check_bounds(where, bounds, nb, hkv, d, dtype, device):
    if (bounds.shape != (nb, hkv, 2, d) or bounds.dtype != dtype or not bounds.is_contiguous()
            or bounds.get_device() != device):
        _refuse(where, "bounds must be contiguous [num_blocks, Hkv, 2, D] beside the pools")


def _plain_dims(where, key_cache, value_cache, device):
    """(num_blocks, Hkv, block size, head size, page and head strides) of fp16 or fp32 pools."""
    shape = key_cache.shape
    if (len(shape) != 4 or value_cache.shape != shape or value_cache.dtype != key_cache.dtype
            or not key_cache.is_contiguous() or not value_cache.is_contiguous() or device < 0
            or key_cache.get_device() != device or value_cache.get_device() != device):
        _refuse(where, "pools must be contiguous [num_blocks, Hkv, block_size, D] on one CUDA "
                "device")
    nb, hkv, bs, d = shape
    return nb, hkv, bs, d, hkv * bs * d, bs * d


def page_bounds(key_cache, block_tables, seq_lens, bounds, *, num_new_tokens=0, k_scale=None,
                num_blocks=None, device_status=None, stream=None):
    """Writes into `bounds` [num_blocks, Hkv, 2, D] the lowest and highest key
    per channel of the pages that hold the last num_new_tokens tokens of each
    sequence (0: of all its pages), over their valid tokens. key_cache is an
    fp16 or fp32 pool [num_blocks, Hkv, P, D] (bounds of its type) or, with
    k_scale, a 4-bit pool (q4_pool_shape; bounds fp16). Returns `bounds`."""
    import torch
    where = "page_bounds"
    device = key_cache.get_device()
    if k_scale is None:
        kind = _dtype_size(key_cache)
        nb, hkv, bs, d, page, head = _plain_dims(where, key_cache, key_cache, device)
        dtype, name = key_cache.dtype, "nxt_page_bounds"
    else:
        kind = k_scale
        nb, hkv, bs, d, page, head = _q4_dims(where, key_cache, key_cache, device)
        dtype, name = torch.float16, "nxt_page_bounds_q4"
    _check_bounds(where, bounds, nb, hkv, d, dtype, device)
    B = seq_lens.numel()
    if (block_tables.dtype != torch.int32 or block_tables.dim() != 2 or block_tables.shape[0] < B
            or seq_lens.dtype != torch.int32 or seq_lens.dim() != 1
            or not block_tables.is_contiguous() or not seq_lens.is_contiguous()
            or block_tables.get_device() != device or seq_lens.get_device() != device):
        _refuse(where, "block_tables must be int32 [B, max_blocks] and seq_lens int32 [B], beside "
                "the pool")
    st, leave = _launch_on(device, stream)
    try:
        _native_call(name, bounds.data_ptr(), key_cache.data_ptr(), block_tables.data_ptr(),
                     seq_lens.data_ptr(), B, hkv, d, block_tables.shape[1], bs, kind, page, head,
                     _known_blocks(where, num_blocks, nb), num_new_tokens,
                     _status(where, device_status, device), st)
    finally:
        if leave is not None:
            leave.close()
    return bounds


def _check_sparse(where, query, key_cache, value_cache, bounds, block_tables, seq_lens, out,
                  device, q4):
    import torch
    if q4:
        B, Hq, dims = _check_q4_step(where, query, key_cache, value_cache, block_tables, seq_lens,
                                     out, device)
    else:
        B, Hq, D = _check_step(where, query, block_tables, seq_lens, out, device)
        dims = _plain_dims(where, key_cache, value_cache, device)
        if (query.dtype not in (torch.float16, torch.float32) or key_cache.dtype != query.dtype
                or D != dims[3]):
            _refuse(where, "query and pools must be fp16 or fp32, of one type and head size")
    _check_bounds(where, bounds, dims[0], dims[1], dims[3], query.dtype, device)
    return B, Hq, dims


def select_pages(query, key_cache, bounds, block_tables, seq_lens, max_pages, *, sink_pages=0,
                 recent_pages=1, scale=None, num_blocks=None, device_status=None, stream=None):
    """The pages that sparse attention keeps: (tables int32 [B * Hkv,
    max_pages], lens int32 [B * Hkv], pages int32 [B, Hkv, max_pages]).
    key_cache is an fp16 or fp32 pool, or a 4-bit one (q4_pool_shape). With
    key_cache.view(NB * Hkv, 1, ...), query.view(B * Hkv, G, D), tables and
    lens are the inputs of any attention call over the pool."""
    import torch
    device = query.get_device()
    q4 = key_cache.dtype == torch.uint8
    B, Hq, (nb, hkv, bs, d, page, head) = _check_sparse(
        "select_pages", query, key_cache, key_cache, bounds, block_tables, seq_lens, None, device,
        q4)
    st, leave = _launch_on(device, stream)
    try:
        new = lambda *s: torch.empty(s, dtype=torch.int32, device=query.device)
        tables, lens, pages = new(B * hkv, max_pages), new(B * hkv), new(B, hkv, max_pages)
        _native_call("nxt_select_pages", tables.data_ptr(), lens.data_ptr(), pages.data_ptr(),
                     query.data_ptr(), bounds.data_ptr(), block_tables.data_ptr(),
                     seq_lens.data_ptr(), B, Hq, d, hkv, d ** -0.5 if scale is None else scale,
                     block_tables.shape[1], bs, query.element_size(), page, head,
                     _known_blocks("select_pages", num_blocks, nb), max_pages, sink_pages,
                     recent_pages, None, 0, _status("select_pages", device_status, device), st)
    finally:
        if leave is not None:
            leave.close()
    return tables, lens, pages


def paged_attention_sparse(query, key_cache, value_cache, bounds, block_tables, seq_lens,
                           max_pages, *, sink_pages=0, recent_pages=1, k_scale=None, v_scale=None,
                           scale=None, out=None, selected=None, num_blocks=None, workspace=None,
                           device_status=None, stream=None):
    """Decode attention over at most max_pages pages per sequence and KV head:
    the first sink_pages, the last recent_pages and the best of the others by
    their bounds (page_bounds). Pools as for paged_attention, or 4-bit ones
    with k_scale and v_scale. ``selected`` (int32 [B, Hkv, max_pages]) receives
    the kept pages' indices within each sequence, -1 past the last."""
    import torch
    where = "paged_attention_sparse"
    device = query.get_device()
    q4 = k_scale is not None
    if q4 != (v_scale is not None):
        _refuse(where, "k_scale and v_scale go together")
    B, Hq, (nb, hkv, bs, d, page, head) = _check_sparse(
        where, query, key_cache, value_cache, bounds, block_tables, seq_lens, out, device, q4)
    if selected is not None and (
            selected.dtype != torch.int32 or not selected.is_contiguous()
            or selected.shape != (B, hkv, max_pages) or selected.get_device() != device):
        _refuse(where, "selected must be contiguous int32 [B, Hkv, max_pages] on the query's device")
    if q4:
        name, kind = "nxt_paged_attention_q4_sparse_ex", (k_scale, v_scale)
    else:
        name, kind = "nxt_paged_attention_sparse_ex", (query.element_size(),)
    st, leave = _launch_on(device, stream)
    try:
        if out is None:
            out = torch.empty_like(query)
        _native_call(name, out.data_ptr(), query.data_ptr(), key_cache.data_ptr(),
                     value_cache.data_ptr(), bounds.data_ptr(), block_tables.data_ptr(),
                     seq_lens.data_ptr(), _opt_ptr(selected), B, Hq, d, hkv,
                     d ** -0.5 if scale is None else scale, block_tables.shape[1], bs, *kind, page,
                     head, _known_blocks(where, num_blocks, nb), max_pages, sink_pages,
                     recent_pages, *_workspace(where, workspace, device),
                     _status(where, device_status, device), st)
    finally:
        if leave is not None:
            leave.close()
    return out


def sparse_workspace_size(num_seqs, num_heads, head_size, num_kv_heads, max_num_blocks_per_seq,
                          max_pages, block_size=16, dtype_size=2) -> int:
    """Workspace bytes of a paged_attention_sparse call on the current device."""
    return int(_native.xpa().nxt_paged_attention_sparse_workspace_size(
        num_seqs, num_heads, head_size, num_kv_heads, max_num_blocks_per_seq, block_size,
        dtype_size, max_pages))


# ── block-table builder ────────────────────────────────────────────────────
class BlockTables:
    """One decode step's kernel inputs on the device, built by
    nxt_build_block_tables: tables [B, max_blocks] int32, seq_lens [B],
    slots [B] int64 (the newest token's slot), prefix (PrefixGroups or None)."""

    def __init__(self, buffer, offsets, B, max_blocks, bounds):
        import torch
        self.buffer = buffer

        def view(key, n, dtype):
            o = offsets[key]
            es = torch.tensor([], dtype=dtype).element_size()
            return buffer[o:o + n * es].view(dtype)
        self.tables = view(_native.NXT_BT_TABLES, B * max_blocks, torch.int32).view(B, max_blocks)
        self.seq_lens = view(_native.NXT_BT_SEQ_LENS, B, torch.int32)
        self.slots = view(_native.NXT_BT_SLOTS, B, torch.int64)
        pp = view(_native.NXT_BT_PREFIX_PAGES, B, torch.int32)
        go = view(_native.NXT_BT_GROUP_OFFSETS, B + 1, torch.int32)
        mem = view(_native.NXT_BT_GROUP_MEMBERS, B, torch.int32)
        self.prefix = (PrefixGroups(None, B, prefix_pages=pp, offsets=go, members=mem,
                                    bounds=bounds) if bounds[0] > 0 else None)


def build_block_tables(page_lists, seq_lens, max_blocks, *, block_size=16, prefix_node=None,
                       prefix_pages=None, device=None, stream=None, staging=None):
    """page_lists: per sequence, its physical pages in token order; seq_lens:
    context tokens (newest included); prefix_node / prefix_pages: per
    sequence, the radix node of its shared prefix (-1: none) and the whole
    pages it covers. Returns BlockTables on `device`."""
    import numpy as np
    import torch
    B = len(page_lists)
    counts = np.array([len(p) for p in page_lists], dtype=np.int64)
    offs = np.zeros(B + 1, dtype=np.int32)
    np.cumsum(counts, out=offs[1:])
    ids = (np.concatenate([np.asarray(p, dtype=np.int32) for p in page_lists])
           if B and offs[-1] else np.zeros(1, dtype=np.int32))
    sl = np.ascontiguousarray(seq_lens, dtype=np.int32)
    node = None if prefix_node is None else np.ascontiguousarray(prefix_node, dtype=np.int32)
    ppg = None if prefix_pages is None else np.ascontiguousarray(prefix_pages, dtype=np.int32)
    lib = _native.xpa()
    offsets = (ctypes.c_size_t * _native.NXT_BT_NUM_ARRAYS)()
    total = lib.nxt_block_tables_layout(B, int(max_blocks), int(offs[-1]), offsets)
    buf = torch.empty(max(total, 16), dtype=torch.uint8, device=device)
    g = (ctypes.c_int * 3)()
    ptr = lambda a: None if a is None else a.ctypes.data
    st_ptr, st_bytes = (None, 0) if staging is None else (staging.data_ptr(),
                                                          staging.numel() * staging.element_size())
    rc = lib.nxt_build_block_tables(
        ptr(offs), ptr(ids), ptr(sl), ptr(node), ptr(ppg), B, int(max_blocks), int(block_size),
        _ptr(buf), total, st_ptr, st_bytes, ctypes.addressof(g),
        ctypes.addressof(g) + 4, ctypes.addressof(g) + 8, _stream_ptr(stream))
    if rc != _native.NXT_PA_OK:
        raise PagedAttentionError(rc, "nxt_build_block_tables")
    return BlockTables(buf, list(offsets), B, int(max_blocks), (g[0], g[1], g[2]))
