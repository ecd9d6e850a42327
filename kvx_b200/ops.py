"""Torch-tensor front end of the C-ABI library.

The write operator keeps the name, argument order and checks of the operator the
reference's vLLM patch registers (``reshape_and_cache_flash_kvx``, reference:
patches/vllm/kvx.patch:176-275): it fills the ABI descriptors from tensor sizes and strides
without canonicalising them, passes torch's current CUDA stream and raises when the status
is not OK.  Torch is used for device memory and streams only; all data movement happens in
``libkvx_b200.so``.  Nothing here falls back to PyTorch indexing.

When ``lib/libkvx_b200_torch.so`` is built, calls on 4-D caches go through the operators it
registers with torch's dispatcher (``torch.ops.kvx_b200.*``), which do the same descriptor
filling in C++ and cost a few microseconds of host time per call; otherwise, and for 5-D
packed caches and the prefill entry point, the descriptors are filled here through ctypes.
"""
from __future__ import annotations

import ctypes as C
import math
import os
import re
from typing import Optional

import torch

from . import abi
from ._lib import lib

_FLOAT_CODES = {torch.float16: abi.DTYPE_F16, torch.bfloat16: abi.DTYPE_BF16,
                torch.float32: abi.DTYPE_F32}
_INDEX_CODES = {torch.int32: abi.DTYPE_S32, torch.int64: abi.DTYPE_S64}
_FP8_TORCH = (torch.float8_e4m3fn, torch.uint8)


class KvxError(RuntimeError):
    """A launcher returned a status other than ``KVX_STATUS_OK``."""

    def __init__(self, what: str, status: int):
        super().__init__(f"{what} failed with status={status} ({abi.STATUS_NAMES.get(status, '?')})")
        self.status = status


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


_NATIVE = None          # torch.ops.kvx_b200 once libkvx_b200_torch.so is loaded; False if it is not built
_NO_SCALE: dict = {}    # one empty float32 tensor per device, standing for "no scale"
_STATUS_RE = re.compile(r"(kvx [\w ]+?) failed with status=(\d+)")


def native_ops():
    """``torch.ops.kvx_b200`` (the dispatcher-registered operators of ``csrc/kvx_torch_ops.cpp``),
    or None when that library has not been built; the ctypes route below is then used."""
    global _NATIVE
    if _NATIVE is None:
        path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "libkvx_b200_torch.so")
        if os.path.exists(path):
            lib()  # libkvx_b200.so first, so that the operator library binds to the same copy
            torch.ops.load_library(path)
            _NATIVE = torch.ops.kvx_b200
        else:
            _NATIVE = False
    return _NATIVE or None


def _scale_arg(scale: Optional[torch.Tensor], device: torch.device) -> torch.Tensor:
    if scale is not None:
        return scale
    t = _NO_SCALE.get(device)
    if t is None:
        t = _NO_SCALE[device] = torch.empty(0, dtype=torch.float32, device=device)
    return t


def _no_scratch(device: torch.device) -> torch.Tensor:
    """An empty float32 tensor, standing for "no workspace given"."""
    return _scale_arg(None, device)


def _call_native(op, *args) -> None:
    _returning_native(op, *args)


def _returning_native(op, *args):
    try:
        return op(*args)
    except RuntimeError as exc:
        m = _STATUS_RE.search(str(exc))
        if m is None:
            raise
        raise KvxError(m.group(1), int(m.group(2))) from None


def _cache_code(t: torch.Tensor, kv_cache_dtype: str) -> int:
    if kv_cache_dtype in ("fp8", "fp8_e4m3"):
        if t.dtype not in _FP8_TORCH:
            raise TypeError("an fp8 cache must be a float8_e4m3fn or uint8 tensor")
        return abi.DTYPE_F8_E4M3
    if kv_cache_dtype != "auto":
        raise ValueError(f"unsupported kv_cache_dtype {kv_cache_dtype!r}")
    if t.dtype not in _FLOAT_CODES:
        raise TypeError(f"unsupported cache dtype {t.dtype}")
    return _FLOAT_CODES[t.dtype]


def cache_desc_from_tensors(key_cache: torch.Tensor, value_cache: torch.Tensor,
                            kv_cache_dtype: str = "auto", heads: Optional[int] = None,
                            layout: Optional[int] = None) -> abi.CacheDesc:
    """Describe a pair of 4-D (NHD / HND) or 5-D (HND_PACKED) page tensors.

    For 4-D tensors the layout is inferred unless given.  The reference's operator decides
    by one stride (NHD when stride(2) == head_dim, reference: patches/vllm/kvx.patch:132-135,
    :222-229), which misreads a contiguous ``[blocks, heads, block_size, dim]`` tensor; the
    rule here agrees with it wherever it is right and also accepts that tensor and vLLM's
    permuted view of HND memory: ``stride(1) < stride(2)`` is a ``[blocks, block_size, heads,
    dim]`` view of HND memory; otherwise the axis whose size equals ``heads`` names the
    layout; when ``block_size == heads`` (or ``heads`` is not given) the reference's stride
    rule decides.
    """
    if key_cache.shape != value_cache.shape:
        raise ValueError("key/value cache shape mismatch")
    code = _cache_code(key_cache, kv_cache_dtype)
    k_shape, k_stride = list(key_cache.shape), list(key_cache.stride())
    v_shape, v_stride = list(value_cache.shape), list(value_cache.stride())
    if key_cache.dim() == 5:
        layout = abi.LAYOUT_HND_PACKED
        nb, heads, dhi, bs, pack = key_cache.shape
        dim = dhi * pack
    else:
        dim = key_cache.shape[3]
        if layout is None and k_stride[1] < k_stride[2]:
            layout = abi.LAYOUT_HND  # a logical-NHD view of HND memory: describe the memory
            for shape, stride in ((k_shape, k_stride), (v_shape, v_stride)):
                shape[1], shape[2] = shape[2], shape[1]
                stride[1], stride[2] = stride[2], stride[1]
        elif layout is None:
            nhd, hnd = k_shape[2] == heads, k_shape[1] == heads
            if heads is not None and nhd != hnd:
                layout = abi.LAYOUT_NHD if nhd else abi.LAYOUT_HND
            else:
                layout = abi.LAYOUT_NHD if k_stride[2] == dim else abi.LAYOUT_HND
        if layout == abi.LAYOUT_NHD:
            nb, bs, heads, _ = k_shape
        else:
            nb, heads, bs, _ = k_shape
    c = abi.CacheDesc()
    c.size = C.sizeof(abi.CacheDesc)
    c.num_blocks, c.block_size, c.num_kv_heads, c.head_dim = nb, bs, heads, dim
    c.k = abi.tensor_desc(key_cache.data_ptr(), code, k_shape, k_stride, layout)
    c.v = abi.tensor_desc(value_cache.data_ptr(), code, v_shape, v_stride, layout)
    c.pool.size = C.sizeof(abi.PoolDesc)
    return c


def _scale_desc(scale: Optional[torch.Tensor], heads: int) -> abi.ScaleDesc:
    if scale is None:
        return abi.scale_desc(None, abi.SCALE_NONE, heads)
    if scale.dtype != torch.float32 or not scale.is_cuda:
        raise TypeError("scales must be float32 CUDA tensors")
    if scale.numel() == 1:
        return abi.scale_desc(scale.data_ptr(), abi.SCALE_PER_TENSOR, heads)
    if scale.dim() == 1 and scale.numel() == heads:
        return abi.scale_desc(scale.data_ptr(), abi.SCALE_PER_HEAD, heads, scale.stride(0))
    raise ValueError("a scale must have 1 or num_kv_heads elements")


def reshape_and_cache_flash_kvx(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor,
                                value_cache: torch.Tensor, slot_mapping: torch.Tensor,
                                kv_cache_dtype: str = "auto", k_scale: Optional[torch.Tensor] = None,
                                v_scale: Optional[torch.Tensor] = None,
                                tokens_per_seq: Optional[int] = None) -> None:
    """Scatter ``key`` / ``value`` ``[num_tokens, heads, dim]`` into the paged caches.

    ``slot_mapping[t] = block * block_size + offset``; negative slots are padding and are
    skipped.  ``kv_cache_dtype="auto"`` copies bits; ``"fp8"`` quantises to e4m3 with
    ``k_scale`` / ``v_scale`` (1 or ``heads`` float32 values).  ``tokens_per_seq`` selects
    the prefill entry point, whose result is identical.
    """
    native = native_ops() if tokens_per_seq is None and key_cache.dim() == 4 else None
    if native is not None:
        dev = key.device
        _call_native(native.reshape_and_cache_flash_kvx, key, value, key_cache, value_cache, slot_mapping,
                     kv_cache_dtype, _scale_arg(k_scale, dev), _scale_arg(v_scale, dev))
        return
    if not (key.is_cuda and value.is_cuda and key_cache.is_cuda and value_cache.is_cuda):
        raise ValueError("key/value and cache tensors must be CUDA tensors")
    if key.dtype != value.dtype or key.dtype not in _FLOAT_CODES:
        raise TypeError("key/value dtype mismatch or unsupported")
    if key.dim() != 3 or value.shape != key.shape:
        raise ValueError("key/value must be [num_tokens, num_heads, head_dim]")
    if slot_mapping.dtype not in _INDEX_CODES or slot_mapping.dim() != 1:
        raise TypeError("slot_mapping must be a 1-D int32 or int64 tensor")
    num_tokens = slot_mapping.shape[0]
    heads, dim = key.shape[1], key.shape[2]
    cache = cache_desc_from_tensors(key_cache, value_cache, kv_cache_dtype, heads)
    w = abi.WriteDesc()
    w.size = C.sizeof(abi.WriteDesc)
    w.io.size = C.sizeof(abi.KvIoDesc)
    w.io.num_tokens, w.io.num_kv_heads, w.io.head_dim = num_tokens, heads, dim
    code = _FLOAT_CODES[key.dtype]
    shape = (num_tokens, heads, dim)  # the patch sizes the batch by slot_mapping (kvx.patch:208)
    w.io.key = abi.tensor_desc(key.data_ptr(), code, shape, key.stride(), abi.LAYOUT_INVALID)
    w.io.value = abi.tensor_desc(value.data_ptr(), code, shape, value.stride(), abi.LAYOUT_INVALID)
    w.slots.size = C.sizeof(abi.SlotMapping)
    w.slots.dtype, w.slots.token_count = _INDEX_CODES[slot_mapping.dtype], num_tokens
    w.slots.invalid_slot = -1
    w.slots.slots = slot_mapping.data_ptr()
    w.k_scale_desc = _scale_desc(k_scale, heads)
    w.v_scale_desc = _scale_desc(v_scale, heads)
    if tokens_per_seq is None:
        status = lib().kvx_launch_write_kv(C.byref(cache), C.byref(w), _stream())
    else:
        status = lib().kvx_launch_write_kv_prefill(C.byref(cache), C.byref(w), int(tokens_per_seq), _stream())
    if status != abi.STATUS_OK:
        raise KvxError("kvx cache write", status)


def gather_kv(key_cache: torch.Tensor, value_cache: torch.Tensor, block_table: torch.Tensor,
              seq_lens: torch.Tensor, key_out: torch.Tensor, value_out: torch.Tensor,
              kv_cache_dtype: str = "auto", k_scale: Optional[torch.Tensor] = None,
              v_scale: Optional[torch.Tensor] = None) -> None:
    """Materialise ``out[s, tok] = cache[block_table[s, tok // bs], tok % bs]`` for
    ``tok < seq_lens[s]``; other positions of ``key_out`` / ``value_out`` stay untouched.

    ``block_table`` is ``[seq_count, max_blocks_per_seq]`` (int32 or int64, same dtype as
    ``seq_lens``); outputs are dense ``[seq_count, max_seq_len, heads, dim]``.
    """
    native = native_ops() if key_cache.dim() == 4 else None
    if native is not None:
        dev = key_out.device
        _call_native(native.gather_kv, key_cache, value_cache, block_table, seq_lens, key_out, value_out,
                     kv_cache_dtype, _scale_arg(k_scale, dev), _scale_arg(v_scale, dev))
        return
    if block_table.dim() != 2 or not block_table.is_contiguous():
        raise ValueError("block_table must be a contiguous [seq_count, max_blocks_per_seq] tensor")
    if block_table.dtype not in _INDEX_CODES or seq_lens.dtype != block_table.dtype:
        raise TypeError("block_table and seq_lens must share an int32 or int64 dtype")
    if key_out.dim() != 4 or key_out.shape != value_out.shape or key_out.dtype not in _FLOAT_CODES:
        raise ValueError("outputs must be [seq_count, max_seq_len, heads, dim] float tensors")
    seqs, max_len, heads, dim = key_out.shape
    cache = cache_desc_from_tensors(key_cache, value_cache, kv_cache_dtype, heads)
    g = abi.gather_desc(seqs, max_len, heads, dim, _FLOAT_CODES[key_out.dtype], key_out.data_ptr(),
                        value_out.data_ptr(), _INDEX_CODES[block_table.dtype], block_table.data_ptr(),
                        block_table.shape[1], seq_lens.data_ptr())
    for t, src in ((g.io.key, key_out), (g.io.value, value_out)):
        for i, s in enumerate(src.stride()):
            t.stride[i] = s
    g.block_table.seq_count = block_table.shape[0]
    g.seq_lens.seq_count = seq_lens.shape[0]
    if cache.k.dtype == abi.DTYPE_F8_E4M3:
        ks, vs = _scale_desc(k_scale, heads), _scale_desc(v_scale, heads)
        status = lib().kvx_launch_gather_kv_f8e4m3(C.byref(cache), C.byref(g), C.byref(ks), C.byref(vs), _stream())
    else:
        status = lib().kvx_launch_gather_kv(C.byref(cache), C.byref(g), _stream())
    if status != abi.STATUS_OK:
        raise KvxError("kvx cache gather", status)


def gather_kv_varlen(key_cache: torch.Tensor, value_cache: torch.Tensor, block_table: torch.Tensor,
                     seq_lens: torch.Tensor, out_indptr: torch.Tensor, key_out: torch.Tensor,
                     value_out: torch.Tensor, max_seq_len: int, kv_cache_dtype: str = "auto",
                     k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None) -> None:
    """The gather into un-padded ``[rows, heads, dim]`` outputs (the form variable-length
    attention kernels take, with ``out_indptr`` as their cumulative sequence lengths): token
    ``tok`` of sequence ``s`` goes to row ``out_indptr[s] + tok`` for ``tok < min(seq_lens[s],
    max_seq_len, out_indptr[s + 1] - out_indptr[s])``; other rows stay untouched."""
    if block_table.dim() != 2 or not block_table.is_contiguous():
        raise ValueError("block_table must be a contiguous [seq_count, max_blocks_per_seq] tensor")
    if block_table.dtype not in _INDEX_CODES or seq_lens.dtype != block_table.dtype:
        raise TypeError("block_table and seq_lens must share an int32 or int64 dtype")
    if out_indptr.dtype not in _INDEX_CODES or out_indptr.numel() != block_table.shape[0] + 1:
        raise ValueError("out_indptr must hold seq_count + 1 int32 or int64 row numbers")
    if key_out.dim() != 3 or key_out.shape != value_out.shape or key_out.dtype not in _FLOAT_CODES:
        raise ValueError("outputs must be [rows, heads, dim] float tensors")
    rows, heads, dim = key_out.shape
    seqs = block_table.shape[0]
    cache = cache_desc_from_tensors(key_cache, value_cache, kv_cache_dtype, heads)
    g = abi.gather_desc(seqs, max_seq_len, heads, dim, _FLOAT_CODES[key_out.dtype], key_out.data_ptr(),
                        value_out.data_ptr(), _INDEX_CODES[block_table.dtype], block_table.data_ptr(),
                        block_table.shape[1], seq_lens.data_ptr())
    code = _FLOAT_CODES[key_out.dtype]
    g.io.num_tokens = rows
    g.io.key = abi.tensor_desc(key_out.data_ptr(), code, key_out.shape, key_out.stride(), abi.LAYOUT_INVALID)
    g.io.value = abi.tensor_desc(value_out.data_ptr(), code, value_out.shape, value_out.stride(), abi.LAYOUT_INVALID)
    g.seq_lens.seq_count = seq_lens.shape[0]
    ks, vs = _scale_desc(k_scale, heads), _scale_desc(v_scale, heads)
    status = lib().kvx_launch_gather_kv_varlen(C.byref(cache), C.byref(g), out_indptr.data_ptr(),
                                               _INDEX_CODES[out_indptr.dtype], C.byref(ks), C.byref(vs), _stream())
    if status != abi.STATUS_OK:
        raise KvxError("kvx cache gather", status)


def paged_attention_decode(query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                           block_table: torch.Tensor, seq_lens: torch.Tensor, scale: float,
                           max_seq_len: Optional[int] = None, out: Optional[torch.Tensor] = None,
                           workspace: Optional[torch.Tensor] = None, kv_cache_dtype: str = "auto",
                           k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                           num_kv_heads: Optional[int] = None) -> torch.Tensor:
    """Decode attention that reads the paged cache in place (``include/kvx_attention.h``):
    ``query`` ``[seq_count, q_heads, dim]`` attends over each sequence's cached tokens, found
    through ``block_table`` / ``seq_lens`` as the gather finds them; returns ``out`` (same shape
    and dtype).  ``max_seq_len`` bounds the context (default: all the table can address).
    ``workspace`` is reusable uint8 scratch of :func:`attention_workspace_bytes` bytes; it is
    allocated per call when not given.  ``num_kv_heads`` names the cache's head axis when the
    layout cannot be read off the strides (a contiguous ``[blocks, heads, block_size, dim]``
    tensor)."""
    if query.dim() != 3 or query.dtype not in _FLOAT_CODES or not query.is_contiguous():
        raise ValueError("query must be a contiguous [seq_count, q_heads, dim] float tensor")
    if block_table.dim() != 2 or not block_table.is_contiguous():
        raise ValueError("block_table must be a contiguous [seq_count, max_blocks_per_seq] tensor")
    if block_table.dtype not in _INDEX_CODES or seq_lens.dtype != block_table.dtype:
        raise TypeError("block_table and seq_lens must share an int32 or int64 dtype")
    seqs, q_heads, dim = query.shape
    if out is None:
        out = torch.empty_like(query)
    cache = cache_desc_from_tensors(key_cache, value_cache, kv_cache_dtype, num_kv_heads)
    if max_seq_len is None:
        max_seq_len = block_table.shape[1] * cache.block_size
    need = lib().kvx_paged_attention_workspace_bytes(seqs, q_heads, cache.num_kv_heads, dim, max_seq_len)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=query.device)
    native = native_ops() if key_cache.dim() == 4 else None
    if native is not None:
        dev = query.device
        _call_native(native.paged_attention_decode, out, query, key_cache, value_cache, block_table, seq_lens,
                     float(scale), int(max_seq_len), int(cache.num_kv_heads), workspace, kv_cache_dtype,
                     _scale_arg(k_scale, dev), _scale_arg(v_scale, dev))
        return out
    a = abi.attention_desc(seqs, q_heads, dim, _FLOAT_CODES[query.dtype], query.data_ptr(), out.data_ptr(),
                           float(scale), int(max_seq_len), _INDEX_CODES[block_table.dtype], block_table.data_ptr(),
                           block_table.shape[1], seq_lens.data_ptr())
    a.seq_lens.seq_count = seq_lens.shape[0]
    ks, vs = _scale_desc(k_scale, cache.num_kv_heads), _scale_desc(v_scale, cache.num_kv_heads)
    status = lib().kvx_launch_paged_attention_decode(
        C.byref(cache), C.byref(a), C.byref(ks), C.byref(vs), workspace.data_ptr(),
        workspace.numel() * workspace.element_size(), _stream())
    if status != abi.STATUS_OK:
        raise KvxError("kvx paged attention", status)
    return out


def paged_attention_chunk(query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                          block_table: torch.Tensor, seq_lens: torch.Tensor, query_indptr: torch.Tensor,
                          scale: float, causal: bool = True, max_seq_len: Optional[int] = None,
                          out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
                          kv_cache_dtype: str = "auto", k_scale: Optional[torch.Tensor] = None,
                          v_scale: Optional[torch.Tensor] = None,
                          num_kv_heads: Optional[int] = None) -> torch.Tensor:
    """Attention of several new tokens per sequence over the paged cache
    (``include/kvx_attention.h``): row ``query_indptr[s] + i`` of ``query`` ``[rows, q_heads, dim]``
    is new token ``i`` of sequence ``s`` at position ``seq_lens[s] - n + i`` (``n`` new tokens, whose
    K and V are in the pages already) and attends to the cached tokens up to its own position, or
    to all of them when not ``causal``.  Returns ``out`` (same shape and dtype); rows of no sequence
    keep what ``out`` held.  Token rows of ``query`` and ``out`` may be slices of wider rows.
    ``workspace`` is reusable uint8 scratch of :func:`chunk_attention_workspace_bytes` bytes,
    allocated per call when not given; ``max_seq_len`` and ``num_kv_heads`` as in
    :func:`paged_attention_decode`."""
    if query.dim() != 3 or query.dtype not in _FLOAT_CODES:
        raise ValueError("query must be a [rows, q_heads, dim] float tensor")
    if block_table.dim() != 2 or not block_table.is_contiguous():
        raise ValueError("block_table must be a contiguous [seq_count, max_blocks_per_seq] tensor")
    if block_table.dtype not in _INDEX_CODES or seq_lens.dtype != block_table.dtype:
        raise TypeError("block_table and seq_lens must share an int32 or int64 dtype")
    seqs = block_table.shape[0]
    if seq_lens.dim() != 1 or seq_lens.numel() != seqs or not seq_lens.is_contiguous():
        raise ValueError("seq_lens must be contiguous with one entry per row of block_table")
    if query_indptr.dtype not in _INDEX_CODES or query_indptr.dim() != 1 or query_indptr.numel() != seqs + 1 \
            or not query_indptr.is_contiguous():
        raise ValueError("query_indptr must hold seq_count + 1 int32 or int64 row numbers")
    if max_seq_len is not None and max_seq_len < 1:
        raise ValueError("max_seq_len must be positive")
    rows, q_heads, dim = query.shape
    if out is None:
        out = torch.empty((rows, q_heads, dim), dtype=query.dtype, device=query.device)
    native = native_ops() if key_cache.dim() == 4 and query.is_cuda else None
    if native is not None:
        dev = query.device
        _call_native(native.paged_attention_chunk, out, query, key_cache, value_cache, block_table, seq_lens, query_indptr,
                     float(scale), bool(causal), 0 if max_seq_len is None else int(max_seq_len), int(num_kv_heads or 0),
                     _no_scratch(dev) if workspace is None else workspace, kv_cache_dtype, _scale_arg(k_scale, dev),
                     _scale_arg(v_scale, dev))
        return out
    if out.shape != query.shape or out.dtype != query.dtype:
        raise ValueError("out must have the shape and dtype of query")
    for name, t in (("key_cache", key_cache), ("value_cache", value_cache), ("block_table", block_table),
                    ("seq_lens", seq_lens), ("query_indptr", query_indptr), ("out", out)):
        if not t.is_cuda or t.device != query.device:
            raise ValueError(f"{name} must be on the query's CUDA device")
    cache = cache_desc_from_tensors(key_cache, value_cache, kv_cache_dtype, num_kv_heads)
    if cache.head_dim != dim:
        raise ValueError("query and cache differ in head_dim")
    if max_seq_len is None:
        max_seq_len = min(block_table.shape[1] * cache.block_size, 2 ** 31 - 2048)
    need = chunk_attention_workspace_bytes(seqs, rows, q_heads, cache.num_kv_heads, dim, max_seq_len)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=query.device)
    a = abi.chunk_attention_desc(seqs, rows, q_heads, dim, _FLOAT_CODES[query.dtype], query.data_ptr(), out.data_ptr(),
                                 float(scale), causal, int(max_seq_len), _INDEX_CODES[block_table.dtype],
                                 block_table.data_ptr(), block_table.shape[1], seq_lens.data_ptr(),
                                 _INDEX_CODES[query_indptr.dtype], query_indptr.data_ptr())
    for t, src in ((a.query, query), (a.out, out)):
        for i, s in enumerate(src.stride()):
            t.stride[i] = s
    ks, vs = _scale_desc(k_scale, cache.num_kv_heads), _scale_desc(v_scale, cache.num_kv_heads)
    with torch.cuda.device(query.device):
        status = lib().kvx_launch_paged_attention_chunk(
            C.byref(cache), C.byref(a), C.byref(ks), C.byref(vs), workspace.data_ptr(),
            workspace.numel() * workspace.element_size(), _stream())
    if status != abi.STATUS_OK:
        raise KvxError("kvx chunk attention", status)
    return out


def chunk_attention_workspace_bytes(seq_count: int, rows: int, q_heads: int, kv_heads: int, dim: int,
                                    max_seq_len: int) -> int:
    return lib().kvx_paged_attention_chunk_workspace_bytes(seq_count, rows, q_heads, kv_heads, dim, max_seq_len)


def attention_workspace_bytes(seq_count: int, q_heads: int, kv_heads: int, dim: int, max_seq_len: int) -> int:
    return lib().kvx_paged_attention_workspace_bytes(seq_count, q_heads, kv_heads, dim, max_seq_len)


def rotary_inv_freq(rotary_dim: int, base: float = 10000.0, scaling: str = "none", scale: float = 1.0,
                    original_length: int = 8192, low: float = 1.0, high: Optional[float] = None,
                    device: Optional[torch.device] = None) -> tuple[torch.Tensor, float]:
    """``(inv_freq, factor)`` for :func:`rotary_embedding`: float64 radians per position of the
    ``rotary_dim / 2`` pairs, and the factor on the turned values.

    ``scaling`` stretches a model trained on ``original_length`` positions by ``scale``:
    ``"none"``; ``"linear"``, every frequency divided by ``scale``; ``"ntk"``, a larger base, so that
    the slowest pair is divided by ``scale`` and the fastest kept; ``"bands"``, pairs that turn more
    than ``high`` times over the original length kept, fewer than ``low`` times divided, linear in
    the turns in between; ``"ramp"``, the same decision linear in the pair's index between the pairs
    that turn ``high`` and ``low`` times, with the factor ``0.1 ln(scale) + 1``.  ``high`` is 4 for
    ``"bands"`` and 32 for ``"ramp"`` unless given."""
    if rotary_dim <= 0 or rotary_dim % 2 != 0:
        raise ValueError("rotary_dim must be positive and even")
    if not scale > 0 or not base > 1:
        raise ValueError("scale must be positive and base above 1")
    pair = torch.arange(rotary_dim // 2, dtype=torch.float64)
    factor = 1.0
    if scaling == "ntk":
        if rotary_dim <= 2:
            raise ValueError("ntk scaling needs a rotary_dim above 2")
        base = base * scale ** (rotary_dim / (rotary_dim - 2))
    freq = base ** (-2.0 * pair / rotary_dim)
    if scaling == "linear":
        freq = freq / scale
    elif scaling in ("bands", "ramp"):
        if high is None:
            high = 4.0 if scaling == "bands" else 32.0
        if not high > low > 0:
            raise ValueError("high and low must be turns with high > low > 0")
        if scaling == "bands":
            keep = (original_length * freq / (2 * math.pi) - low) / (high - low)
        else:
            at = [rotary_dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (high, low)]
            first, last = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rotary_dim - 1)
            keep = 1.0 - (pair - first) / max(last - first, 1e-3)
            factor = 0.1 * math.log(scale) + 1.0 if scale > 1 else 1.0
        keep = keep.clamp(0.0, 1.0)
        freq = freq * keep + freq / scale * (1.0 - keep)
    elif scaling not in ("none", "ntk"):
        raise ValueError(f"unknown scaling {scaling!r}")
    return freq.to(device if device is not None else "cpu"), factor


def _rotary_desc(query: Optional[torch.Tensor], query_out: Optional[torch.Tensor], tokens: int, device: torch.device,
                 positions: torch.Tensor, inv_freq: torch.Tensor, interleaved: bool, factor: float,
                 inverse: bool) -> abi.RotaryDesc:
    if positions.dtype not in _INDEX_CODES or positions.dim() != 1 or positions.numel() != tokens or not positions.is_contiguous():
        raise ValueError("positions must hold one int32 or int64 per token")
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous float64 vector")
    if positions.device != device or inv_freq.device != device:
        raise ValueError("positions and inv_freq must be on the query's device")
    r = abi.RotaryDesc()
    r.size = C.sizeof(abi.RotaryDesc)
    r.rotary_dim = 2 * inv_freq.numel()
    r.flags = (abi.ROTARY_INTERLEAVED if interleaved else 0) | (abi.ROTARY_INVERSE if inverse else 0)
    r.position_dtype, r.positions = _INDEX_CODES[positions.dtype], positions.data_ptr()
    r.inv_freq, r.factor = inv_freq.data_ptr(), float(factor)
    if query is not None:
        code = _FLOAT_CODES[query.dtype]
        r.query = abi.tensor_desc(query.data_ptr(), code, query.shape, query.stride(), abi.LAYOUT_INVALID)
        r.query_out = abi.tensor_desc(query_out.data_ptr(), code, query_out.shape, query_out.stride(), abi.LAYOUT_INVALID)
    return r


def rotary_embedding(query: torch.Tensor, key: Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor,
                     interleaved: bool = False, factor: float = 1.0, inverse: bool = False,
                     query_out: Optional[torch.Tensor] = None,
                     key_out: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rotary positions (``include/kvx_rotary.h``): turns the first ``2 * len(inv_freq)`` dims of every
    head of ``query`` (and ``key``, unless None) ``[tokens, heads, dim]`` by ``positions * inv_freq`` and
    returns ``(query_out, key_out)``, new tensors unless given; ``query_out=query`` turns in place.
    Token rows may be slices of wider rows.  ``inverse`` turns back: called on the gradients of the
    outputs it gives those of the inputs.  ``inv_freq`` and ``factor`` as from
    :func:`rotary_inv_freq`."""
    if query.dim() != 3 or query.dtype not in _FLOAT_CODES or not query.is_cuda:
        raise ValueError("query must be a [tokens, heads, dim] float CUDA tensor")
    if key is not None and (key.dim() != 3 or key.dtype != query.dtype or key.device != query.device
                            or key.shape[0] != query.shape[0] or key.shape[2] != query.shape[2]):
        raise ValueError("key must match query in device, dtype, tokens and dim")
    if query_out is None:
        query_out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    if key is not None and key_out is None:
        key_out = torch.empty(key.shape, dtype=key.dtype, device=key.device)
    native = native_ops()
    if native is not None:
        none = _no_scratch(query.device)
        _call_native(native.rotary_embedding, query, none if key is None else key, positions, inv_freq, bool(interleaved),
                     float(factor), bool(inverse), query_out, none if key is None else key_out)
        return query_out, (None if key is None else key_out)
    for t, o in ((query, query_out), (key, key_out)):
        if t is not None and (o.shape != t.shape or o.dtype != t.dtype or o.device != t.device):
            raise ValueError("an output must match its input")
    r = _rotary_desc(query, query_out, query.shape[0], query.device, positions, inv_freq, interleaved, factor, inverse)
    if key is not None:
        code = _FLOAT_CODES[key.dtype]
        r.key = abi.tensor_desc(key.data_ptr(), code, key.shape, key.stride(), abi.LAYOUT_INVALID)
        r.key_out = abi.tensor_desc(key_out.data_ptr(), code, key_out.shape, key_out.stride(), abi.LAYOUT_INVALID)
    with torch.cuda.device(query.device):
        status = lib().kvx_launch_rotary(C.byref(r), _stream())
    if status != abi.STATUS_OK:
        raise KvxError("kvx rotary", status)
    return query_out, (None if key is None else key_out)


def rotary_and_cache(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, positions: torch.Tensor,
                     inv_freq: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                     slot_mapping: torch.Tensor, interleaved: bool = False, factor: float = 1.0,
                     query_out: Optional[torch.Tensor] = None, kv_cache_dtype: str = "auto",
                     k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`rotary_embedding` of ``query`` and ``key`` and :func:`reshape_and_cache_flash_kvx` of the
    turned keys and of ``value`` in one pass: the pages hold the same bits, ``key`` stays as it is.
    Returns ``query_out`` (new unless given; ``query`` itself turns in place).  Tokens with a negative
    slot, and those behind the last slot of a shorter ``slot_mapping`` (a batch padded to a fixed
    size), are turned but not cached."""
    if query_out is None:
        query_out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    native = native_ops() if key_cache.dim() == 4 and query.is_cuda else None
    if native is not None:
        dev = query.device
        _call_native(native.rotary_and_cache, query, key, value, positions, inv_freq, key_cache, value_cache, slot_mapping,
                     bool(interleaved), float(factor), query_out, kv_cache_dtype, _scale_arg(k_scale, dev),
                     _scale_arg(v_scale, dev))
        return query_out
    if key.dim() != 3 or key.dtype not in _FLOAT_CODES or value.shape != key.shape or value.dtype != key.dtype:
        raise ValueError("key/value must be matching [tokens, heads, dim] float tensors")
    if query.dim() != 3 or query.dtype != key.dtype or query.shape[0] != key.shape[0] or query.shape[2] != key.shape[2]:
        raise ValueError("query must match key in dtype, tokens and dim")
    if query_out.shape != query.shape or query_out.dtype != query.dtype:
        raise ValueError("query_out must match query")
    if slot_mapping.dtype not in _INDEX_CODES or slot_mapping.dim() != 1 or slot_mapping.numel() > key.shape[0] \
            or not slot_mapping.is_contiguous():
        raise ValueError("slot_mapping must be a contiguous int32 or int64 vector, one slot per token at most")
    for name, t in (("key", key), ("value", value), ("key_cache", key_cache), ("value_cache", value_cache),
                    ("slot_mapping", slot_mapping), ("query_out", query_out)):
        if not t.is_cuda or t.device != query.device:
            raise ValueError(f"{name} must be on the query's CUDA device")
    rows, heads, dim = key.shape
    tokens = slot_mapping.numel()
    cache = cache_desc_from_tensors(key_cache, value_cache, kv_cache_dtype, heads)
    w = abi.write_desc(tokens, heads, dim, _FLOAT_CODES[key.dtype], key.data_ptr(), value.data_ptr(),
                       _INDEX_CODES[slot_mapping.dtype], slot_mapping.data_ptr(), k_scale=_scale_desc(k_scale, heads),
                       v_scale=_scale_desc(v_scale, heads))
    for t, src in ((w.io.key, key), (w.io.value, value)):
        for i, s in enumerate(src.stride()):
            t.stride[i] = s
    some = query.numel() > 0
    r = _rotary_desc(query if some else None, query_out if some else None, rows, query.device, positions, inv_freq,
                     interleaved, factor, False)
    r.query.shape[0] = r.query_out.shape[0] = tokens
    with torch.cuda.device(query.device):
        status = lib().kvx_launch_rotary_write_kv(C.byref(cache), C.byref(w), C.byref(r), _stream())
    if status != abi.STATUS_OK:
        raise KvxError("kvx rotary write", status)
    if tokens < rows and some:
        rotary_embedding(query[tokens:], None, positions[tokens:], inv_freq, interleaved, factor, query_out=query_out[tokens:])
    return query_out


def _any_cache_desc(key_cache: torch.Tensor, value_cache: torch.Tensor) -> abi.CacheDesc:
    """Page tensors by their strides alone: whole pages are moved, whatever their axes mean."""
    if key_cache.shape != value_cache.shape or key_cache.dtype != value_cache.dtype:
        raise ValueError("key/value cache mismatch")
    kind = "fp8" if key_cache.dtype in _FP8_TORCH else "auto"
    return cache_desc_from_tensors(key_cache, value_cache, kind, layout=abi.LAYOUT_NHD)


def copy_pages(key_caches, value_caches, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copies page ``src[i]`` to page ``dst[i]`` in every key and value cache (lists, one entry per
    layer), any dtype and layout, one launch for many layers (``include/kvx_pages_ops.h``).  Pairs
    read the pages as they were before the call; pairs with a number outside the pool (``-1``
    marks an unused entry), with a destination that a later pair names again, or with a source that
    is a destination take no part."""
    key_caches, value_caches = list(key_caches), list(value_caches)
    if len(key_caches) != len(value_caches) or not key_caches:
        raise ValueError("one value cache per key cache")
    if src.dtype not in _INDEX_CODES or src.dim() != 1 or dst.shape != src.shape or dst.dtype != src.dtype or not src.is_cuda:
        raise ValueError("src and dst must be matching int32 or int64 CUDA vectors")
    native = native_ops()
    if native is not None:
        _call_native(native.copy_pages, key_caches, value_caches, src, dst)
        return
    if not src.is_contiguous() or not dst.is_contiguous():
        raise ValueError("src and dst must be contiguous")
    for t in [dst] + key_caches + value_caches:
        if t.device != src.device:
            raise ValueError("caches must be on the device of the page numbers")
    caches = (abi.CacheDesc * len(key_caches))(*[_any_cache_desc(k, v) for k, v in zip(key_caches, value_caches)])
    need = lib().kvx_copy_pages_workspace_bytes(src.numel())
    scratch = torch.empty(max(need, 16), dtype=torch.uint8, device=src.device)
    with torch.cuda.device(src.device):
        status = lib().kvx_launch_copy_pages(caches, len(key_caches), src.data_ptr(), dst.data_ptr(), _INDEX_CODES[src.dtype],
                                             src.numel(), scratch.data_ptr(), need, _stream())
    if status != abi.STATUS_OK:
        raise KvxError("kvx page copy", status)


def _table_args(block_table: torch.Tensor, seq_lens: Optional[torch.Tensor], page_refs: torch.Tensor, rows=()):
    if block_table.dim() != 2 or not block_table.is_contiguous() or block_table.dtype not in _INDEX_CODES \
            or not block_table.is_cuda:
        raise ValueError("block_table must be a contiguous [seq_count, max_blocks_per_seq] int32 or int64 CUDA tensor")
    dev, code = block_table.device, _INDEX_CODES[block_table.dtype]
    if page_refs.dtype != torch.int32 or page_refs.dim() != 1 or not page_refs.is_contiguous() or page_refs.device != dev:
        raise ValueError("page_refs must be a contiguous int32 vector on the table's device")
    if seq_lens is not None and (seq_lens.dtype != block_table.dtype or seq_lens.shape != (block_table.shape[0],)
                                 or not seq_lens.is_contiguous() or seq_lens.device != dev):
        raise ValueError("seq_lens must have the table's dtype and one entry per row")
    for r in rows:
        if r.dtype != block_table.dtype or r.dim() != 1 or not r.is_contiguous() or r.device != dev:
            raise ValueError("row numbers must be contiguous vectors of the table's dtype on its device")
    t = abi.block_table_desc(block_table.shape[0], block_table.shape[1], code, block_table.data_ptr())
    s = None if seq_lens is None else abi.seq_lens_desc(seq_lens.shape[0], code, seq_lens.data_ptr())
    return t, s


def free_sequences(block_table: torch.Tensor, seq_lens: torch.Tensor, page_refs: torch.Tensor, rows: torch.Tensor) -> None:
    """Frees the table rows ``rows``: their pages give a reference back (``page_refs``, int32 per page,
    0 = free), entries become -1 and lengths 0 (``include/kvx_pages_ops.h``)."""
    native = native_ops() if block_table.is_cuda else None
    if native is not None:
        _call_native(native.free_sequences, block_table, seq_lens, page_refs, rows)
        return
    t, s = _table_args(block_table, seq_lens, page_refs, (rows,))
    with torch.cuda.device(block_table.device):
        status = lib().kvx_launch_free_sequences(C.byref(t), C.byref(s), page_refs.data_ptr(), page_refs.numel(),
                                                 rows.data_ptr(), rows.numel(), _stream())
    if status != abi.STATUS_OK:
        raise KvxError("kvx sequence free", status)


def fork_sequences(block_table: torch.Tensor, seq_lens: torch.Tensor, page_refs: torch.Tensor, parents: torch.Tensor,
                   children: torch.Tensor, block_size: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Forks row ``parents[i]`` into row ``children[i]``: full pages are shared, a partly filled last
    page is duplicated into a free page (``include/kvx_pages_ops.h``).  Returns ``(src, dst)`` for
    :func:`copy_pages`: -1 where nothing is to be copied, -2 where the pair was not forked (a row
    outside the table or named twice, or no free page left; the child is then unchanged)."""
    native = native_ops() if block_table.is_cuda else None
    if native is not None:
        return _returning_native(native.fork_sequences, block_table, seq_lens, page_refs, parents, children, int(block_size))
    t, s = _table_args(block_table, seq_lens, page_refs, (parents, children))
    if parents.numel() != children.numel():
        raise ValueError("one child per parent")
    n = parents.numel()
    src, dst = torch.empty_like(parents), torch.empty_like(parents)
    need = lib().kvx_fork_workspace_bytes(n)
    scratch = torch.empty(max(need, 16), dtype=torch.uint8, device=block_table.device)
    with torch.cuda.device(block_table.device):
        status = lib().kvx_launch_fork_sequences(C.byref(t), C.byref(s), page_refs.data_ptr(), page_refs.numel(), int(block_size),
                                                 parents.data_ptr(), children.data_ptr(), n, src.data_ptr(), dst.data_ptr(),
                                                 scratch.data_ptr(), need, _stream())
    if status != abi.STATUS_OK:
        raise KvxError("kvx sequence fork", status)
    return src, dst


def compact_pages(block_table: torch.Tensor, page_refs: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Plans the move of all live pages to the front of the pool and renames them in ``block_table``
    and ``page_refs`` (``include/kvx_pages_ops.h``).  Returns ``(src, dst)``, ``num_blocks // 2`` entries
    with -1 behind the last move, for :func:`copy_pages`, to be run before the pages are read."""
    native = native_ops() if block_table.is_cuda else None
    if native is not None:
        return _returning_native(native.compact_pages, block_table, page_refs)
    t, _ = _table_args(block_table, None, page_refs)
    n = max(1, page_refs.numel() // 2)
    src, dst = (torch.empty(n, dtype=block_table.dtype, device=block_table.device) for _ in range(2))
    with torch.cuda.device(block_table.device):
        status = lib().kvx_launch_compact_pages(C.byref(t), page_refs.data_ptr(), page_refs.numel(), src.data_ptr(),
                                                dst.data_ptr(), _stream())
    if status != abi.STATUS_OK:
        raise KvxError("kvx page compaction", status)
    return src, dst


def scales_workspace(heads: int, device: torch.device) -> torch.Tensor:
    """Zeroed scratch for :func:`compute_kv_scales`; reusable across calls on one stream."""
    n = lib().kvx_kv_scales_workspace_bytes(heads)
    return torch.zeros(n, dtype=torch.uint8, device=device)


def compute_kv_scales(key: torch.Tensor, value: torch.Tensor, per_head: bool = True,
                      workspace: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``absmax / 448`` of K and of V per head (or per tensor), as float32 CUDA tensors."""
    if key.dim() != 3 or key.shape != value.shape or key.dtype != value.dtype:
        raise ValueError("key/value must be matching [num_tokens, heads, dim] tensors")
    tokens, heads, dim = key.shape
    n = heads if per_head else 1
    k_out = torch.empty(n, dtype=torch.float32, device=key.device)
    v_out = torch.empty(n, dtype=torch.float32, device=key.device)
    if workspace is None:
        workspace = scales_workspace(heads, key.device)
    io = abi.KvIoDesc()
    io.size = C.sizeof(abi.KvIoDesc)
    io.num_tokens, io.num_kv_heads, io.head_dim = tokens, heads, dim
    code = _FLOAT_CODES[key.dtype]
    io.key = abi.tensor_desc(key.data_ptr(), code, key.shape, key.stride(), abi.LAYOUT_INVALID)
    io.value = abi.tensor_desc(value.data_ptr(), code, value.shape, value.stride(), abi.LAYOUT_INVALID)
    status = lib().kvx_launch_kv_scales(C.byref(io), abi.SCALE_PER_HEAD if per_head else abi.SCALE_PER_TENSOR,
                                        k_out.data_ptr(), v_out.data_ptr(), workspace.data_ptr(),
                                        workspace.numel(), _stream())
    if status != abi.STATUS_OK:
        raise KvxError("kvx scale reduction", status)
    return k_out, v_out
