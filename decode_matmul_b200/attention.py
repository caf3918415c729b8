"""Attention between the products: what appends to a paged key-value cache, and what reads it.

The qkv product leaves fp32 [tokens, (heads + 2 kv_heads) * head_dim]; :func:`append_kv` turns it into rotated queries and
new rows of the cache, :func:`paged_attention` (one new token per sequence) and :func:`prompt_attention` (packed prompts)
attend over the cache, and their 16-bit result is what the o product reads.  As in :mod:`ops`, PyTorch is used for device
memory and streams only, and nothing here synchronises the device.

The cache of a layer is ``k_pages`` and ``v_pages``, fp16 or bf16 [num_pages, kv_heads, page_size, head_dim] with any strides
that leave the last dimension contiguous, ``page_table`` int32 [sequences, max_pages] and ``seq_lens`` int32
[sequences], the lengths with the tokens of the present call.  All of it is device memory: a captured graph goes on
working as sequences grow.  What the tables say beyond the cache is not followed and shows in ``status()``.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .ops import _on_device_of, _req

_TYPE_16 = {torch.float16: _lib.T_F16, torch.bfloat16: _lib.T_BF16}
_TYPE_IN = {torch.float32: _lib.T_F32, **_TYPE_16}


def rotary_frequencies(head_dim: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """float64 [head_dim / 2]: radians per position of every pair, ``base ** (-2 i / head_dim)``."""
    _req(head_dim > 0 and head_dim % 2 == 0, "head_dim must be even")
    return base ** (torch.arange(head_dim // 2, dtype=torch.float64, device=device) * (-2.0 / head_dim))


def _check_cache(k, v, table, lens):
    """Checks a cache and returns (its description for the library, dtype, device index, kv_heads, head_dim, sequences)."""
    for t, name in ((k, "k_pages"), (v, "v_pages"), (table, "page_table"), (lens, "seq_lens")):
        if not isinstance(t, torch.Tensor):
            raise RuntimeError(f"{name} must be a tensor")
    dtype, index = k.dtype, k.get_device()
    _req(dtype in _TYPE_16, "k_pages must have dtype torch.float16 or torch.bfloat16")
    _req(k.dim() == 4, "k_pages must be [num_pages, kv_heads, page_size, head_dim]")
    pages, kv_heads, page_size, head_dim = k.shape
    stride = k.stride()
    _req(head_dim in (64, 128), "head_dim must be 64 or 128")
    _req(page_size >= 16 and page_size & (page_size - 1) == 0, "page_size must be a power of two, 16 or more")
    _req(v.dtype == dtype and v.shape == k.shape, "v_pages must have the dtype and shape of k_pages")
    _req(v.stride() == stride, "v_pages must have the strides of k_pages")
    _req(stride[3] == 1, "the last dimension of k_pages and v_pages must be contiguous")
    _req(table.dtype == torch.int32 and table.dim() == 2, "page_table must be int32 [sequences, max_pages]")
    seqs, max_pages = table.shape
    _req(seqs > 0 and max_pages > 0, "page_table must not be empty")
    _req(max_pages == 1 or table.stride(1) == 1, "the rows of page_table must be contiguous")
    _req(lens.dtype == torch.int32 and lens.dim() == 1 and lens.size(0) == seqs, "seq_lens must be int32 [sequences]")
    _req(seqs == 1 or lens.stride(0) == 1, "seq_lens must be contiguous")
    _req(index >= 0, "k_pages must be a CUDA tensor")
    for t, name in ((v, "v_pages"), (table, "page_table"), (lens, "seq_lens")):
        if t.get_device() != index:
            raise RuntimeError(f"{name} must be on the device of k_pages")
    cache = _lib.PagedCacheArg(k.data_ptr(), v.data_ptr(), table.data_ptr(), lens.data_ptr(), pages, stride[0], stride[1], stride[2],
                               table.stride(0) if seqs > 1 else max_pages, _TYPE_16[dtype], kv_heads, head_dim, page_size, seqs, max_pages)
    return cache, dtype, index, kv_heads, head_dim, seqs


def _check_cu(cu, index, seqs):
    _req(isinstance(cu, torch.Tensor) and cu.dtype == torch.int32 and cu.dim() == 1 and cu.size(0) == seqs + 1,
         "cu_seqlens must be int32 [sequences + 1]")
    _req(cu.get_device() == index, "cu_seqlens must be on the device of k_pages")
    _req(cu.is_contiguous(), "cu_seqlens must be contiguous")


def _check_rows(t, name, dtype, index, head_dim):
    """A [tokens, heads, head_dim] tensor whose rows of heads are contiguous; returns the elements from one row to the next."""
    _req(isinstance(t, torch.Tensor) and t.dim() == 3 and t.size(2) == head_dim, f"{name} must be [tokens, heads, {head_dim}]")
    _req(t.dtype == dtype, f"{name} must have dtype {dtype}")
    _req(t.get_device() == index, f"{name} must be on the device of k_pages")
    tokens, heads, _ = t.shape
    stride = t.stride()
    _req(stride[2] == 1 and (heads == 1 or stride[1] == head_dim), f"the heads of a row of {name} must be contiguous")
    return stride[0] if tokens > 1 else heads * head_dim


def append_kv(qkv, k_pages, v_pages, page_table, seq_lens, freqs=None, output=None, *, cu_seqlens=None, interleaved=False, pdl=False):
    """Rotated queries [tokens, heads, head_dim] of the cache's type, and new rows of the cache, from the result of a qkv
    product.

    ``qkv`` is fp32, fp16 or bf16 [tokens, (heads + 2 kv_heads) * head_dim]: query heads, key heads, value heads.  Rows
    ``cu_seqlens[b]`` to ``cu_seqlens[b + 1]`` (int32 [sequences + 1]) are the last tokens of sequence b, whose
    ``seq_lens[b]`` counts them; without ``cu_seqlens`` there is one token per sequence.  Queries and keys are rotated by
    their position times ``freqs`` (float64 [head_dim / 2], :func:`rotary_frequencies`; None: not rotated), the two
    halves of a head as pairs or, ``interleaved``, neighbours.  Rows behind the last sequence are skipped."""
    cache, dtype, index, kv_heads, head_dim, seqs = _check_cache(k_pages, v_pages, page_table, seq_lens)
    _req(isinstance(qkv, torch.Tensor) and qkv.dtype in _TYPE_IN, "qkv must have dtype torch.float32, torch.float16 or torch.bfloat16")
    _req(qkv.get_device() == index, "qkv must be on the device of k_pages")
    _req(qkv.dim() == 2 and (qkv.size(1) == 1 or qkv.stride(1) == 1), "qkv must be [tokens, width] with contiguous rows")
    tokens, width = qkv.shape
    heads = width // head_dim - 2 * kv_heads
    _req(heads >= 1 and (heads + 2 * kv_heads) * head_dim == width, "qkv must be (heads + 2 kv_heads) * head_dim wide")
    if cu_seqlens is None:
        _req(tokens == seqs, "without cu_seqlens qkv has one row per sequence")
    else:
        _check_cu(cu_seqlens, index, seqs)
    if freqs is not None:
        _req(isinstance(freqs, torch.Tensor) and freqs.dtype == torch.float64 and freqs.shape == (head_dim // 2,) and freqs.is_contiguous(),
             "freqs must be contiguous float64 [head_dim / 2]")
        _req(freqs.get_device() == index, "freqs must be on the device of k_pages")
    with _on_device_of(k_pages):
        if output is None:
            output = torch.empty((tokens, heads, head_dim), dtype=dtype, device=k_pages.device)
            out_ld = heads * head_dim
        else:
            out_ld = _check_rows(output, "output", dtype, index, head_dim)
            _req(output.size(0) == tokens and output.size(1) == heads, "output must be [tokens, heads, head_dim]")
        if tokens == 0:
            return output
        rc = _lib.lib().dmm_append_kv(qkv.data_ptr(), _TYPE_IN[qkv.dtype], qkv.stride(0) if tokens > 1 else width, tokens, heads,
                                      None if freqs is None else freqs.data_ptr(), 1 if interleaved else 0, output.data_ptr(), out_ld,
                                      ctypes.byref(cache), None if cu_seqlens is None else cu_seqlens.data_ptr(),
                                      _lib.FLAG_PDL if pdl else 0, torch._C._cuda_getCurrentRawStream(index))
    _lib.check(rc, "append_kv")
    return output


def attention_workspace_bytes(tokens: int, sequences: int, heads: int, kv_heads: int, head_dim: int) -> int:
    """Bytes of scratch a call of :func:`paged_attention` (tokens = sequences) or :func:`prompt_attention` needs on the
    current device (``dmm_attention_workspace_bytes``)."""
    return int(_lib.lib().dmm_attention_workspace_bytes(tokens, sequences, heads, kv_heads, head_dim))


def _attend(name, q, k_pages, v_pages, page_table, seq_lens, cu_seqlens, scale, output, workspace, pdl):
    cache, dtype, index, kv_heads, head_dim, seqs = _check_cache(k_pages, v_pages, page_table, seq_lens)
    q_ld = _check_rows(q, "q", dtype, index, head_dim)
    tokens, heads, _ = q.shape
    _req(heads > 0 and heads % kv_heads == 0, "the number of query heads must be a multiple of kv_heads")
    if cu_seqlens is None:
        _req(tokens == seqs, "q must have one row per sequence")
    else:
        _check_cu(cu_seqlens, index, seqs)
    L = _lib.lib()
    with _on_device_of(k_pages):
        if output is None:
            output = torch.empty((tokens, heads, head_dim), dtype=dtype, device=k_pages.device)
            out_ld = heads * head_dim
        else:
            out_ld = _check_rows(output, "output", dtype, index, head_dim)
            _req(output.shape == q.shape, "output must have the shape of q")
            _req(tokens == 0 or output.data_ptr() != q.data_ptr(), "output must not be q")
        if tokens == 0:
            return output
        need = L.dmm_attention_workspace_bytes(tokens, seqs, heads, kv_heads, head_dim)
        if workspace is None:
            # scratch of this call's own: from the caching allocator, which knows about streams and captured graphs
            if need:
                workspace = torch.empty((need,), dtype=torch.uint8, device=k_pages.device)
        else:
            _req(isinstance(workspace, torch.Tensor) and workspace.get_device() == index and workspace.is_contiguous(),
                 f"workspace must be a contiguous tensor on device {index}")
        ws, ws_bytes = (None, 0) if workspace is None else (workspace.data_ptr(), workspace.numel() * workspace.element_size())
        scale = head_dim ** -0.5 if scale is None else float(scale)
        flags, stream = _lib.FLAG_PDL if pdl else 0, torch._C._cuda_getCurrentRawStream(index)
        if cu_seqlens is None:
            rc = L.dmm_paged_attention(q.data_ptr(), q_ld, heads, scale, output.data_ptr(), out_ld, ctypes.byref(cache), ws, ws_bytes,
                                       flags, stream)
        else:
            rc = L.dmm_prompt_attention(q.data_ptr(), q_ld, tokens, heads, scale, output.data_ptr(), out_ld, ctypes.byref(cache),
                                        cu_seqlens.data_ptr(), ws, ws_bytes, flags, stream)
    _lib.check(rc, name)
    return output


def paged_attention(q, k_pages, v_pages, page_table, seq_lens, scale=None, output=None, *, workspace=None, pdl=False):
    """Attention of one new token per sequence: [sequences, heads, head_dim] of the cache's type.

    ``q`` is [sequences, heads, head_dim]; query head h reads key head h // (heads / kv_heads), over the ``seq_lens[b]``
    keys of its sequence.  ``scale`` defaults to head_dim ** -0.5.  A sequence of length 0 gets zeros.  ``workspace``: scratch
    of at least :func:`attention_workspace_bytes` bytes, not shared with calls that may overlap on the GPU; by default the
    call allocates its own."""
    return _attend("paged_attention", q, k_pages, v_pages, page_table, seq_lens, None, scale, output, workspace, pdl)


def prompt_attention(q, k_pages, v_pages, page_table, seq_lens, cu_seqlens, scale=None, output=None, *, workspace=None, pdl=False):
    """Causal attention of packed prompts, or of the next chunk of each: [tokens, heads, head_dim] of the cache's type.

    Rows ``cu_seqlens[b]`` to ``cu_seqlens[b + 1]`` of ``q`` are the last tokens of sequence b; row i of n sees the keys
    j <= seq_lens[b] - n + i, which :func:`append_kv` has put into the cache, its own among them.  A row that sees no key
    gets zeros; rows behind the last sequence are left as they are.  ``scale`` and ``workspace`` as in :func:`paged_attention`."""
    _req(cu_seqlens is not None, "cu_seqlens must be given")
    return _attend("prompt_attention", q, k_pages, v_pages, page_table, seq_lens, cu_seqlens, scale, output, workspace, pdl)
