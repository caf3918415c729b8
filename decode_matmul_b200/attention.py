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

import torch

from . import _lib

_TYPE_16 = {torch.float16: _lib.T_F16, torch.bfloat16: _lib.T_BF16}
_pack = _lib.paged_cache.pack
_scratch = {}  # bytes of scratch by device and head size, on which alone they depend
_TYPE_IN = {torch.float32: _lib.T_F32, **_TYPE_16}


def rotary_frequencies(head_dim: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """float64 [head_dim / 2]: radians per position of every pair, ``base ** (-2 i / head_dim)``."""
    if head_dim <= 0 or head_dim % 2:
        _no("head_dim must be even")
    return base ** (torch.arange(head_dim // 2, dtype=torch.float64, device=device) * (-2.0 / head_dim))


def _no(msg: str):
    raise RuntimeError(msg)


# A call on few tokens takes a few microseconds on the GPU: the checks ask every tensor once and make no text before it is needed.
def _check_cache(k, v, table, lens):
    """Checks a cache and returns (its description for the library, dtype, device index, kv_heads, head_dim, sequences)."""
    if not (isinstance(k, torch.Tensor) and isinstance(v, torch.Tensor) and isinstance(table, torch.Tensor) and isinstance(lens, torch.Tensor)):
        _no("k_pages, v_pages, page_table and seq_lens must be tensors")
    dtype, index, shape, stride = k.dtype, k.get_device(), k.shape, k.stride()
    kind = _TYPE_16.get(dtype)
    if kind is None:
        _no("k_pages must have dtype torch.float16 or torch.bfloat16")
    if len(shape) != 4:
        _no("k_pages must be [num_pages, kv_heads, page_size, head_dim]")
    pages, kv_heads, page_size, head_dim = shape
    if not pages or not kv_heads:
        _no("k_pages must not be empty")
    if head_dim != 128 and head_dim != 64:
        _no("head_dim must be 64 or 128")
    if page_size < 16 or page_size & (page_size - 1):
        _no("page_size must be a power of two, 16 or more")
    if v.dtype is not dtype or v.shape != shape:
        _no("v_pages must have the dtype and shape of k_pages")
    if v.stride() != stride:
        _no("v_pages must have the strides of k_pages")
    if stride[3] != 1:
        _no("the last dimension of k_pages and v_pages must be contiguous")
    if table.dtype is not torch.int32 or table.dim() != 2:
        _no("page_table must be int32 [sequences, max_pages]")
    seqs, max_pages = table.shape
    if seqs == 0 or max_pages == 0:
        _no("page_table must not be empty")
    table_ld, table_step = table.stride()
    if table_step != 1 and max_pages > 1:
        _no("the rows of page_table must be contiguous")
    if lens.dtype is not torch.int32 or lens.shape != (seqs,):
        _no("seq_lens must be int32 [sequences]")
    if not lens.is_contiguous():
        _no("seq_lens must be contiguous")
    if index < 0:
        _no("k_pages must be a CUDA tensor")
    if v.get_device() != index or table.get_device() != index or lens.get_device() != index:
        _no("v_pages, page_table and seq_lens must be on the device of k_pages")
    cache = _pack(k.data_ptr(), v.data_ptr(), table.data_ptr(), lens.data_ptr(), pages, stride[0], stride[1], stride[2],
                  table_ld if seqs > 1 else max_pages, kind, kv_heads, head_dim, page_size, seqs, max_pages)
    return cache, dtype, index, kv_heads, head_dim, seqs


def _check_cu(cu, index, seqs):
    if not isinstance(cu, torch.Tensor) or cu.dtype is not torch.int32 or cu.shape != (seqs + 1,):
        _no("cu_seqlens must be int32 [sequences + 1]")
    if cu.get_device() != index:
        _no("cu_seqlens must be on the device of k_pages")
    if not cu.is_contiguous():
        _no("cu_seqlens must be contiguous")


def _check_rows(t, name, dtype, index, head_dim):
    """A [tokens, heads, head_dim] tensor whose rows of heads are contiguous; returns (tokens, heads, elements from one row to the next)."""
    if not isinstance(t, torch.Tensor) or t.dim() != 3 or t.size(2) != head_dim:
        _no(f"{name} must be [tokens, heads, {head_dim}]")
    if t.dtype is not dtype:
        _no(f"{name} must have dtype {dtype}")
    if t.get_device() != index:
        _no(f"{name} must be on the device of k_pages")
    tokens, heads, _ = t.shape
    ld, head, step = t.stride()
    if step != 1 or (head != head_dim and heads > 1):
        _no(f"the heads of a row of {name} must be contiguous")
    return tokens, heads, ld if tokens > 1 else heads * head_dim


def _overlap(a, a_ld, a_width, b, b_ld, b_width, rows):
    """Whether rows of a and b (widths and distances in bytes) share memory: rows of one buffer side by side do not."""
    a_at, b_at = a.data_ptr(), b.data_ptr()
    if a_at + (rows - 1) * a_ld + a_width <= b_at or b_at + (rows - 1) * b_ld + b_width <= a_at:
        return False
    if a_ld != b_ld or rows == 1:
        return True
    apart = (b_at - a_at) % a_ld
    return apart < a_width or apart + b_width > a_ld


def append_kv(qkv, k_pages, v_pages, page_table, seq_lens, freqs=None, output=None, *, cu_seqlens=None, interleaved=False, pdl=False):
    """Rotated queries [tokens, heads, head_dim] of the cache's type, and new rows of the cache, from the result of a qkv
    product.

    ``qkv`` is fp32, fp16 or bf16 [tokens, (heads + 2 kv_heads) * head_dim]: query heads, key heads, value heads.  Rows
    ``cu_seqlens[b]`` to ``cu_seqlens[b + 1]`` (int32 [sequences + 1]) are the last tokens of sequence b, whose
    ``seq_lens[b]`` counts them; without ``cu_seqlens`` there is one token per sequence, and the row of a sequence of length 0 is
    skipped.  Queries and keys are rotated by their position times ``freqs`` (float64 [head_dim / 2],
    :func:`rotary_frequencies`; None: not rotated), the two halves of a head as pairs or, ``interleaved``, neighbours.  Rows behind the last sequence are skipped.  No two tokens
    of a call may have the same place in the cache; ``output`` may be the query heads of a 16-bit ``qkv`` themselves."""
    cache, dtype, index, kv_heads, head_dim, seqs = _check_cache(k_pages, v_pages, page_table, seq_lens)
    kind = _TYPE_IN.get(qkv.dtype) if isinstance(qkv, torch.Tensor) else None
    if kind is None:
        _no("qkv must have dtype torch.float32, torch.float16 or torch.bfloat16")
    if qkv.get_device() != index:
        _no("qkv must be on the device of k_pages")
    if qkv.dim() != 2 or qkv.stride(1) != 1:
        _no("qkv must be [tokens, width] with contiguous rows")
    tokens, width = qkv.shape
    heads = width // head_dim - 2 * kv_heads
    if heads < 1 or (heads + 2 * kv_heads) * head_dim != width:
        _no("qkv must be (heads + 2 kv_heads) * head_dim wide")
    if cu_seqlens is not None:
        _check_cu(cu_seqlens, index, seqs)
    elif tokens != seqs:
        _no("without cu_seqlens qkv has one row per sequence")
    if freqs is not None:
        if not isinstance(freqs, torch.Tensor) or freqs.dtype is not torch.float64 or freqs.shape != (head_dim // 2,) or not freqs.is_contiguous():
            _no("freqs must be contiguous float64 [head_dim / 2]")
        if freqs.get_device() != index:
            _no("freqs must be on the device of k_pages")
    if output is None:
        output = k_pages.new_empty((tokens, heads, head_dim))
        out_ld = heads * head_dim
    else:
        rows, out_heads, out_ld = _check_rows(output, "output", dtype, index, head_dim)
        if rows != tokens or out_heads != heads:
            _no("output must be [tokens, heads, head_dim]")
        size = qkv.element_size()
        if tokens > 0 and _overlap(qkv, size * (qkv.stride(0) if tokens > 1 else width), size * width, output, 2 * out_ld, 2 * heads * head_dim, tokens) and (
                output.data_ptr() != qkv.data_ptr() or qkv.dtype is not dtype or (tokens > 1 and out_ld != qkv.stride(0))):
            _no("output must be the query heads of qkv or share no memory with it")
    if tokens == 0:
        return output
    args = (qkv.data_ptr(), kind, qkv.stride(0) if tokens > 1 else width, tokens, heads, None if freqs is None else freqs.data_ptr(),
            1 if interleaved else 0, output.data_ptr(), out_ld, cache, None if cu_seqlens is None else cu_seqlens.data_ptr(),
            _lib.FLAG_PDL if pdl else 0, torch._C._cuda_getCurrentRawStream(index))
    call = _lib.lib().dmm_append_kv
    if index == torch.cuda.current_device():
        rc = call(*args)
    else:
        with torch.cuda.device(index):
            rc = call(*args)
    if rc:
        _lib.check(rc, "append_kv")
    return output


def attention_workspace_bytes(tokens: int, sequences: int, heads: int, kv_heads: int, head_dim: int) -> int:
    """Bytes of scratch that calls of :func:`paged_attention` (tokens = sequences) or :func:`prompt_attention` need on the
    current device, for any lengths; at present ``head_dim`` alone decides (``dmm_attention_workspace_bytes``)."""
    return int(_lib.lib().dmm_attention_workspace_bytes(tokens, sequences, heads, kv_heads, head_dim))


def _attend(name, q, k_pages, v_pages, page_table, seq_lens, cu_seqlens, scale, output, workspace, pdl):
    cache, dtype, index, kv_heads, head_dim, seqs = _check_cache(k_pages, v_pages, page_table, seq_lens)
    tokens, heads, q_ld = _check_rows(q, "q", dtype, index, head_dim)
    if heads == 0 or heads % kv_heads:
        _no("the number of query heads must be a multiple of kv_heads")
    if cu_seqlens is not None:
        _check_cu(cu_seqlens, index, seqs)
    elif tokens != seqs:
        _no("q must have one row per sequence")
    if output is None:
        output = torch.empty_like(q) if q.is_contiguous() else q.new_empty((tokens, heads, head_dim))
        out_ld = heads * head_dim
    else:
        rows, out_heads, out_ld = _check_rows(output, "output", dtype, index, head_dim)
        if rows != tokens or out_heads != heads:
            _no("output must have the shape of q")
        if tokens > 0 and _overlap(q, 2 * q_ld, 2 * heads * head_dim, output, 2 * out_ld, 2 * heads * head_dim, tokens):
            _no("output must not be q or share memory with it")
    if tokens == 0:
        return output
    if scale is None:
        scale = head_dim ** -0.5
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            rc = _launch(q, q_ld, tokens, heads, scale, output, out_ld, cache, cu_seqlens, workspace, pdl, index, seqs, kv_heads, head_dim)
    else:
        rc = _launch(q, q_ld, tokens, heads, scale, output, out_ld, cache, cu_seqlens, workspace, pdl, index, seqs, kv_heads, head_dim)
    if rc:
        _lib.check(rc, name)
    return output


def _launch(q, q_ld, tokens, heads, scale, output, out_ld, cache, cu_seqlens, workspace, pdl, index, seqs, kv_heads, head_dim):
    """Scratch and the call into the library, on the current device."""
    L = _lib.lib()
    if workspace is None:
        # scratch of this call's own, of 16-bit values: the caching allocator knows about streams and captured graphs
        ws_bytes = _scratch.get((index, head_dim))
        if ws_bytes is None:
            ws_bytes = _scratch[index, head_dim] = L.dmm_attention_workspace_bytes(tokens, seqs, heads, kv_heads, head_dim)
        workspace = q.new_empty(((ws_bytes + 1) // 2,))
    elif not isinstance(workspace, torch.Tensor) or workspace.get_device() != index or not workspace.is_contiguous():
        _no(f"workspace must be a contiguous tensor on device {index}")
    else:
        ws_bytes = workspace.numel() * workspace.element_size()
    flags, stream = _lib.FLAG_PDL if pdl else 0, torch._C._cuda_getCurrentRawStream(index)
    if cu_seqlens is None:
        return L.dmm_paged_attention(q.data_ptr(), q_ld, heads, scale, output.data_ptr(), out_ld, cache, workspace.data_ptr(), ws_bytes, flags, stream)
    return L.dmm_prompt_attention(q.data_ptr(), q_ld, tokens, heads, scale, output.data_ptr(), out_ld, cache, cu_seqlens.data_ptr(),
                                  workspace.data_ptr(), ws_bytes, flags, stream)


def paged_attention(q, k_pages, v_pages, page_table, seq_lens, scale=None, output=None, *, workspace=None, pdl=False):
    """Attention of one new token per sequence: [sequences, heads, head_dim] of the cache's type.

    ``q`` is [sequences, heads, head_dim]; query head h reads key head h // (heads / kv_heads), over the ``seq_lens[b]``
    keys of its sequence.  ``scale`` defaults to head_dim ** -0.5.  A sequence of length 0 gets zeros.  Sequences may share pages.
    The weights of the softmax are rounded to the cache's type before they multiply the values; scores, maxima and sums are fp32.
    ``output`` shares no memory with q, the cache or the workspace.  ``workspace``: scratch of at least
    :func:`attention_workspace_bytes` bytes, not shared with calls that may overlap on the GPU; by default the call allocates
    its own."""
    return _attend("paged_attention", q, k_pages, v_pages, page_table, seq_lens, None, scale, output, workspace, pdl)


def prompt_attention(q, k_pages, v_pages, page_table, seq_lens, cu_seqlens, scale=None, output=None, *, workspace=None, pdl=False):
    """Causal attention of packed prompts, or of the next chunk of each: [tokens, heads, head_dim] of the cache's type.

    Rows ``cu_seqlens[b]`` to ``cu_seqlens[b + 1]`` of ``q`` are the last tokens of sequence b; row i of n sees the keys
    j <= seq_lens[b] - n + i, which :func:`append_kv` has put into the cache, its own among them.  A row that sees no key
    gets zeros; rows behind the last sequence are left as they are.  ``scale`` and ``workspace`` as in :func:`paged_attention`."""
    if cu_seqlens is None:
        _no("cu_seqlens must be given")
    return _attend("prompt_attention", q, k_pages, v_pages, page_table, seq_lens, cu_seqlens, scale, output, workspace, pdl)
