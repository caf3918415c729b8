"""The bookkeeping of a paged cache, and what the attention operators check before an address reaches the library: on the CPU, with
tensors that pass for CUDA ones and a library that only records its arguments."""
import contextlib
import ctypes
import os
import re

import pytest
import torch

import decode_matmul_b200 as dmm
from decode_matmul_b200 import _lib, attention


def make(**kw):
    args = dict(layers=2, kv_heads=3, head_dim=64, num_pages=7, page_size=16, max_seqs=3, device="cpu")
    args.update(kw)
    return dmm.PagedCache(**args)


def table_of(cache, seq):
    return cache.page_table[seq, :-(-cache.lengths[seq] // cache.page_size)].tolist()


def test_sequences_grow_by_pages():
    c = make()
    assert c.k(1).shape == (7, 3, 16, 64) and c.v(1).data_ptr() != c.k(1).data_ptr()
    cu = c.extend([17, 0, 16])
    assert cu.tolist() == [0, 17, 17, 33] and cu.dtype == torch.int32
    assert c.lengths == [17, 0, 16] and c.seq_lens.tolist() == [17, 0, 16] and c.free_pages == 4
    assert c.extend([1, 1, 1]) is None
    assert c.seq_lens.tolist() == [18, 1, 17] and c.free_pages == 2
    used = table_of(c, 0) + table_of(c, 1) + table_of(c, 2)
    assert len(used) == 5 and len(set(used)) == 5 and all(0 <= p < 7 for p in used)
    first = table_of(c, 0)
    c.extend([14, 0, 0])
    assert table_of(c, 0) == first and c.free_pages == 2  # the last page was not full


def test_too_much_changes_nothing():
    c = make(max_pages=4)
    c.extend([30, 5, 0])
    before = (list(c.lengths), c.free_pages, c.page_table.clone(), c.seq_lens.clone())
    for new, what in (([40, 0, 0], "longer"), ([0, 40, 33], "free"), ([1, 1], "numbers"), ([1, -1, 1], "numbers")):
        with pytest.raises(RuntimeError, match=what):
            c.extend(new)
        assert (c.lengths, c.free_pages) == before[:2] and torch.equal(c.page_table, before[2]) and torch.equal(c.seq_lens, before[3])


def test_released_pages_serve_others():
    c = make(num_pages=3, max_seqs=2)
    c.extend([33, 0])
    with pytest.raises(RuntimeError, match="free"):
        c.extend([0, 1])
    c.release(0)
    assert c.free_pages == 3 and c.seq_lens.tolist() == [0, 0]
    c.extend([0, 48])
    assert sorted(table_of(c, 1)) == [0, 1, 2]
    with pytest.raises(RuntimeError, match="no sequence"):
        c.release(2)


@pytest.mark.parametrize("kw", [dict(dtype=torch.float32), dict(head_dim=96), dict(page_size=8), dict(page_size=48), dict(num_pages=0), dict(max_pages=0)])
def test_caches_that_no_kernel_reads(kw):
    with pytest.raises(RuntimeError):
        make(**kw)


# ------------------------------------------------ what reaches the library ------------------------------------------------
FIELDS = ("k", "v", "page_table", "seq_lens", "num_pages", "page_stride", "head_stride", "row_stride", "table_stride", "type", "kv_heads",
          "head_dim", "page_size", "num_seqs", "max_pages")


class Dev(torch.Tensor):
    """A CPU tensor that says it lives on CUDA device ``index``."""
    index = 0

    def get_device(self):
        return self.index

    def new_empty(self, shape, **kw):
        return dev(shape, self.dtype, self.index)


def dev(shape, dtype, index=0):
    t = torch.zeros(shape, dtype=dtype).as_subclass(Dev)
    t.index = index
    return t


@pytest.fixture
def calls(monkeypatch):
    seen = []

    class Fake:
        def dmm_attention_workspace_bytes(self, *a):
            return 1001

        def _call(self, name, args):
            cache = next(a for a in args if isinstance(a, bytes))
            seen.append((name, args, dict(zip(FIELDS, _lib.paged_cache.unpack(cache)))))
            return 0

        def dmm_append_kv(self, *a):
            return self._call("append", a)

        def dmm_paged_attention(self, *a):
            return self._call("paged", a)

        def dmm_prompt_attention(self, *a):
            return self._call("prompt", a)

    fake = Fake()
    monkeypatch.setattr(attention._lib, "lib", lambda: fake)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 7)
    monkeypatch.setattr(torch, "empty_like", lambda t: dev(t.shape, t.dtype, t.index))
    return seen


def cache_of(seqs=2, dtype=torch.float16, index=0, **kw):
    shape = dict(pages=9, kv_heads=2, page=16, dim=64, width=5)
    shape.update(kw)
    k = dev((shape["pages"], shape["kv_heads"], shape["page"], shape["dim"]), dtype, index)
    v = dev(k.shape, dtype, index)
    return k, v, dev((seqs, shape["width"]), torch.int32, index), dev((seqs,), torch.int32, index)


def test_the_caches_description(calls):
    k, v, table, lens = cache_of()
    q = dev((2, 8, 64), torch.float16)
    out = dmm.paged_attention(q, k, v, table, lens)
    name, args, cache = calls.pop()
    assert name == "paged" and args[0] == q.data_ptr() and args[1] == 512 and args[2] == 8 and args[3] == 0.125 and args[4] == out.data_ptr()
    assert args[-1] == 7 and args[-3] == 1001  # the current stream; the workspace's size
    assert cache == dict(k=k.data_ptr(), v=v.data_ptr(), page_table=table.data_ptr(), seq_lens=lens.data_ptr(), num_pages=9, page_stride=2048,
                         head_stride=1024, row_stride=64, table_stride=5, type=_lib.T_F16, kv_heads=2, head_dim=64, page_size=16, num_seqs=2, max_pages=5)
    # rows of tokens first, and one row of a wider table
    k, v = (dev((9, 16, 2, 64), torch.bfloat16).permute(0, 2, 1, 3) for _ in range(2))
    for t in (k, v):
        t.index = 0
    wide = dev((4, 11), torch.int32)
    row = wide[2:3, :5]
    row.index = 0
    one = dev((1,), torch.int32)
    dmm.prompt_attention(dev((3, 2, 64), torch.bfloat16), k, v, row, one, dev((2,), torch.int32), 0.5, pdl=True)
    name, args, cache = calls.pop()
    assert name == "prompt" and args[2] == 3 and args[4] == 0.5 and args[-2] == _lib.FLAG_PDL
    assert (cache["page_stride"], cache["head_stride"], cache["row_stride"], cache["table_stride"], cache["type"]) == (2048, 64, 128, 5, _lib.T_BF16)


def test_append_passes_its_types(calls):
    k, v, table, lens = cache_of()
    for tin, kind in ((torch.float32, _lib.T_F32), (torch.float16, _lib.T_F16), (torch.bfloat16, _lib.T_BF16)):
        qkv = dev((2, 8 * 64), tin)
        q = dmm.append_kv(qkv, k, v, table, lens, dev((32,), torch.float64), interleaved=True)
        name, args, _ = calls.pop()
        assert name == "append" and args[1] == kind and args[2:5] == (512, 2, 4) and args[6] == 1 and q.shape == (2, 4, 64)
    dmm.append_kv(dev((6, 512), torch.float32), k, v, table, lens, cu_seqlens=dev((3,), torch.int32))
    assert calls.pop()[1][5] is None


REFUSED = [
    (dict(q=lambda: dev((2, 8, 64), torch.bfloat16)), "dtype"), (dict(q=lambda: dev((2, 8, 64), torch.float16, 1)), "device"),
    (dict(q=lambda: dev((2, 7, 64), torch.float16)), "multiple"), (dict(q=lambda: dev((3, 8, 64), torch.float16)), "one row"),
    (dict(q=lambda: dev((2, 8, 32), torch.float16)), "64"), (dict(lens=lambda: dev((3,), torch.int32)), "seq_lens"),
    (dict(lens=lambda: dev((2,), torch.int64)), "seq_lens"), (dict(table=lambda: dev((2, 5), torch.int64)), "page_table"),
    (dict(table=lambda: dev((2, 0), torch.int32)), "empty"), (dict(table=lambda: dev((2, 5), torch.int32, 1)), "device"),
    (dict(v=lambda: dev((8, 2, 16, 64), torch.float16)), "v_pages"), (dict(v=lambda: dev((9, 2, 16, 64), torch.bfloat16)), "v_pages"),
    (dict(k=lambda: torch.zeros((9, 2, 16, 64), dtype=torch.float16), v=lambda: torch.zeros((9, 2, 16, 64), dtype=torch.float16)), "CUDA"),
]


@pytest.mark.parametrize("change,match", REFUSED)
def test_refused_before_the_library(calls, change, match):
    k, v, table, lens = cache_of()
    args = dict(q=dev((2, 8, 64), torch.float16), k=k, v=v, table=table, lens=lens)
    args.update({name: make_() for name, make_ in change.items()})
    with pytest.raises(RuntimeError, match=match):
        dmm.paged_attention(*args.values())
    assert not calls


def test_c_entries_refuse_by_status():
    """Every check of the C entries returns before any CUDA call."""
    L = _lib.lib()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 255) & ~255

    def cache(**kw):
        args = dict(k=p, v=p, page_table=p, seq_lens=p, num_pages=4, page_stride=2048, head_stride=1024, row_stride=64, table_stride=3, type=_lib.T_F16,
                    kv_heads=2, head_dim=64, page_size=16, num_seqs=2, max_pages=3)
        args.update(kw)
        return _lib.paged_cache.pack(*(args[f] or 0 for f in FIELDS))

    def paged(c, q=p, q_ld=256, heads=4, out=p, out_ld=256, ws=p, ws_bytes=0, flags=0):
        return L.dmm_paged_attention(q, q_ld, heads, 1.0, out, out_ld, c, ws, ws_bytes, flags, None)

    null, shape, align, arg, small, unsupported = -1, -2, -3, -4, -5, -6
    assert paged(None) == null and paged(cache(k=None)) == null and paged(cache(seq_lens=None)) == null and paged(cache(), q=None) == null
    assert paged(cache(type=0)) == arg and paged(cache(), flags=1) == arg
    assert paged(cache(head_dim=96)) == unsupported and paged(cache(page_size=24)) == unsupported and paged(cache(page_size=8)) == unsupported
    assert paged(cache(k=p + 8)) == align and paged(cache(row_stride=68)) == align and paged(cache(), q=p + 2) == align and paged(cache(), q_ld=260) == align
    for bad in (dict(num_pages=0), dict(num_seqs=0), dict(max_pages=0), dict(table_stride=2), dict(page_stride=1024), dict(row_stride=0),
                dict(head_stride=64), dict(page_stride=-2048), dict(max_pages=1 << 27, table_stride=1 << 27)):
        assert paged(cache(**bad)) == shape, bad
    assert paged(cache(), heads=3) == shape and paged(cache(), heads=0) == shape and paged(cache(), heads=2 * 129) == shape
    assert paged(cache(), q_ld=248) == shape and paged(cache(), out_ld=128) == shape
    assert paged(cache()) == small and paged(cache(), ws=None) == small
    assert paged(cache(), ws=p + 16, ws_bytes=1 << 40) == align
    # overlapping heads are fine where there is one of them
    assert paged(cache(kv_heads=1, head_stride=0, page_stride=1024)) == small
    assert L.dmm_prompt_attention(p, 256, 5, 4, 1.0, p, 256, cache(), None, p, 0, 0, None) == null
    assert L.dmm_prompt_attention(p, 256, 0, 4, 1.0, p, 256, cache(), p, p, 0, 0, None) == shape
    assert L.dmm_append_kv(p, 3, 512, 2, 4, None, 0, p, 256, cache(), None, 0, None) == arg
    assert L.dmm_append_kv(p, 0, 512, 3, 4, None, 0, p, 256, cache(), None, 0, None) == shape  # one row per sequence
    assert L.dmm_append_kv(p, 0, 504, 2, 4, None, 0, p, 256, cache(), None, 0, None) == shape
    assert L.dmm_append_kv(None, 0, 512, 2, 4, None, 0, p, 256, cache(), None, 0, None) == null
    assert L.dmm_attention_workspace_bytes(2, 2, 4, 2, 64) > 0


def test_the_fields_are_those_of_the_header():
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "dmm.h")).read()
    body = re.search(r"typedef struct dmm_paged_cache \{(.*?)\} dmm_paged_cache;", header, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    fields = [(name.strip().lstrip("*"), "P" if "*" in decl + name else "q" if "int64" in decl else "i")
              for decl, names in re.findall(r"((?:const )?\w+)\s+([^;]+);", body) for name in names.split(",")]
    assert tuple(n for n, _ in fields) == FIELDS and "".join(t for _, t in fields) == "PPPPqqqqqiiiiii"
    assert _lib.paged_cache.size == 96


def test_rotary_frequencies():
    f = dmm.rotary_frequencies(128, 500.0)
    assert f.dtype == torch.float64 and f.shape == (64,) and float(f[0]) == 1.0
    assert torch.allclose(f, 500.0 ** (-torch.arange(64, dtype=torch.float64) / 64), rtol=1e-15)
    with pytest.raises(RuntimeError):
        dmm.rotary_frequencies(7)


def test_idle_sequences_sit_out_a_step():
    c = make()
    c.extend([15, 3, 16])
    c.release(1)
    assert c.extend([1, 0, 1], idle=True) is None
    assert c.lengths == [16, 0, 17] and c.seq_lens.tolist() == [16, 0, 17] and c.free_pages == 4
    used = table_of(c, 0) + table_of(c, 2)
    assert len(used) == len(set(used)) == 3
    before = (list(c.lengths), c.free_pages, c.page_table.clone(), c.seq_lens.clone())
    for new in ([0, 0, 1], [1, 2, 1], [2, 0, 1]):  # a sequence that has tokens would get one; more than one token
        with pytest.raises(RuntimeError, match="idle"):
            c.extend(new, idle=True)
        assert (c.lengths, c.free_pages) == before[:2] and torch.equal(c.page_table, before[2]) and torch.equal(c.seq_lens, before[3])
    assert c.extend([1, 1, 1], idle=True) is None and c.seq_lens.tolist() == [17, 1, 18]
    assert c.extend([1, 0, 1]).tolist() == [0, 1, 1, 2]  # without it rows are packed, as ever
    c = make()
    assert c.extend([0, 0, 0], idle=True) is None and c.free_pages == 7


@pytest.mark.parametrize("shape", [(9, 0, 16, 64), (0, 2, 16, 64)])
def test_an_empty_cache_is_refused(calls, shape):
    _, _, table, lens = cache_of()
    k, v = dev(shape, torch.float16), dev(shape, torch.float16)
    with pytest.raises(RuntimeError, match="empty"):
        dmm.paged_attention(dev((2, 8, 64), torch.float16), k, v, table, lens)
    with pytest.raises(RuntimeError, match="empty"):
        dmm.append_kv(dev((2, 512), torch.float32), k, v, table, lens)
    assert not calls
