"""The attention operators on the GPU against their definitions in 64 bits."""
import math

import pytest
import torch

import decode_matmul_b200 as dmm
from attention_reference import append, attention, check_attention, half_step

pytestmark = pytest.mark.gpu
FP16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
BAD_PAGE = 8


def make_cache(gen, total, Hkv, D, page, dtype, layout="heads", spare=2, width=0):
    """Pages of random keys and values in random order, a table and lengths for sequences of ``total`` tokens.  What no token
    of a sequence owns is NaN: the rest of last pages, pages of no sequence."""
    need = [-(-n // page) for n in total]
    count = sum(need) + spare
    order = torch.randperm(count, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(total), max(max(need), 1) + width), count - 1, dtype=torch.int32, device="cuda")
    shape = {"heads": (count, Hkv, page, D), "rows": (count, page, Hkv, D), "both": (count, 2, Hkv, page, D)}[layout]

    def view(t):
        return t if layout == "heads" else t.permute(0, 2, 1, 3)

    if layout == "both":
        whole = torch.full(shape, math.nan, dtype=dtype, device="cuda")
        k, v = whole[:, 0], whole[:, 1]
    else:
        k, v = (view(torch.full(shape, math.nan, dtype=dtype, device="cuda")) for _ in range(2))
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        pos = torch.arange(total[b], device="cuda")
        where = table[b].long()[pos // page]
        for t, shift in ((k, 1.0), (v, 0.25)):
            rows = torch.randn((total[b], Hkv, D), generator=gen, device="cuda") + shift * torch.randn((D,), generator=gen, device="cuda")
            t[where, :, pos % page] = rows.to(dtype)
        at += n
    return k, v, table, torch.tensor(total, dtype=torch.int32, device="cuda")


def cu_of(new):
    return torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------ append ------------------------------------------------
APPENDS = [
    # new, past, H, Hkv, D, page, type of qkv, of the cache, interleaved, layout
    ([1], [0], 64, 8, 128, 16, F32, FP16, False, "heads"),
    ([1], [4095], 64, 8, 128, 64, F32, FP16, False, "heads"),
    ([1] * 5, [0, 15, 16, 17, 300], 32, 32, 128, 16, F32, BF16, False, "rows"),
    ([1, 1, 1], [5, 0, 64], 3, 1, 64, 32, FP16, FP16, True, "both"),
    ([7, 0, 33, 1, 128], [0, 9, 1000, 63, 2], 8, 2, 128, 64, F32, FP16, True, "heads"),
    ([40, 513], [70000, 3], 14, 2, 64, 128, BF16, BF16, False, "rows"),
    ([300] * 2, [0, 17], 5, 5, 128, 256, F32, BF16, True, "both"),
    ([2500], [0], 64, 8, 128, 32, F32, FP16, False, "heads"),
]


@pytest.mark.parametrize("new,past,H,Hkv,D,page,tin,dtype,interleaved,layout", APPENDS)
def test_append(new, past, H, Hkv, D, page, tin, dtype, interleaved, layout):
    gen = generator(1)
    total = [n + p for n, p in zip(new, past)]
    k, v, table, lens = make_cache(gen, total, Hkv, D, page, dtype, layout)
    k0, v0 = k.clone(), v.clone()
    T = sum(new)
    extra = 3 if new != [1] * len(new) else 0  # rows behind the last sequence
    qkv = (2 * torch.randn((T + extra, (H + 2 * Hkv) * D), generator=gen, device="cuda")).to(tin)
    freqs = dmm.rotary_frequencies(D, device="cuda")
    out = torch.full((T + extra, H, D), 7.0, dtype=dtype, device="cuda")
    cu = None if new == [1] * len(new) else cu_of(new)
    got = dmm.append_kv(qkv, k, v, table, lens, freqs, out, cu_seqlens=cu, interleaved=interleaved)
    assert got is out and dmm.status() == 0
    y, off, pos, seq = append(qkv[:T], H, Hkv, D, lens, cu, freqs, interleaved)
    u = half_step(dtype)
    tiny = 2.0 ** -25 if dtype == FP16 else 0.0
    bound = u * y.abs() + 2 * off + tiny
    assert (((out[:T].double() - y[:, :H]).abs() - bound[:, :H]).max()) <= 0
    assert bool((out[T:] == 7.0).all())
    where, row = table[seq, pos // page].long(), pos % page
    assert ((k[where, :, row].double() - y[:, H:H + Hkv]).abs() - bound[:, H:H + Hkv]).max() <= 0
    assert torch.equal(v[where, :, row], qkv[:T].view(T, -1, D)[:, H + Hkv:].to(dtype))
    k0[where, :, row], v0[where, :, row] = k[where, :, row], v[where, :, row]
    for a, b in ((k, k0), (v, v0)):  # everything else as it was
        assert torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))


def test_append_without_rotation_copies():
    gen = generator(2)
    k, v, table, lens = make_cache(gen, [20, 3], 2, 64, 16, FP16)
    qkv = torch.randn((2, 8 * 64), generator=gen, device="cuda")
    q = dmm.append_kv(qkv, k, v, table, lens)
    rows = qkv.view(2, 8, 64).to(FP16)
    assert torch.equal(q, rows[:, :4])
    for b, n in enumerate((20, 3)):
        page, row = int(table[b, (n - 1) // 16]), (n - 1) % 16
        assert torch.equal(k[page, :, row], rows[b, 4:6]) and torch.equal(v[page, :, row], rows[b, 6:])


def test_append_strided_input_and_output():
    gen = generator(3)
    k, v, table, lens = make_cache(gen, [4, 9], 1, 64, 16, BF16)
    wide = torch.randn((5, 4 * 64 + 32), generator=gen, device="cuda")
    out = torch.zeros((5, 5, 64), dtype=BF16, device="cuda")
    cu = cu_of([2, 3])
    freqs = dmm.rotary_frequencies(64, 500.0, device="cuda")
    a = dmm.append_kv(wide[:, 16:16 + 256], k, v, table, lens, freqs, out[:, 1:3], cu_seqlens=cu)
    b = dmm.append_kv(wide[:, 16:16 + 256].contiguous(), k, v, table, lens, freqs, cu_seqlens=cu)
    assert torch.equal(a, b) and bool((out[:, 0] == 0).all()) and bool((out[:, 3:] == 0).all())


def test_append_far_positions_keep_their_angle():
    # position 10^6: a 32-bit angle would be off by 0.03; every page of the table is the same physical one
    gen = generator(4)
    pos, page = 1_000_003, 128
    table = torch.zeros((1, pos // page + 1), dtype=torch.int32, device="cuda")
    k = torch.zeros((1, 1, page, 128), dtype=FP16, device="cuda")
    v = torch.zeros_like(k)
    lens = torch.tensor([pos + 1], dtype=torch.int32, device="cuda")
    qkv = torch.randn((1, 3 * 128), generator=gen, device="cuda")
    freqs = dmm.rotary_frequencies(128, device="cuda")
    q = dmm.append_kv(qkv, k, v, table, lens, freqs)
    y, off, _, _ = append(qkv, 1, 1, 128, lens, None, freqs, False)
    assert ((q.double() - y[:, :1]).abs() <= half_step(FP16) * y[:, :1].abs() + 2 * off[:, :1] + 2.0 ** -25).all()


# ------------------------------------------------ decode ------------------------------------------------
DECODES = [
    # lengths, H, Hkv, D, page, type, layout
    ([1], 64, 8, 128, 16, FP16, "heads"),
    ([4096], 64, 8, 128, 64, FP16, "heads"),
    ([0, 1, 15, 16, 17, 127, 128, 129], 32, 32, 128, 16, FP16, "rows"),
    ([0], 8, 1, 128, 64, BF16, "heads"),
    ([33, 1000, 0, 257], 6, 2, 64, 32, BF16, "both"),
    ([5000, 3, 777], 14, 2, 128, 128, FP16, "rows"),
    ([2049, 31], 16, 1, 64, 256, FP16, "heads"),
    ([513, 64], 40, 2, 128, 16, BF16, "heads"),   # a group of 20
    ([700], 128, 1, 64, 16, FP16, "heads"),       # a group of 128
    ([70001], 8, 1, 128, 64, BF16, "heads"),
    ([100 + 37 * i for i in range(40)], 8, 4, 128, 16, FP16, "rows"),
    ([1 + i % 5 for i in range(300)], 4, 4, 64, 16, FP16, "heads"),
]


@pytest.mark.parametrize("lens,H,Hkv,D,page,dtype,layout", DECODES)
def test_paged_attention(lens, H, Hkv, D, page, dtype, layout):
    gen = generator(5)
    k, v, table, seq_lens = make_cache(gen, lens, Hkv, D, page, dtype, layout, width=3)
    q = torch.randn((len(lens), H, D), generator=gen, device="cuda").to(dtype)
    got = dmm.paged_attention(q, k, v, table, seq_lens)
    assert dmm.status() == 0
    want, bound = attention(q, k, v, table, seq_lens, None)
    assert check_attention(got, want, bound) == q.numel()
    assert torch.equal(got, dmm.paged_attention(q, k, v, table, seq_lens))  # the same bits again


# ------------------------------------------------ prompt ------------------------------------------------
PROMPTS = [
    # new, past, H, Hkv, D, page, type, layout
    ([1], [0], 64, 8, 128, 16, FP16, "heads"),
    ([128], [0], 8, 1, 128, 64, FP16, "heads"),
    ([257], [0], 4, 4, 128, 16, FP16, "rows"),
    ([1, 0, 31, 32, 33, 127, 129, 300], [0] * 8, 16, 2, 128, 16, FP16, "heads"),
    ([5, 130, 1], [1000, 127, 64], 8, 2, 128, 32, BF16, "both"),
    ([100, 17, 200], [0, 4000, 3], 14, 2, 64, 128, BF16, "rows"),
    ([64, 3], [5, 0], 3, 1, 64, 256, FP16, "heads"),
    ([77], [2000], 40, 2, 128, 16, FP16, "heads"),    # a group of 20
    ([9, 40], [0, 100], 128, 1, 64, 16, BF16, "heads"),  # a group of 128
    ([1000], [0], 32, 32, 128, 64, FP16, "heads"),
    ([1500], [0], 10, 2, 128, 16, BF16, "rows"),
    ([1 + (7 * i) % 50 for i in range(60)], [(13 * i) % 90 for i in range(60)], 8, 8, 64, 16, FP16, "heads"),
    # few rows over long contexts: an item of the kernel is shared by several CTAs, or a CTA has parts of several
    ([3], [20000], 8, 1, 128, 64, FP16, "heads"),
    ([40, 1, 300, 2], [9000, 12000, 130, 0], 8, 1, 128, 16, BF16, "rows"),
    ([200], [7777], 4, 4, 64, 128, FP16, "both"),
    ([50 + i for i in range(40)], [300 * i for i in range(40)], 4, 2, 128, 32, FP16, "heads"),
    # more items than CTAs, some of them long: what begins last is short
    ([1100, 5, 700, 64, 1, 333], [0] * 6, 20, 20, 128, 16, BF16, "heads"),
    ([2300], [0], 64, 8, 64, 64, FP16, "heads"),
]


@pytest.mark.parametrize("new,past,H,Hkv,D,page,dtype,layout", PROMPTS)
def test_prompt_attention(new, past, H, Hkv, D, page, dtype, layout):
    gen = generator(6)
    total = [n + p for n, p in zip(new, past)]
    k, v, table, lens = make_cache(gen, total, Hkv, D, page, dtype, layout)
    T = sum(new)
    q = torch.randn((T + 5, H, D), generator=gen, device="cuda").to(dtype)
    q[T:] = math.nan  # rows behind the last sequence
    out = torch.full_like(q, 7.0)
    got = dmm.prompt_attention(q, k, v, table, lens, cu_of(new), output=out)
    assert got is out and dmm.status() == 0
    want, bound = attention(q, k, v, table, lens, cu_of(new))
    assert check_attention(out, want, bound) == T * H * D
    assert bool((out[T:] == 7.0).all())
    again = dmm.prompt_attention(q, k, v, table, lens, cu_of(new))
    assert torch.equal(out[:T], again[:T])


def test_prompt_rows_that_see_nothing_are_zero():
    # more new tokens than keys: the first rows have no key at all; a sequence without any key
    gen = generator(7)
    k, v, table, lens = make_cache(gen, [10, 0, 200], 2, 128, 16, FP16)
    new = [150, 7, 300]
    q = torch.randn((sum(new), 8, 128), generator=gen, device="cuda").to(FP16)
    got = dmm.prompt_attention(q, k, v, table, lens, cu_of(new))
    want, bound = attention(q, k, v, table, lens, cu_of(new))
    assert check_attention(got, want, bound) == q.numel()
    assert bool((got[:140] == 0).all()) and bool((got[150:157] == 0).all()) and bool((got[157:257] == 0).all())


@pytest.mark.parametrize("value", [math.inf, math.nan, -math.inf])
@pytest.mark.parametrize("group", [1, 8])
def test_values_behind_a_row_do_not_reach_it(value, group):
    # a key and a value that is not finite at position 70: rows before it know nothing of it
    gen = generator(8)
    k, v, table, lens = make_cache(gen, [200], 2, 128, 16, FP16)
    q = torch.randn((200, 2 * group, 128), generator=gen, device="cuda").to(FP16)
    want, bound = attention(q, k, v, table, lens, cu_of([200]))
    k[int(table[0, 70 // 16]), :, 70 % 16] = value
    v[int(table[0, 70 // 16]), :, 70 % 16] = value
    got = dmm.prompt_attention(q, k, v, table, lens, cu_of([200]))
    assert check_attention(got[:70], want[:70], bound[:70]) == 70 * 2 * group * 128
    assert not bool(torch.isfinite(got[70:]).any()) or value == -math.inf


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_one_value_that_is_not_finite(value, dtype):
    """One element of one value: the rows that see it have it in one column, every other value is as without it.  Also where
    the context is long and several CTAs share an item."""
    for new, past, at in ((300, 0, 140), (40, 9000, 9020), (40, 9000, 100)):
        gen = generator(20)
        T = new + past
        k, v, table, lens = make_cache(gen, [T], 1, 128, 64, dtype)
        q = torch.randn((new, 8, 128), generator=gen, device="cuda").to(dtype)
        want, bound = attention(q, k, v, table, lens, cu_of([new]))
        v[int(table[0, at // 64]), 0, at % 64, 17] = value
        got = dmm.prompt_attention(q, k, v, table, lens, cu_of([new]))
        seen = torch.arange(past, T, device="cuda") >= at
        assert not bool(torch.isfinite(got[seen][:, :, 17]).any()) and bool(seen.any())
        got[seen, :, 17] = 0
        want[seen, :, 17] = 0
        assert check_attention(got, want, bound) == got.numel()


def test_keys_that_are_not_finite_stay_with_their_rows():
    # a key of -infinity against positive queries has weight 0: the rows that see it are those without it
    gen = generator(21)
    k, v, table, lens = make_cache(gen, [150, 40], 2, 64, 16, FP16)
    q = torch.rand((190, 4, 64), generator=gen, device="cuda").to(FP16) + 0.1
    k[int(table[0, 2]), :, 5] = -60000.0
    want, bound = attention(q, k, v, table, lens, cu_of([150, 40]))
    k[int(table[0, 2]), :, 5] = -math.inf
    got = dmm.prompt_attention(q, k, v, table, lens, cu_of([150, 40]))
    assert check_attention(got, want, bound) == got.numel()
    one = dmm.paged_attention(q[torch.tensor([149, 189], device="cuda")], k, v, table, lens)
    assert check_attention(one, want[[149, 189]], bound[[149, 189]]) == one.numel()


@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_large_scores(dtype):
    # scores of some hundreds: all but one weight vanish, and the running maximum rises far along the keys
    gen = generator(9)
    k, v, table, lens = make_cache(gen, [900, 333], 2, 128, 64, dtype)
    for b, n in enumerate((900, 333)):
        for pos in range(0, n, 50):
            k[int(table[b, pos // 64]), :, pos % 64] *= 1.0 + pos / 40
    q = (4 * torch.randn((1233, 4, 128), generator=gen, device="cuda")).to(dtype)
    got = dmm.prompt_attention(q, k, v, table, lens, cu_of([900, 333]))
    want, bound = attention(q, k, v, table, lens, cu_of([900, 333]))
    assert check_attention(got, want, bound) == q.numel()
    last = torch.tensor([899, 1232], device="cuda")
    one = dmm.paged_attention(q[last].contiguous(), k, v, table, lens)
    assert check_attention(one, want[last], bound[last]) == one.numel()


def test_scale_and_strided_rows():
    gen = generator(10)
    k, v, table, lens = make_cache(gen, [50, 90], 2, 64, 16, BF16)
    wide = torch.randn((140, 12, 64), generator=gen, device="cuda").to(BF16)
    out = torch.zeros((140, 9, 64), dtype=BF16, device="cuda")
    for scale in (0.0, 0.3, -0.125):
        dmm.prompt_attention(wide[:, 2:8], k, v, table, lens, cu_of([50, 90]), scale, out[:, 1:7])
        want, bound = attention(wide[:, 2:8], k, v, table, lens, cu_of([50, 90]), scale)
        assert check_attention(out[:, 1:7], want, bound) == 140 * 6 * 64
        assert bool((out[:, 0] == 0).all()) and bool((out[:, 7:] == 0).all())
        got = dmm.paged_attention(wide[49::90, 2:8], k, v, table, lens, scale, out[:2, 1:7])
        rows = torch.tensor([49, 139], device="cuda")
        assert check_attention(got, want[rows], bound[rows]) == got.numel()


def test_cache_beyond_32_bit_offsets():
    # 2^32 + elements in each of the two halves of one 8.6 GB tensor: the last page and the first are used
    page, Hkv, D = 256, 8, 128
    count = 2 ** 32 // (page * Hkv * D) // 2 + 2
    pages = torch.empty((count, 2, Hkv, page, D), dtype=FP16, device="cuda")
    k, v = pages[:, 0], pages[:, 1]
    assert pages.numel() > 2 ** 32
    gen = generator(11)
    table = torch.tensor([[count - 1, 0, count - 2]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([600], dtype=torch.int32, device="cuda")
    qkv = torch.randn((600, 32 * 128), generator=gen, device="cuda")
    q = dmm.append_kv(qkv, k, v, table, lens, cu_seqlens=cu_of([600]))
    assert torch.equal(v[count - 1, :, 5], qkv[5].view(32, 128)[24:].to(FP16))
    got = dmm.prompt_attention(q, k, v, table, lens, cu_of([600]))
    want, bound = attention(q, k, v, table, lens, cu_of([600]))
    assert check_attention(got, want, bound) == q.numel()
    one = dmm.paged_attention(q[599:], k, v, table, lens)
    assert check_attention(one, want[599:], bound[599:]) == one.numel()


def test_bad_tables_raise_a_status_and_touch_nothing():
    gen = generator(12)
    k, v, table, lens = make_cache(gen, [64, 40], 2, 64, 16, FP16)
    k0, v0 = k.clone(), v.clone()
    bad = table.clone()
    bad[0, 3], bad[1, 2] = -1, k.shape[0]
    qkv = torch.randn((2, 8 * 64), generator=gen, device="cuda")
    q = dmm.append_kv(qkv, k, v, bad, lens)
    assert dmm.status() == BAD_PAGE
    assert torch.equal(k.view(torch.int16), k0.view(torch.int16)) and torch.equal(v.view(torch.int16), v0.view(torch.int16))
    # a page that is not there reads as zeros: keys of score 0 and values of 0
    kz, vz = torch.cat((k, torch.zeros_like(k[:1]))), torch.cat((v, torch.zeros_like(v[:1])))
    bz = bad.clone()
    bz[0, 3], bz[1, 2] = k.shape[0], k.shape[0]
    got = dmm.paged_attention(q, k, v, bad, lens)
    assert dmm.status() == BAD_PAGE
    want, bound = attention(q, kz, vz, bz, lens, None)
    assert check_attention(got, want, bound) == got.numel()
    new = [64, 40]
    qp = torch.randn((104, 4, 64), generator=gen, device="cuda").to(FP16)
    got = dmm.prompt_attention(qp, k, v, bad, lens, cu_of(new))
    assert dmm.status() == BAD_PAGE
    want, bound = attention(qp, kz, vz, bz, lens, cu_of(new))
    assert check_attention(got, want, bound) == got.numel()


@pytest.mark.parametrize("lens_,cu_", [([64, 1000], [0, 64, 104]), ([64, -5], [0, 64, 104]), ([64, 40], [0, 64, 200]), ([64, 40], [0, 64, 30]),
                                       ([64, 40], [-3, 64, 104])])
def test_bad_lengths_raise_a_status(lens_, cu_):
    # lengths beyond the table, below zero; cu_seqlens that leave the rows or descend
    gen = generator(13)
    k, v, table, lens = make_cache(gen, [64, 40], 2, 64, 16, FP16)
    k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    lens.copy_(torch.tensor(lens_))
    cu = torch.tensor(cu_, dtype=torch.int32, device="cuda")
    qkv = torch.randn((104, 8 * 64), generator=gen, device="cuda")
    out = torch.full((104, 4, 64), 7.0, dtype=FP16, device="cuda")
    dmm.append_kv(qkv, k, v, table, lens, output=out, cu_seqlens=cu)
    assert dmm.status() == BAD_PAGE
    q = torch.randn((104, 4, 64), generator=gen, device="cuda").to(FP16)
    out.fill_(7.0)
    dmm.prompt_attention(q, k, v, table, lens, cu, output=out)
    assert dmm.status() == BAD_PAGE
    if cu_ == [0, 64, 104]:  # the other sequence is served all the same
        want, bound = attention(q[:64], k, v, table[:1], lens[:1], cu_of([64]))
        assert check_attention(out[:64], want, bound) == 64 * 4 * 64
    if lens_ != [64, 40]:
        dmm.paged_attention(q[:2], k, v, table, lens)
        assert dmm.status() == BAD_PAGE


# ------------------------------------------------ together ------------------------------------------------
@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_chunks_then_tokens_as_one_prompt(dtype):
    """A prompt appended whole, the same in chunks, and the same with its end token by token: one answer each row."""
    gen = generator(14)
    H, Hkv, D, page, T = 8, 2, 128, 16, 211
    qkv = torch.randn((T, (H + 2 * Hkv) * D), generator=gen, device="cuda")
    freqs = dmm.rotary_frequencies(D, device="cuda")

    def cache():
        return (torch.zeros((20, Hkv, page, D), dtype=dtype, device="cuda"), torch.zeros((20, Hkv, page, D), dtype=dtype, device="cuda"),
                torch.randperm(20, generator=gen, device="cuda").to(torch.int32)[None].contiguous())

    k, v, table = cache()
    lens = torch.tensor([T], dtype=torch.int32, device="cuda")
    q = dmm.append_kv(qkv, k, v, table, lens, freqs, cu_seqlens=cu_of([T]))
    whole = dmm.prompt_attention(q, k, v, table, lens, cu_of([T]))
    want, bound = attention(q, k, v, table, lens, cu_of([T]))
    check_attention(whole, want, bound)
    k2, v2, table2 = cache()
    at = 0
    for n in (100, 77, 29, 1, 1, 1, 1, 1):
        rows = qkv[at:at + n]
        at += n
        lens.fill_(at)
        if n == 1:
            one = dmm.append_kv(rows, k2, v2, table2, lens, freqs)
            got = dmm.paged_attention(one, k2, v2, table2, lens)
        else:
            one = dmm.append_kv(rows, k2, v2, table2, lens, freqs, cu_seqlens=cu_of([n]))
            got = dmm.prompt_attention(one, k2, v2, table2, lens, cu_of([n]))
        assert torch.equal(one, q[at - n:at])
        check_attention(got, want[at - n:at], bound[at - n:at])
    assert at == T and dmm.status() == 0


def test_captured_graph_follows_growing_sequences():
    gen = generator(15)
    H, Hkv, D, page = 16, 2, 128, 16
    past = [5, 250, 31]
    k, v, table, lens = make_cache(gen, [p + 40 for p in past], Hkv, D, page, FP16)
    k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    lens.copy_(torch.tensor(past))
    freqs = dmm.rotary_frequencies(D, device="cuda")
    qkv = torch.zeros((3, (H + 2 * Hkv) * D), device="cuda")

    def step():
        lens.add_(1)
        q = dmm.append_kv(qkv, k, v, table, lens, freqs, pdl=True)
        return q, dmm.paged_attention(q, k, v, table, lens, pdl=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    lens.copy_(torch.tensor(past))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, out = step()
    lens.copy_(torch.tensor(past))
    for i in range(20):
        qkv.copy_(torch.randn(qkv.shape, generator=gen, device="cuda"))
        graph.replay()
        assert lens.tolist() == [p + i + 1 for p in past]
        want, bound = attention(q, k, v, table, lens, None)
        assert check_attention(out, want, bound) == out.numel()
    assert dmm.status() == 0


def test_two_streams_at_once():
    gen = generator(16)
    cases = []
    for lens in ([3000, 17, 900], [40, 2500]):
        k, v, table, seq_lens = make_cache(gen, lens, 4, 128, 64, FP16)
        q = torch.randn((len(lens), 8, 128), generator=gen, device="cuda").to(FP16)
        qp = torch.randn((sum(lens), 8, 128), generator=gen, device="cuda").to(FP16)
        args = (k, v, table, seq_lens)
        cases.append((q, qp, args, cu_of(lens), dmm.paged_attention(q, *args), dmm.prompt_attention(qp, *args, cu_of(lens))))
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for s, (q, qp, args, cu, _, _) in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append((dmm.paged_attention(q, *args), dmm.prompt_attention(qp, *args, cu)))
        torch.cuda.synchronize()
        for (a, b), case in zip(got, cases):
            assert torch.equal(a, case[4]) and torch.equal(b, case[5])


def test_workspace_of_the_callers():
    gen = generator(17)
    k, v, table, lens = make_cache(gen, [3000, 5], 2, 128, 16, FP16)
    q = torch.randn((2, 8, 128), generator=gen, device="cuda").to(FP16)
    need = dmm.attention_workspace_bytes(2, 2, 8, 2, 128)
    want = dmm.paged_attention(q, k, v, table, lens)
    ws = torch.full((max(need, 1),), 255, dtype=torch.uint8, device="cuda")
    assert torch.equal(dmm.paged_attention(q, k, v, table, lens, workspace=ws), want)
    # of any content, and of either operator: what the last call left in it does not count
    qp = torch.randn((12, 8, 128), generator=gen, device="cuda").to(FP16)
    prompt = dmm.prompt_attention(qp, k, v, table, lens, cu_of([10, 2]))
    for _ in range(3):
        assert torch.equal(dmm.prompt_attention(qp, k, v, table, lens, cu_of([10, 2]), workspace=ws), prompt)
        assert torch.equal(dmm.paged_attention(q, k, v, table, lens, workspace=ws), want)
    if need:
        with pytest.raises(RuntimeError, match="workspace"):
            dmm.paged_attention(q, k, v, table, lens, workspace=ws[:need - 1])


def test_refusals():
    gen = generator(18)
    k, v, table, lens = make_cache(gen, [20, 30], 2, 64, 16, FP16)
    q = torch.zeros((2, 4, 64), dtype=FP16, device="cuda")
    qkv = torch.zeros((2, 8 * 64), device="cuda")
    cu = cu_of([1, 1])

    def no(match, f, *a, **kw):
        with pytest.raises(RuntimeError, match=match):
            f(*a, **kw)

    no("CUDA", dmm.paged_attention, q, k.cpu(), v.cpu(), table, lens)
    no("device", dmm.paged_attention, q, k, v, table.cpu(), lens)
    no("device", dmm.paged_attention, q.cpu(), k, v, table, lens)
    no("int32", dmm.paged_attention, q, k, v, table.long(), lens)
    no("int32", dmm.paged_attention, q, k, v, table, lens[:1])
    no("dtype", dmm.paged_attention, q.float(), k, v, table, lens)
    no("dtype", dmm.paged_attention, q, k.float(), v.float(), table, lens)
    no("v_pages", dmm.paged_attention, q, k, v[:-1], table, lens)
    no("strides", dmm.paged_attention, q, k, v.transpose(1, 2).contiguous().transpose(1, 2), table, lens)
    no("multiple of kv_heads", dmm.paged_attention, q[:, :3].contiguous(), k, v, table, lens)
    no("one row per sequence", dmm.paged_attention, q[:1], k, v, table, lens)
    no("not be q", dmm.paged_attention, q, k, v, table, lens, None, q)
    no("shape of q", dmm.paged_attention, q, k, v, table, lens, None, torch.zeros((2, 2, 64), dtype=FP16, device="cuda"))
    no("64", dmm.paged_attention, q[..., :32], k, v, table, lens)
    no("cu_seqlens", dmm.prompt_attention, q, k, v, table, lens, None)
    no("cu_seqlens", dmm.prompt_attention, q, k, v, table, lens, cu.long())
    no("cu_seqlens", dmm.prompt_attention, q, k, v, table, lens, cu[:2])
    no("one row per sequence", dmm.append_kv, qkv[:1], k, v, table, lens)
    no("wide", dmm.append_kv, qkv[:, :-32].contiguous(), k, v, table, lens)
    no("wide", dmm.append_kv, qkv[:, :256].contiguous(), k, v, table, lens)
    no("freqs", dmm.append_kv, qkv, k, v, table, lens, torch.zeros(32, device="cuda"))
    no("qkv", dmm.append_kv, qkv.double(), k, v, table, lens)
    # head sizes, page sizes and strides that no kernel is built for
    no("head_dim", dmm.paged_attention, torch.zeros((2, 4, 32), dtype=FP16, device="cuda"), k[..., :32], v[..., :32], table, lens)
    no("page_size", dmm.paged_attention, q, k[:, :, :8], v[:, :, :8], table, lens)
    big = torch.zeros((4, 2, 16, 68), dtype=FP16, device="cuda")
    no("aligned|multiple", dmm.paged_attention, q, big[..., :64], big[..., :64], table, lens)
    no("overlap|shape", dmm.append_kv, qkv, k[:1].expand(4, 2, 16, 64), v[:1].expand(4, 2, 16, 64), table, lens)
    odd = torch.zeros(2 * 4 * 64 + 1, dtype=FP16, device="cuda")[1:].view(2, 4, 64)
    no("aligned", dmm.paged_attention, odd, k, v, table, lens)


def test_no_tokens_is_no_work():
    gen = generator(19)
    k, v, table, lens = make_cache(gen, [20, 30], 2, 64, 16, FP16)
    q = torch.zeros((0, 4, 64), dtype=FP16, device="cuda")
    assert dmm.prompt_attention(q, k, v, table, lens, cu_of([0, 0])).shape == (0, 4, 64)
    assert dmm.append_kv(torch.zeros((0, 512), device="cuda"), k, v, table, lens, cu_seqlens=cu_of([0, 0])).shape == (0, 4, 64)


@pytest.mark.parametrize("new,past,H,Hkv,D,page,dtype", [
    (5, 3000, 8, 1, 128, 64, FP16),
    (1, 2000, 16, 1, 64, 16, BF16),
    (260, 15000, 1, 1, 64, 128, FP16),   # two pairs of tiles
    (16, 15000, 64, 1, 128, 16, BF16),
    (3, 700, 8, 1, 128, 32, FP16),       # short enough for one CTA
])
def test_prompt_with_fewer_key_tiles_than_ctas(new, past, H, Hkv, D, page, dtype):
    gen = generator(22)
    k, v, table, lens = make_cache(gen, [new + past], Hkv, D, page, dtype)
    q = torch.randn((new, H, D), generator=gen, device="cuda").to(dtype)
    want, bound = attention(q, k, v, table, lens, cu_of([new]))
    for _ in range(2):
        got = dmm.prompt_attention(q, k, v, table, lens, cu_of([new]))
        assert check_attention(got, want, bound) == got.numel()


def test_captured_prompts_of_other_lengths():
    """One captured call, replayed for lengths whose work is shared out in either way, beside another captured call on the same workspace."""
    gen = generator(23)
    H, Hkv, D, page = 8, 1, 128, 16
    k, v, table, lens = make_cache(gen, [9000, 700, 5000], Hkv, D, page, FP16)
    full = lens.clone()
    ws = torch.empty(dmm.attention_workspace_bytes(300, 3, H, Hkv, D), dtype=torch.uint8, device="cuda")
    q = torch.randn((300, H, D), generator=gen, device="cuda").to(FP16)
    cu = cu_of([100, 100, 100])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        dmm.prompt_attention(q, k, v, table, lens, cu, workspace=ws, pdl=True)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            first = dmm.prompt_attention(q, k, v, table, lens, cu, workspace=ws, pdl=True)
            out = dmm.prompt_attention(first, k, v, table, lens, cu, workspace=ws, pdl=True)
        graphs.append((graph, first, out))
    for at, new in (([9000, 700, 5000], [100, 100, 100]), ([100, 100, 100], [100, 100, 100]), ([300, 0, 17], [280, 0, 17]),
                    ([9000, 0, 0], [3, 0, 0]), ([200, 700, 5000], [1, 298, 1])):
        lens.copy_(torch.tensor(at))
        cu.copy_(cu_of(new))
        q.copy_(torch.randn(q.shape, generator=gen, device="cuda"))
        for graph, first, out in graphs:
            for t in (first, out):
                t.fill_(0)
            graph.replay()
            rows = sum(new)
            for x, y in ((q, first), (first, out)):
                want, bound = attention(x, k, v, table, lens, cu)
                assert check_attention(y, want, bound) == rows * H * D
    assert dmm.status() == 0
    lens.copy_(full)


@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_scale_of_zero_means_the_average(dtype):
    # also where a score would be infinite in the type of the queries
    gen = generator(24)
    k, v, table, lens = make_cache(gen, [300, 20], 2, 128, 16, dtype)
    big = 60000.0 if dtype == FP16 else 1e15
    q = (big * torch.randn((320, 4, 128), generator=gen, device="cuda").clamp(-1, 1)).to(dtype)
    want, bound = attention(q, k, v, table, lens, cu_of([300, 20]), 0.0)
    got = dmm.prompt_attention(q, k, v, table, lens, cu_of([300, 20]), 0.0)
    assert check_attention(got, want, bound) == got.numel()
    rows = torch.tensor([299, 319], device="cuda")
    one = dmm.paged_attention(q[rows], k, v, table, lens, 0.0)
    assert check_attention(one, want[rows], bound[rows]) == one.numel()


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_in_place(dtype, interleaved):
    gen = generator(25)
    new, past = [70, 1, 0, 9], [5, 0, 3, 500]
    total = [n + p for n, p in zip(new, past)]
    k, v, table, lens = make_cache(gen, total, 2, 64, 16, dtype)
    k2, v2 = k.clone(), v.clone()
    qkv = torch.randn((sum(new), 9 * 64), generator=gen, device="cuda").to(dtype)
    freqs, cu = dmm.rotary_frequencies(64, device="cuda"), cu_of(new)
    want = dmm.append_kv(qkv, k, v, table, lens, freqs, cu_seqlens=cu, interleaved=interleaved)
    same = qkv.clone()
    heads = same.view(-1, 9, 64)[:, :5]
    assert dmm.append_kv(same, k2, v2, table, lens, freqs, heads, cu_seqlens=cu, interleaved=interleaved) is heads
    assert torch.equal(heads, want) and torch.equal(same[:, 5 * 64:], qkv[:, 5 * 64:])
    assert torch.equal(torch.nan_to_num(k), torch.nan_to_num(k2)) and torch.equal(torch.nan_to_num(v), torch.nan_to_num(v2))


def test_outputs_in_the_way_of_inputs_are_refused():
    gen = generator(26)
    k, v, table, lens = make_cache(gen, [20, 30], 2, 64, 16, FP16)
    wide = torch.randn((2, 12, 64), generator=gen, device="cuda").to(FP16)
    q, cu = wide[:, :4], cu_of([1, 1])
    want = dmm.paged_attention(q.contiguous(), k, v, table, lens)
    for call in (lambda out: dmm.paged_attention(q, k, v, table, lens, None, out), lambda out: dmm.prompt_attention(q, k, v, table, lens, cu, None, out)):
        for at in (0, 1, 3):
            with pytest.raises(RuntimeError, match="share memory"):
                call(wide[:, at:at + 4])
        with pytest.raises(RuntimeError, match="share memory"):
            call(torch.as_strided(wide, (2, 4, 64), (13 * 64, 64, 1), 64))
    assert torch.equal(dmm.paged_attention(q, k, v, table, lens, None, wide[:, 4:8]), want)  # side by side in one buffer
    qkv = wide[:, :8].flatten(1)
    for at in (1, 4):
        with pytest.raises(RuntimeError, match="share no memory"):
            dmm.append_kv(qkv, k, v, table, lens, None, qkv.view(2, 8, 64)[:, at:at + 4])
    big = torch.zeros((2, 8 * 64), device="cuda")
    with pytest.raises(RuntimeError, match="share no memory"):
        dmm.append_kv(big, k, v, table, lens, None, big.view(FP16).view(2, 16, 64)[:, :4])


def test_scores_that_are_all_minus_infinity_give_zeros():
    # a weight of 0 for every key: as without keys.  Short and long, so that parts are joined as well
    gen = generator(27)
    k, v, table, lens = make_cache(gen, [40, 9000, 17], 1, 128, 64, BF16)
    for b, n in enumerate((40, 9000)):
        pos = torch.arange(n, device="cuda")
        k[table[b].long()[pos // 64], :, pos % 64] = -math.inf
    q = torch.rand((3, 4, 128), generator=gen, device="cuda").to(BF16) + 0.5
    want, bound = attention(q, k, v, table, lens, None)
    for got in (dmm.paged_attention(q, k, v, table, lens), dmm.prompt_attention(q, k, v, table, lens, cu_of([1, 1, 1]))):
        assert bool((got[:2] == 0).all())
        assert check_attention(got[2], want[2], bound[2]) == 4 * 128


@pytest.mark.parametrize("new,past,at", [(40, 9000, 8999), (40, 9000, 9000), (40, 9000, 9001), (40, 200, 200), (40, 200, 130), (9, 0, 0), (300, 100, 100)])
def test_a_value_at_the_edge_of_what_every_row_sees(new, past, at):
    # infinite in one column: the rows that see it have the infinity there (or NaN), each once, and nothing else changes
    gen = generator(28)
    k, v, table, lens = make_cache(gen, [new + past], 2, 64, 16, FP16)
    q = torch.randn((new, 8, 64), generator=gen, device="cuda").to(FP16)
    want, bound = attention(q, k, v, table, lens, cu_of([new]))
    v[int(table[0, at // 16]), 1, at % 16, 5] = math.inf
    got = dmm.prompt_attention(q, k, v, table, lens, cu_of([new]))
    seen = torch.arange(past, past + new, device="cuda") >= at
    assert not bool(torch.isfinite(got[seen][:, 4:, 5]).any()) and bool(seen.any())
    got[seen, 4:, 5] = 0
    want[seen, 4:, 5] = 0
    assert check_attention(got, want, bound) == got.numel()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("group", [1, 8, 16, 40])
@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_many_sequences_of_a_few_tokens(D, group, dtype):
    # a warp has a new sequence, key head and queries with every 16 keys, or with every second and third
    gen = generator(29)
    lens_ = [(7 * i) % 17 for i in range(150)] + [(11 * i) % 49 for i in range(150)] + [16, 32, 1, 0, 500, 3, 17]
    k, v, table, lens = make_cache(gen, lens_, 4, D, 16, dtype)
    q = torch.randn((len(lens_), 4 * group, D), generator=gen, device="cuda").to(dtype)
    want, bound = attention(q, k, v, table, lens, None)
    got = dmm.paged_attention(q, k, v, table, lens)
    assert check_attention(got, want, bound) == got.numel()
    assert torch.equal(got, dmm.paged_attention(q, k, v, table, lens)) and dmm.status() == 0
