"""What the attention operators answer at the edges of what they are given: weights far below the largest, values that are not
finite inside a sequence, places of a batch that are idle."""
import math

import pytest
import torch

import decode_matmul_b200 as dmm
from attention_reference import attention, check_attention, gather
from decode_matmul_b200.linear import LinearStack
from test_gpu_attention import cu_of, generator, make_cache

pytestmark = pytest.mark.gpu
FP16, BF16 = torch.float16, torch.bfloat16


def tight(bound, v, table, lens, cu, group):
    """The bound with what subnormal weights may lose put where it belongs: fp16 weights are 2^7 times as large as the reference's
    bound takes them, the largest is 2^7 at least, and a weight that is rounded to a multiple of 2^-24 is off by 2^-25 at most, which
    is 2^-32 of the largest."""
    bound = bound.clone()
    for b, n in enumerate(lens.tolist()):
        vmax = gather(v, table[b], n).abs().amax(dim=(1, 2)).repeat_interleave(group)[None, :, None]
        rows = slice(b, b + 1) if cu is None else slice(int(cu[b]), int(cu[b + 1]))
        bound[rows] -= n * (2.0 ** -25 - 2.0 ** -32) * vmax
    return bound


@pytest.mark.parametrize("seqs,new,n,kv_heads,group,D", [
    (1, None, 300, 2, 4, 64), (1, None, 40000, 2, 4, 128),  # a sequence among many warps, each with a maximum of its own
    (40, None, 300, 32, 1, 128), (40, None, 1500, 32, 1, 64), (80, None, 700, 16, 12, 64),  # a warp has a sequence's key head alone
    (1, 3, 300, 2, 4, 64), (1, 3, 40000, 2, 4, 128), (1, 600, 2048, 8, 8, 64), (1, 600, 2048, 8, 8, 128), (5, 100, 1000, 16, 2, 128),
])
@pytest.mark.parametrize("above", [10.0, 14.0, 16.0])
def test_a_flat_tail_beside_a_heavy_key(seqs, new, n, kv_heads, group, D, above):
    """The first key has nearly all of the weight and a value of zero, so the result is what the others add: weights of e^-10 to
    e^-16 each, which fp16 holds with 10 to no bits when the largest is 1.  new: None for one token of each sequence."""
    gen = generator(1)
    k, v, table, lens = make_cache(gen, [n] * seqs, kv_heads, D, 64, FP16)
    pos = torch.arange(n, device="cuda")
    for b in range(seqs):
        page, row = table[b].long()[pos // 64], pos % 64
        k[page, :, row] = (0.5 * torch.randn((n, kv_heads, D), generator=gen, device="cuda")).to(FP16)
        k[page, :, row, 0] = 0.0
        v[page, :, row] = (1.0 + 0.5 * torch.randn((n, kv_heads, D), generator=gen, device="cuda")).to(FP16)
        k[page[0], :, 0], v[page[0], :, 0] = 0.0, 0.0
        k[page[0], :, 0, 0] = above
    q = (0.05 * torch.randn((seqs * (new or 1), kv_heads * group, D), generator=gen, device="cuda")).to(FP16)
    q[..., 0] = 1.0
    if new is None:
        got, cu = dmm.paged_attention(q, k, v, table, lens, 1.0), None
    else:
        cu = cu_of([new] * seqs)
        got = dmm.prompt_attention(q, k, v, table, lens, cu, 1.0)
    want, bound = attention(q, k, v, table, lens, cu, 1.0)
    assert check_attention(got, want, tight(bound, v, table, lens, cu, group)) == got.numel()


@pytest.mark.parametrize("dtype", [FP16, BF16])
def test_scores_of_millions(dtype):
    # where a product of a score and the scale is rounded to whole numbers the weights may be any power of 2, but never infinite
    gen = generator(2)
    k, v, table, lens = make_cache(gen, [700], 1, 128, 64, dtype)
    pos = torch.arange(700, device="cuda")
    k[table[0].long()[pos // 64], :, pos % 64] = 512.0
    q = torch.full((3, 4, 128), 258.0, dtype=dtype, device="cuda")
    for i in range(40):  # 258 * 512 * 128 times scales of 0.05 to 12
        scale = 0.05 * 1.15 ** i
        want, bound = attention(q, k, v, table, lens, cu_of([3]), scale)
        for got, rows in ((dmm.prompt_attention(q, k, v, table, lens, cu_of([3]), scale), slice(0, 3)), (dmm.paged_attention(q[2:], k, v, table, lens, scale), slice(2, 3))):
            assert check_attention(got, want[rows], bound[rows]) == got.numel() and bool(torch.isfinite(got).all())


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("group", [1, 8, 12])
def test_one_value_of_one_sequence_of_a_batch(what, dtype, group):
    """Sequences that a warp has whole, that a CTA's warps join, and that CTAs join: one element of one value shows in its column of
    the heads that read it, and nowhere else."""
    gen = generator(3)
    lens_ = [17, 3, 400, 1, 30000, 250, 0, 16]
    k, v, table, lens = make_cache(gen, lens_, 2, 128, 16, dtype)
    q = torch.randn((len(lens_), 2 * group, 128), generator=gen, device="cuda").to(dtype)
    want, bound = attention(q, k, v, table, lens, None)
    for seq, pos in ((0, 0), (0, 16), (2, 399), (4, 0), (4, 15003), (4, 29999), (7, 15)):
        at = (int(table[seq, pos // 16]), 1, pos % 16, 77)
        kept = v[at].clone()
        v[at] = what
        got = dmm.paged_attention(q, k, v, table, lens)
        v[at] = kept
        assert not bool(torch.isfinite(got[seq, group:, 77]).any())
        mended, rest = got.clone(), want.clone()
        mended[seq, group:, 77] = 0
        rest[seq, group:, 77] = 0
        assert check_attention(mended, rest, bound) == got.numel()
    assert dmm.status() == 0


@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan])
def test_a_key_that_is_not_finite_shows_in_the_rows_that_see_it(what):
    # against queries of either sign its score is inf - inf
    gen = generator(4)
    k, v, table, lens = make_cache(gen, [200, 30], 2, 128, 16, FP16)
    q = torch.randn((230, 16, 128), generator=gen, device="cuda").to(FP16)
    want, bound = attention(q, k, v, table, lens, cu_of([200, 30]))
    k[int(table[0, 70 // 16]), 1, 70 % 16] = what
    got = dmm.prompt_attention(q, k, v, table, lens, cu_of([200, 30]))
    assert not bool(torch.isfinite(got[70:200, 8:]).any())
    got[70:200, 8:] = 0
    want[70:200, 8:] = 0
    assert check_attention(got, want, bound) == got.numel()
    last = torch.tensor([199, 229], device="cuda")
    one = dmm.paged_attention(q[last], k, v, table, lens)
    assert not bool(torch.isfinite(one[0, 8:]).any())
    one[0, 8:] = 0
    assert check_attention(one, want[last], bound[last]) == one.numel()


@pytest.mark.parametrize("new,length,at", [(256, 256, 255), (256, 256, 130), (256, 100, 50), (250, 700, 640), (200, 30, 0)])
@pytest.mark.parametrize("D", [64, 128])
def test_a_value_that_only_the_second_tile_of_rows_sees(new, length, at, D):
    """Two tiles of 128 rows are worked on together; the first is done, or has nothing to do, while the values that the second sees are
    still looked at."""
    gen = generator(6)
    k, v, table, lens = make_cache(gen, [length] * 4, 64, D, 64, BF16)
    q = torch.randn((4 * new, 64, D), generator=gen, device="cuda").to(BF16)
    cu = cu_of([new] * 4)
    want, bound = attention(q, k, v, table, lens, cu)
    for b in (0, 1, 3):
        v[int(table[b, at // 64]), :, at % 64, 9] = math.inf
    sees = torch.arange(length - new, length, device="cuda") >= at
    for _ in range(3):
        got = dmm.prompt_attention(q, k, v, table, lens, cu)
        rest = want.clone()
        for b in (0, 1, 3):
            rows = torch.nonzero(sees)[:, 0] + b * new
            assert not bool(torch.isfinite(got[rows, :, 9]).any())
            got[rows, :, 9] = 0
            rest[rows, :, 9] = 0
        assert check_attention(got, rest, bound) == got.numel()
    assert dmm.status() == 0


def test_a_context_whose_item_takes_most_of_a_second():
    """2^26 keys of every key head, all of them one page, and an item of one row for each CTA: warps that have nothing to do for it wait as
    long as it takes."""
    gen = generator(7)
    n, page, heads = 2 ** 26, 4096, torch.cuda.get_device_properties(0).multi_processor_count
    k = torch.randn((1, heads, page, 64), generator=gen, device="cuda").to(BF16)
    v = (1.0 + 0.1 * torch.randn((1, heads, page, 64), generator=gen, device="cuda")).to(BF16)
    table = torch.zeros((1, n // page), dtype=torch.int32, device="cuda")
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    q = torch.randn((1, heads, 64), generator=gen, device="cuda").to(BF16)
    got = dmm.prompt_attention(q, k, v, table, lens, cu_of([1]))
    assert dmm.status() == 0
    # every key is there 2^14 times, which is the same average.  The products add 16 keys at a time, 2^22 times, each off by a step of the
    # sum at most, the sum of weights 128 at a time
    want, bound = attention(q, k, v, table, lens.clamp(max=page), cu_of([1]))
    assert check_attention(got, want, bound + (2.0 ** 22 * 2.0 ** -23 + 2.0 ** 19 * 2.0 ** -24) * want.abs()) == got.numel()


def test_a_sequence_without_tokens_has_an_idle_place_in_a_batch():
    """Without cu_seqlens every sequence has a row; that of an empty one is left alone and raises nothing."""
    gen = generator(5)
    k, v, table, lens = make_cache(gen, [20, 0, 33, 0], 2, 64, 16, FP16)
    k0, v0 = k.clone(), v.clone()
    qkv = torch.randn((4, 8 * 64), generator=gen, device="cuda")
    qkv[1::2] = math.nan
    q = torch.full((4, 4, 64), math.nan, dtype=FP16, device="cuda")
    dmm.append_kv(qkv, k, v, table, lens, dmm.rotary_frequencies(64, device="cuda"), q)
    assert dmm.status() == 0 and bool(torch.isnan(q[1::2]).all()) and bool(torch.isfinite(q[::2]).all())
    for b, n in ((0, 20), (2, 33)):
        at = int(table[b, (n - 1) // 16]), slice(None), (n - 1) % 16
        assert torch.equal(v[at], qkv[b].view(8, 64)[6:].to(FP16))
        k0[at], v0[at] = k[at], v[at]
    assert torch.equal(k.view(torch.int16), k0.view(torch.int16)) and torch.equal(v.view(torch.int16), v0.view(torch.int16))
    got = dmm.paged_attention(q, k, v, table, lens)
    assert dmm.status() == 0 and bool((got[1::2] == 0).all())
    want, bound = attention(torch.nan_to_num(q), k, v, table, lens, None)
    assert check_attention(got, want, bound) == got.numel()


def test_caches_and_stacks_know_their_device():
    # "cuda" is whichever device is current at the time
    here = torch.device("cuda", torch.cuda.current_device())
    assert dmm.PagedCache(1, 1, 64, 2, device="cuda").device == here
    cb = dmm.codebook_to_fp16(dmm.pack_codebook(dmm.synthetic_codebook(42)))
    assert LinearStack(dict(hidden=256, kv_heads=2, head_dim=64, ffn=256, layers=1), cb, "cuda").device == here
