"""The stack with a cache: blocks that attend, against the same blocks in torch, and in the two ways a prompt can be served."""
import math

import pytest
import torch

import decode_matmul_b200 as dmm
from decode_matmul_b200.linear import LinearStack

pytestmark = pytest.mark.gpu
CFG = dict(hidden=512, kv_heads=2, head_dim=64, ffn=1024, layers=2)
WIDE = dict(hidden=1024, kv_heads=4, head_dim=128, ffn=1280, layers=2)


def stack_of(cfg, scale=2.0 ** -6):
    return LinearStack(cfg, dmm.codebook_to_fp16(dmm.pack_codebook(dmm.synthetic_codebook(42))), "cuda", seed=3, scale=scale)


def cache_of(cfg, **kw):
    args = dict(num_pages=40, page_size=16, max_seqs=3, max_pages=20)
    args.update(kw)
    return dmm.PagedCache(cfg["layers"], cfg["kv_heads"], cfg["head_dim"], **args)


def reference(stack, cfg, h, new):
    """The blocks over whole prompts, in 64 bits, rounded to fp16 where the stack rounds: inputs of products, queries, keys,
    values and attention results."""
    half = lambda t: t.to(torch.float16).double()  # noqa: E731
    D, Hkv = cfg["head_dim"], cfg["kv_heads"]
    H = cfg["hidden"] // D
    freqs = dmm.rotary_frequencies(D, device="cuda")
    pos = torch.cat([torch.arange(n, device="cuda") for n in new]).double()
    cos, sin = (pos[:, None] * freqs).cos()[:, None], (pos[:, None] * freqs).sin()[:, None]
    seq = torch.cat([torch.full((n,), b, device="cuda") for b, n in enumerate(new)])
    hidden = (seq[:, None] != seq[None, :]) | (pos[None, :] > pos[:, None])
    h = h.double()
    product = lambda x, lin: half(x) @ dmm.decode_weights(lin.codes, lin.codebook).double().T * lin.scale  # noqa: E731

    def turn(x):
        a, b = x[..., :D // 2], x[..., D // 2:]
        return half(torch.cat((a * cos - b * sin, a * sin + b * cos), -1))

    for blk in stack.layers:
        q, k, v = product(h, blk["qkv"]).view(-1, H + 2 * Hkv, D).split((H, Hkv, Hkv), 1)
        q, k, v = turn(q), turn(k).repeat_interleave(H // Hkv, 1), half(v).repeat_interleave(H // Hkv, 1)
        x = torch.einsum("thd,shd->hts", q, k) / math.sqrt(D)
        p = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
        h = h + product(half(torch.einsum("hts,shd->thd", p, v)).flatten(1), blk["o"])
        g = product(h, blk["gate_up"])
        h = h + product(torch.nn.functional.silu(g[:, :cfg["ffn"]]) * g[:, cfg["ffn"]:], blk["down"])
    return h


def near(a, b, blocks):
    """Relative distance of two results whose every attention may be off by two half steps of fp16 and whose roundings may fall to the
    other side: four half steps for each block."""
    rel = float((a.double() - b.double()).norm() / b.double().norm())
    assert rel <= blocks * 4 * 2.0 ** -11, rel


@pytest.mark.parametrize("cfg", [CFG, WIDE])
@pytest.mark.parametrize("new", [[20, 0, 7], [1, 1, 1], [130, 40, 3]])
def test_a_prompt_through_the_blocks(cfg, new):
    stack, cache = stack_of(cfg), cache_of(cfg)
    gen = torch.Generator(device="cuda").manual_seed(1)
    h = torch.randn((sum(new), cfg["hidden"]), generator=gen, device="cuda")
    want = reference(stack, cfg, h, new)
    got = stack.step(h.clone(), cache=cache, cu_seqlens=cache.extend(new))
    assert dmm.status() == 0
    near(got, want, cfg["layers"])


@pytest.mark.parametrize("cfg", [CFG, WIDE])
def test_token_by_token_is_the_prompt(cfg):
    """Three sequences as one batch of prompts, and the same with their ends token by token, each path with its own launches."""
    stack = stack_of(cfg)
    gen = torch.Generator(device="cuda").manual_seed(2)
    lengths, tail = [37, 18, 50], 6
    rows = [torch.randn((n, cfg["hidden"]), generator=gen, device="cuda") for n in lengths]
    whole = cache_of(cfg)
    want = stack.step(torch.cat(rows), cache=whole, cu_seqlens=whole.extend(lengths)).split(lengths)
    cache = cache_of(cfg)
    got = [list(t) for t in zip(stack.step(torch.cat([r[:-tail] for r in rows]), cache=cache,
                                           cu_seqlens=cache.extend([n - tail for n in lengths])).split([n - tail for n in lengths]))]
    for i in range(tail):
        h = torch.stack([r[len(r) - tail + i] for r in rows])
        out = stack.step(h, cache=cache, cu_seqlens=cache.extend([1, 1, 1]), fused=i % 2 == 0)
        for b in range(3):
            got[b].append(out[b:b + 1].clone())
    assert dmm.status() == 0
    for b in range(3):
        near(torch.cat(got[b]), want[b], 2 * cfg["layers"])


def test_decoding_step_in_a_graph():
    """A captured step serves growing sequences: extend() outside, replay() inside."""
    stack, cache, twin = stack_of(CFG), cache_of(CFG), cache_of(CFG)
    gen = torch.Generator(device="cuda").manual_seed(3)
    start = torch.randn((3 * 20, CFG["hidden"]), generator=gen, device="cuda")
    for c in (cache, twin):
        stack.step(start.clone(), cache=c, cu_seqlens=c.extend([20, 20, 20]))
    # (captured on sequences that have room for every token to come; lengths are set back afterwards)
    h = torch.zeros((3, CFG["hidden"]), device="cuda")
    side = torch.cuda.Stream()
    cache.extend([1, 1, 1])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        stack.step(h, cache=cache)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        stack.step(h, cache=cache)
    cache.seq_lens -= 1
    cache.lengths = [n - 1 for n in cache.lengths]
    for i in range(15):
        x = torch.randn(h.shape, generator=gen, device="cuda")
        assert cache.extend([1, 1, 1]) is None and twin.extend([1, 1, 1]) is None
        h.copy_(x)
        graph.replay()
        want = stack.step(x.clone(), cache=twin)
        near(h, want, CFG["layers"])
    assert dmm.status() == 0 and torch.equal(cache.seq_lens, twin.seq_lens)


def test_a_cache_that_does_not_fit_is_refused():
    stack = stack_of(CFG)
    h = torch.zeros((3, CFG["hidden"]), device="cuda")
    for kw in (dict(layers=1), dict(kv_heads=4), dict(head_dim=128)):
        with pytest.raises(RuntimeError, match="cache must be"):
            stack.step(h, cache=cache_of(dict(CFG, **kw)))
    with pytest.raises(RuntimeError, match="cache must be"):
        stack.step(h, cache=cache_of(CFG, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="one row per sequence"):
        stack.step(h[:2], cache=cache_of(CFG))


def test_without_a_cache_nothing_has_changed():
    stack = stack_of(CFG)
    h = torch.randn((2, CFG["hidden"]), device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    a = stack.step(h.clone(), fused=False)
    b = h.clone()
    for blk in stack.layers:  # q stands in for the attention's result
        q = blk["qkv"](b.to(torch.float16))[:, :CFG["hidden"]]
        blk["o"](q.to(torch.float16).contiguous(), out=b, accumulate=True)
        g = blk["gate_up"](b.to(torch.float16))
        blk["down"]((torch.nn.functional.silu(g[:, :CFG["ffn"]]) * g[:, CFG["ffn"]:]).to(torch.float16), out=b, accumulate=True)
    assert torch.equal(a, b)


def test_a_captured_step_outlives_steps_of_other_batches():
    """Prompts that come between the replays of a captured step take other buffers than the graph's, and leave those alone."""
    stack, cache, twin = stack_of(CFG), cache_of(CFG), cache_of(CFG)
    gen = torch.Generator(device="cuda").manual_seed(5)
    start = torch.randn((3 * 20, CFG["hidden"]), generator=gen, device="cuda")
    for c in (cache, twin):
        stack.step(start.clone(), cache=c, cu_seqlens=c.extend([20, 20, 20]))
    h = torch.zeros((3, CFG["hidden"]), device="cuda")
    cache.extend([1, 1, 1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        stack.step(h, cache=cache)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        stack.step(h, cache=cache)
    kept = [t.data_ptr() for t in stack._buffers(3).values()]
    cache.seq_lens -= 1
    cache.lengths = [n - 1 for n in cache.lengths]
    for i in range(6):
        x = torch.randn((3, CFG["hidden"]), generator=gen, device="cuda")
        assert cache.extend([1, 1, 1]) is None and twin.extend([1, 1, 1]) is None
        h.copy_(x)
        graph.replay()
        near(h, stack.step(x.clone(), cache=twin), CFG["layers"])
        rows = torch.randn((5 + i, CFG["hidden"]), generator=gen, device="cuda")
        for c in (cache, twin):
            stack.step(rows.clone(), cache=c, cu_seqlens=c.extend([i, 5, 0]))
        assert [t.data_ptr() for t in stack._buffers(3).values()] == kept
        assert not {t.data_ptr() for t in stack._buffers(5 + i).values()} & set(kept)
    assert dmm.status() == 0


@pytest.mark.parametrize("fused", [True, False])
def test_rows_behind_the_last_sequence(fused):
    """A padded batch: its last rows are no sequence's; the others are as without them, the cache too."""
    stack, cache, twin = stack_of(CFG), cache_of(CFG), cache_of(CFG)
    gen = torch.Generator(device="cuda").manual_seed(6)
    rows = torch.randn((13, CFG["hidden"]), generator=gen, device="cuda")
    del [torch.full((21, CFG["hidden"]), math.nan, dtype=torch.float16, device="cuda") for _ in range(16)][:]  # (what new tensors may lie on)
    got = stack.step(torch.cat([rows, rows[:8]]), cache=cache, cu_seqlens=cache.extend([4, 0, 9]), fused=fused)
    want = stack.step(rows.clone(), cache=twin, cu_seqlens=twin.extend([4, 0, 9]), fused=fused)
    near(got[:13], want, CFG["layers"])
    assert bool(torch.isfinite(got).all()) and dmm.status() == 0
    near(cache.pages.float(), twin.pages.float(), CFG["layers"])


def test_the_first_step_with_a_cache_is_not_captured():
    stack, cache = stack_of(CFG), cache_of(CFG)
    h = torch.zeros((3, CFG["hidden"]), device="cuda")
    cache.extend([1, 1, 1])
    stack.step(h, fused=False)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            stack.step(h, cache=cache)


def test_a_captured_step_goes_on_while_sequences_come_and_go():
    """One of three sequences ends between replays and another takes its place: the others' rows are what they are without it."""
    stack, cache, twin = stack_of(CFG), cache_of(CFG), cache_of(CFG)
    gen = torch.Generator(device="cuda").manual_seed(7)
    start = torch.randn((3 * 20, CFG["hidden"]), generator=gen, device="cuda")
    for c in (cache, twin):
        stack.step(start.clone(), cache=c, cu_seqlens=c.extend([20, 20, 20]))
    h = torch.zeros((3, CFG["hidden"]), device="cuda")
    cache.extend([1, 1, 1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        stack.step(h, cache=cache)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        stack.step(h, cache=cache)
    cache.seq_lens -= 1
    cache.lengths = [n - 1 for n in cache.lengths]
    for i in range(12):
        if i == 3:
            cache.release(1)
            twin.release(1)
        if i == 8:  # (a new prompt comes in)
            rows = torch.randn((9, CFG["hidden"]), generator=gen, device="cuda")
            for c in (cache, twin):
                stack.step(rows.clone(), cache=c, cu_seqlens=c.extend([0, 9, 0]))
        new = [1, 0, 1] if 3 <= i < 8 else [1, 1, 1]
        x = torch.randn((3, CFG["hidden"]), generator=gen, device="cuda")
        assert cache.extend(new, idle=True) is None
        h.copy_(x)
        graph.replay()
        live = torch.tensor([b for b in range(3) if new[b]], device="cuda")
        near(h[live], stack.step(x[live], cache=twin, cu_seqlens=twin.extend(new)), 2 * CFG["layers"])
        assert bool(torch.isfinite(h).all()) and torch.equal(cache.seq_lens, twin.seq_lens)
    assert dmm.status() == 0
