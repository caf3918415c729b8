"""The attention operators that sit between the quantised products of a transformer block, as cases that can be timed.

Three kinds of work, by ``op``:

* ``append``  the fp32 result of the qkv product becomes rotated 16-bit queries and, through a page table, new rows of a
  paged key-value cache.
* ``decode``  attention of one new token per sequence over that cache.
* ``prompt``  causal attention of packed prompts (or of the next chunk of prompts) over that cache.

``listed()`` and ``draw()`` give the cases, ``prepare()`` makes what a program has in hand before the call, ``run()`` is
one pass: the framework's calls where ``own`` is true, elementary torch operations in 32 bits elsewhere.  ``work()`` is
what a pass cannot do without, ``exact()`` the answer in 64 bits.

The head layouts are those of the two transformer stacks of this framework (64 query heads over 8 key heads, 32 over 32,
128 values each) and of their tensor-parallel shards (32 over 4, 8 over 1).
"""
import math
import random

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
BASE = 10000.0  # of the rotation's frequencies


def _case(name, op, heads, kv_heads, batch, new, past, page, dtype="fp16", head_dim=128, interleaved=False):
    """``new`` and ``past``: the shortest and the longest number of new tokens and of tokens before them, over the sequences."""
    case = dict(op=op, heads=heads, kv_heads=kv_heads, head_dim=head_dim, batch=batch, new_min=new[0], new_max=new[1],
                past_min=past[0], past_max=past[1], page=page, dtype=dtype, interleaved=interleaved)
    return dict(name=name, **case) if name else case


def listed():
    return [
        # one new token of the 70B stack: nothing but latency
        _case("append_70b_b1", "append", 64, 8, 1, (1, 1), (4000, 4000), 64),
        # a decoding step of 32 requests of the 7B stack
        _case("append_7b_b32", "append", 32, 32, 32, (1, 1), (1, 300), 16),
        # the prompt length that the framework's benchmark of products uses
        _case("append_70b_2048", "append", 64, 8, 1, (2048, 2048), (0, 0), 128),
        # several prompts of different lengths that continue earlier chunks, neighbouring values rotated as pairs
        _case("append_70b_ragged", "append", 64, 8, 9, (7, 4096), (0, 70000), 32, "bf16", interleaved=True),
        # one request of the 70B stack at the end of that model's context
        _case("decode_70b_b1", "decode", 64, 8, 1, (1, 1), (4095, 4095), 64),
        # sixteen requests of it, some just begun
        _case("decode_70b_b16", "decode", 64, 8, 16, (1, 1), (0, 4095), 16),
        # a batch of the 7B stack, which has a key head for every query head
        _case("decode_7b_b32", "decode", 32, 32, 32, (1, 1), (100, 2047), 128),
        # one of eight ranks of the 70B stack, a few long contexts
        _case("decode_long", "decode", 8, 1, 5, (1, 1), (3000, 131071), 64, "bf16"),
        # the prompt of the benchmark of products
        _case("prompt_70b_2048", "prompt", 64, 8, 1, (2048, 2048), (0, 0), 64),
        # prompts as they come: from a single token on, of no round length
        _case("prompt_7b_ragged", "prompt", 32, 32, 13, (1, 1531), (0, 0), 16),
        # a long prompt, the largest case
        _case("prompt_70b_8192", "prompt", 64, 8, 1, (8192, 8192), (0, 0), 128),
        # the next chunks of long prompts on one of two ranks: few new rows, many keys
        _case("prompt_chunks", "prompt", 32, 4, 4, (33, 512), (511, 16384), 32, "bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """One more case: groups of 1 to 8 query heads per key head, 64 or 128 values per head, 1 to 64 sequences, prompts of 1
    to 8192 tokens, contexts of up to 131072, pages of 16 to 128 tokens."""
    most = work(next(c for c in listed() if c["name"] == "prompt_70b_8192"))
    while True:
        op = rng.choice(["append", "decode", "prompt"])
        kv_heads = rng.choice([1, 2, 4, 8, 8, 16, 32])
        group = rng.choice([g for g in (1, 2, 3, 4, 5, 6, 7, 8, 8) if g * kv_heads <= 64])
        batch = _log(rng, 1, 64)
        new_max = 1 if op == "decode" or (op == "append" and rng.random() < 0.4) else _log(rng, 16, 8192)
        past_max = rng.choice([0, _log(rng, 1, 131071)]) if op != "decode" else _log(rng, 16, 131071)
        case = _case(None, op, group * kv_heads, kv_heads, batch, (rng.choice([1, _log(rng, 1, new_max)]), new_max),
                     (rng.choice([0, past_max // 3]), past_max), rng.choice([16, 32, 64, 128]), rng.choice(["fp16", "bf16"]),
                     rng.choice([64, 128, 128]), op == "append" and rng.random() < 0.3)
        new, past = _lengths(case)
        scores = batch * case["heads"] * max(new) * (max(new) + max(past))
        cost = work(case)
        cache = (sum(new) + sum(past)) * kv_heads * case["head_dim"] * 4
        # no more than the largest listed case; and the plain form pads every sequence to the longest
        if (cost["flops"] <= most["flops"] and cost["bytes"] <= 2e9 and cache <= 2e9 and (op == "append" or scores <= 64 * 8192 * 8192)
                and (op == "append" or batch * (max(new) + max(past)) * kv_heads * case["head_dim"] * 8 <= 8e9)):
            return case


def _lengths(case):
    """New tokens and earlier tokens of every sequence: the longest first, the shortest last, the others in between."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))

    def some(lo, hi):
        between = [rng.choice([_log(rng, max(lo, 1), max(hi, 1)), rng.randint(lo, hi)]) if hi > lo else hi for _ in range(case["batch"])]
        return [hi] + between[1:-1] + ([lo] if case["batch"] > 1 else [])

    return some(case["new_min"], case["new_max"]), some(case["past_min"], case["past_max"])


def _frequencies(case):
    half = torch.arange(case["head_dim"] // 2, dtype=torch.float64, device="cuda")
    return BASE ** (-2.0 * half / case["head_dim"])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, D, Hkv, H, page = _TYPES[case["dtype"]], case["head_dim"], case["kv_heads"], case["heads"], case["page"]
    new, past = _lengths(case)
    total = [n + p for n, p in zip(new, past)]
    pages = [-(-n // page) for n in total]
    order = torch.randperm(sum(pages) + 3, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((len(new), max(pages)), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    state = dict(case=case, new_max=max(new), len_max=max(total), table=table,
                 seq_lens=torch.tensor(total, dtype=torch.int32, device="cuda"),
                 cu=torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda"),
                 # keys have channels with a mean of their own, as trained ones do
                 k=(randn(len(order), Hkv, page, D) + randn(D)).to(dtype), v=(randn(len(order), Hkv, page, D) + 0.25 * randn(D)).to(dtype))
    if case["op"] == "append":
        state.update(qkv=2.0 * randn(sum(new), (H + 2 * Hkv) * D), freqs=_frequencies(case))
    else:
        state["q"] = randn(sum(new), H, D).to(dtype)
    return state


# ------------------------------------------------ the plain forms ------------------------------------------------
def _rotate(x, cos, sin, interleaved):
    """x [T, heads, D]; cos, sin [T, 1, D / 2]."""
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    a, b = a * cos - b * sin, a * sin + b * cos
    return torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)


def _plain_append(s):
    case = s["case"]
    D, Hkv, H, page = case["head_dim"], case["kv_heads"], case["heads"], case["page"]
    cu, lens = s["cu"].long(), s["seq_lens"].long()
    token = torch.arange(s["qkv"].shape[0], device="cuda")
    seq = torch.bucketize(token, cu[1:], right=True)
    pos = lens[seq] - (cu[seq + 1] - token)
    angle = pos.double()[:, None] * s["freqs"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q, k, v = s["qkv"].view(-1, H + 2 * Hkv, D).split((H, Hkv, Hkv), 1)
    where = s["table"][seq, pos // page].long()
    s["k"][where, :, pos % page] = _rotate(k, cos, sin, case["interleaved"]).to(s["k"].dtype)
    s["v"][where, :, pos % page] = v.to(s["v"].dtype)
    return _rotate(q, cos, sin, case["interleaved"]).to(s["k"].dtype), s["k"], s["v"]


def _plain_attention(s):
    """Every sequence padded to the longest; [batch, kv head, new token x query head of the group, key]."""
    case = s["case"]
    D, Hkv, page, group = case["head_dim"], case["kv_heads"], case["page"], case["heads"] // case["kv_heads"]
    cu, lens, B, Q, L = s["cu"].long(), s["seq_lens"].long(), case["batch"], s["new_max"], s["len_max"]
    key = torch.arange(L, device="cuda")
    where = s["table"][:, key // page].long()
    k = s["k"][where, :, key % page].permute(0, 2, 1, 3).float()  # [B, Hkv, L, D]
    v = s["v"][where, :, key % page].permute(0, 2, 1, 3).float()
    token = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.bucketize(token, cu[1:], right=True)
    row = token - cu[seq]
    q = torch.zeros((B, Q, case["heads"], D), device="cuda")
    q[seq, row] = s["q"].float()
    q = q.view(B, Q, Hkv, group, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, Q * group, D)
    scores = (q * D ** -0.5) @ k.transpose(2, 3)
    last = lens[:, None] - (cu[1:] - cu[:-1])[:, None] + torch.arange(Q, device="cuda")  # [B, Q]: the last key that a row sees
    hidden = key > torch.minimum(last, lens[:, None] - 1)[:, :, None]
    scores.view(B, Hkv, Q, group, L).masked_fill_(hidden[:, None, :, None], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    out = (scores @ v) / scores.sum(-1, keepdim=True)
    out = out.view(B, Hkv, Q, group, D).permute(0, 2, 1, 3, 4).reshape(B, Q, case["heads"], D)
    return out[seq, row].to(s["q"].dtype)


def run(state):
    op = state["case"]["op"]
    if not own:
        return _plain_append(state) if op == "append" else _plain_attention(state)
    import decode_matmul_b200 as dmm

    cache = (state["k"], state["v"], state["table"], state["seq_lens"])
    if op == "append":
        cu = None if state["new_max"] == 1 else state["cu"]
        q = dmm.append_kv(state["qkv"], *cache, state["freqs"], cu_seqlens=cu, interleaved=state["case"]["interleaved"])
        return q, state["k"], state["v"]
    if op == "decode":
        return dmm.paged_attention(state["q"], *cache)
    return dmm.prompt_attention(state["q"], *cache, state["cu"])


def work(case):
    D, Hkv, H = case["head_dim"], case["kv_heads"], case["heads"]
    new, past = _lengths(case)
    tokens, total = sum(new), sum(new) + sum(past)
    if case["op"] == "append":
        # the fp32 result read, 16-bit queries, keys and values written; a product and a sum for each value that turns
        return {"bytes": tokens * (H + 2 * Hkv) * D * 6, "flops": 3 * tokens * (H + Hkv) * D}
    # queries and the rows of the cache read, outputs written; two products for each pair of a query and a key that it sees
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past))
    return {"bytes": (2 * tokens * H + 2 * total * Hkv) * D * 2, "flops": 4 * pairs * H * D}


# ----------------------------------------- the same in 64 bits, sequence by sequence -----------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    D, Hkv, H, page = case["head_dim"], case["kv_heads"], case["heads"], case["page"]
    group = H // Hkv
    new, past = _lengths(case)
    if case["op"] == "append":
        qkv = s["qkv"].double()
        q, k, v = torch.empty((len(qkv), H, D), dtype=torch.float64, device="cuda"), s["k"].double(), s["v"].double()
        t0 = 0
        for b, (n, p) in enumerate(zip(new, past)):
            x = qkv[t0:t0 + n].view(n, H + 2 * Hkv, D)
            # a pair (a, b) as the complex number a + ib, turned by the unit number of its angle
            angle = torch.arange(p, p + n, dtype=torch.float64, device="cuda")[:, None] * s["freqs"]
            turn = torch.polar(torch.ones_like(angle), angle)[:, None]
            z = x[:, :H + Hkv]
            z = z.unflatten(-1, (D // 2, 2)) if case["interleaved"] else z.unflatten(-1, (2, D // 2)).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
            z = (z if case["interleaved"] else z.transpose(-1, -2)).reshape(n, H + Hkv, D)
            q[t0:t0 + n] = z[:, :H]
            rows = torch.arange(p, p + n, device="cuda")
            pg = s["table"][b].long()[rows // page]
            k[pg, :, rows % page] = z[:, H:]
            v[pg, :, rows % page] = x[:, H + Hkv:]
            t0 += n
        return q, k, v
    q = s["q"].double()
    out = torch.empty_like(q)
    t0 = 0
    for b, (n, p) in enumerate(zip(new, past)):
        rows = torch.arange(n + p, device="cuda")
        pg = s["table"][b].long()[rows // page]
        seen = rows[None, :] <= torch.arange(p, p + n, device="cuda")[:, None]
        for h in range(H):
            k, v = s["k"][pg, h // group, rows % page].double(), s["v"][pg, h // group, rows % page].double()
            x = torch.where(seen, q[t0:t0 + n, h] @ k.T / math.sqrt(D), -math.inf)
            out[t0:t0 + n, h] = torch.softmax(x, -1) @ v
        t0 += n
    return out
