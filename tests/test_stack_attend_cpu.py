"""LinearStack.step with a cache over two gloo ranks, each with its key heads and their cache, against the same stack on one: the
oracle stands in for the products and plain torch for the attention operators."""
import math
import os
import sys

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CFG = dict(hidden=256, kv_heads=2, head_dim=64, ffn=512, layers=2)


def _plain_operators(put):
    """Takes the place of the kernels in this process."""
    import decode_matmul_b200 as dmm
    from decode_matmul_b200 import attention, linear
    from oracle import dmm_oracle as o

    def product(self, x, out=None, accumulate=False, path=0, pdl=True):
        codes = dmm.untranspose_tile(self.codes).numpy()
        y = torch.from_numpy(o.decode_matmul_f16(np.ascontiguousarray(x.numpy()), codes, self.codebook.numpy(), self.scale)).float()
        if out is None:
            return y
        out.copy_(out + y if accumulate else y)
        return out

    def spans(lens, cu):
        cu = list(range(len(lens) + 1)) if cu is None else cu.tolist()
        return [(b, cu[b], cu[b + 1], int(n)) for b, n in enumerate(lens.tolist())]

    def append(qkv, k, v, table, lens, freqs, cu_seqlens=None, pdl=False):
        D, page, kv = k.shape[3], k.shape[2], k.shape[1]
        heads = qkv.shape[1] // D - 2 * kv
        x = qkv.view(len(qkv), -1, D).double()
        q = torch.zeros((len(qkv), heads, D), dtype=k.dtype)
        for b, t0, t1, n in spans(lens, cu_seqlens):
            for t in range(t0, t1):
                pos = n - (t1 - t)
                c, s = (pos * freqs).cos(), (pos * freqs).sin()
                r = x[t].clone()
                a, z = x[t, :heads + kv, :D // 2], x[t, :heads + kv, D // 2:]
                r[:heads + kv] = torch.cat((a * c - z * s, a * s + z * c), -1)
                q[t] = r[:heads].to(k.dtype)
                where = int(table[b, pos // page])
                k[where, :, pos % page], v[where, :, pos % page] = r[heads:heads + kv].to(k.dtype), r[heads + kv:].to(k.dtype)
        return q

    def attend(q, k, v, table, lens, cu=None, output=None, pdl=False):
        page, group = k.shape[2], q.shape[1] // k.shape[1]
        out = torch.zeros_like(q) if output is None else output
        for b, t0, t1, n in spans(lens, cu):
            where = [int(table[b, p // page]) for p in range(n)]
            kk, vv = (torch.stack([x[w, :, p % page] for p, w in enumerate(where)]).double().repeat_interleave(group, 1) for x in (k, v))
            for t in range(t0, t1):
                sees = n - (t1 - t) + 1
                w = torch.softmax(torch.einsum("hd,nhd->hn", q[t].double(), kk[:sees]) / math.sqrt(q.shape[2]), -1)
                out[t] = torch.einsum("hn,nhd->hd", w, vv[:sees]).to(q.dtype)
        return out

    put(linear.DecodeLinear, "__call__", product)
    put(attention, "append_kv", append)
    put(attention, "paged_attention", attend)
    put(attention, "prompt_attention", attend)
    put(torch.cuda, "is_current_stream_capturing", lambda: False)


def _steps(stack, world):
    """A prompt of three sequences, then two single tokens of each."""
    import decode_matmul_b200 as dmm

    cache = dmm.PagedCache(CFG["layers"], CFG["kv_heads"] // world, CFG["head_dim"], 9, page_size=16, max_seqs=3, device="cpu")
    gen = torch.Generator().manual_seed(5)
    out = [stack.step(torch.randn((26, CFG["hidden"]), generator=gen), cache=cache, cu_seqlens=cache.extend([20, 1, 5]), fused=False)]
    for _ in range(2):
        out.append(stack.step(torch.randn((3, CFG["hidden"]), generator=gen), cache=cache, cu_seqlens=cache.extend([1, 1, 1]), fused=False))
    return torch.cat(out), cache


def _worker(rank, world, port, results):
    sys.path.insert(0, ROOT)
    import decode_matmul_b200 as dmm
    from decode_matmul_b200.linear import LinearStack

    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    _plain_operators(setattr)
    cb = dmm.synthetic_codebook(42)
    cb = torch.from_numpy(cb) if isinstance(cb, np.ndarray) else cb
    args = dict(logical_seed=11, scale=2.0 ** -8)
    got, part = _steps(LinearStack(CFG, cb, "cpu", world=world, rank=rank, **args), world)
    want, whole = _steps(LinearStack(CFG, cb, "cpu", **args), 1)
    kv = CFG["kv_heads"] // world
    mine = whole.pages[:, :, :, rank * kv:(rank + 1) * kv]
    off = [float((a.double() - b.double()).norm() / b.double().norm()) for a, b in ((got, want), (part.pages, mine))]
    results[rank] = (*off, float(got.norm()))
    dist.destroy_process_group()


def test_two_ranks_attend_as_one():
    """Sums over the ranks come in another order, so values that are rounded to fp16 may fall to the other side: four half steps for each
    block, as between the forms of a step on one GPU."""
    world = 2
    port = 33500 + os.getpid() % 2000
    with mp.Manager() as mgr:
        results = mgr.dict()
        mp.spawn(_worker, args=(world, port, results), nprocs=world, join=True)
        for rank in range(world):
            rows, pages, size = results[rank]
            assert size > 0 and rows <= CFG["layers"] * 4 * 2.0 ** -11 and pages <= CFG["layers"] * 4 * 2.0 ** -11, dict(results)


@pytest.mark.parametrize("cfg,world", [
    (dict(CFG, kv_heads=1, head_dim=128), 2),   # half a key head each
    (dict(CFG, hidden=384, kv_heads=3), 2),     # one and a half
    (dict(CFG, hidden=192, kv_heads=2, ffn=256), 2),  # one and a half query heads
])
def test_heads_that_do_not_shard_are_refused(monkeypatch, cfg, world):
    import decode_matmul_b200 as dmm
    from decode_matmul_b200.linear import LinearStack

    _plain_operators(monkeypatch.setattr)
    monkeypatch.setattr(dist, "all_reduce", lambda t, group=None: None)
    stack = LinearStack(cfg, dmm.synthetic_codebook(42), "cpu", world=world, rank=0, logical_seed=1)
    cache = dmm.PagedCache(cfg["layers"], max(1, cfg["kv_heads"] // world), cfg["head_dim"], 4, page_size=16, device="cpu")
    before = cache.pages.clone()
    with pytest.raises(RuntimeError, match="heads"):
        stack.step(torch.zeros((1, cfg["hidden"])), cache=cache, cu_seqlens=cache.extend([1]), fused=False)
    assert torch.equal(cache.pages, before)
