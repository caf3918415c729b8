"""The check of an item's record before the kernel that joins parts follows it (csrc/dmm_attn_item.h), compiled by itself: no GPU needed."""
import ctypes
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FIELDS = ("seq", "head", "begin", "n", "len", "token0", "first", "end", "slot", "ctas")

_SHIM = """
#include "dmm_attn_item.h"
extern "C" int fields() { return sizeof(dmm::PromptItem) / sizeof(int); }
extern "C" int crosses(const int *f, int x, int ctas, int kv_heads, int tokens) {
    const dmm::PromptItem it = {f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7], f[8], f[9]};
    return dmm::prompt_item_crosses(it, x, ctas, kv_heads, tokens);
}
"""


@pytest.fixture(scope="module")
def item(tmp_path_factory):
    d = tmp_path_factory.mktemp("item")
    (d / "shim.cpp").write_text(_SHIM)
    so = str(d / "shim.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fsanitize-undefined-trap-on-error", "-shared", "-fPIC", "-I",
                    os.path.join(ROOT, "decode_matmul_b200", "csrc"), "-o", so, str(d / "shim.cpp")], check=True)
    lib = ctypes.CDLL(so)
    assert lib.fields() == len(FIELDS)
    return lambda f, *size: lib.crosses((ctypes.c_int * 10)(*(f[k] for k in FIELDS)), *size) != 0


def reaches(f, x, kv_heads, group):
    """Slots of the workspace, rows and query heads of the output that the join of item ``f`` from CTA x on comes to."""
    slots = {f["slot"]} | {2 * (x + s) for s in range(1, f["ctas"])}
    tile_tokens = 128 // group
    rows, heads = set(), set()
    for row in range(256):
        tok = row % 128 // group
        token = f["token0"] + row // 128 * tile_tokens + tok
        if tok < tile_tokens and token < f["n"]:
            rows.add(f["begin"] + token)
            heads.add(f["head"] * group + row % 128 - tok * group)
    return slots, rows, heads


def test_what_passes_stays_within_the_call(item):
    rng = random.Random(1)
    far = [-2 ** 31, -2 ** 31 + 1, -1, 0, 1, 2, 2 ** 30, 2 ** 31 - 2, 2 ** 31 - 1]
    passed = 0
    for _ in range(60000):
        ctas, kv_heads, tokens, group = rng.choice([1, 2, 3, 148]), rng.choice([1, 3, 8]), rng.choice([1, 2, 100, 5000, 2 ** 31 - 1]), rng.choice([1, 3, 8, 128])
        x = rng.randrange(ctas)
        near = dict(seq=[0], head=range(-1, kv_heads + 1), begin=[0, 1, tokens // 2, tokens - 1, tokens], n=[0, 1, 7, tokens // 2, tokens], len=[5], token0=[-1, 0, 1, 6, tokens // 3],
                    first=[0], end=[1], slot=[2 * x, 2 * x + 1, 2 * x + 1, 2 * x + 2], ctas=range(0, ctas - x + 2))
        f = {k: rng.choice(far) if rng.random() < 0.05 else min(rng.choice(list(near[k])), 2 ** 31 - 1) for k in FIELDS}
        if not item(f, x, ctas, kv_heads, tokens):
            continue
        passed += 1
        slots, rows, heads = reaches(f, x, kv_heads, group)
        assert all(0 <= s < 2 * ctas for s in slots) and all(0 <= r < tokens for r in rows) and all(0 <= h < kv_heads * group for h in heads), f
    assert passed > 500


def test_a_workspace_that_was_not_written_names_no_item(item):
    for byte in (0x00, 0x7F, 0x80, 0xFF):
        word = ctypes.c_int(int.from_bytes(bytes([byte]) * 4, "little")).value
        for x in range(148):
            assert not item(dict.fromkeys(FIELDS, word), x, 148, 8, 4096)


def test_items_that_cross_pass(item):
    # the first part of an item of each kind of call: few rows, the last pair of a long prompt, an item over all CTAs
    for f, size in ((dict(head=0, begin=0, n=3, token0=0, slot=1, ctas=148), (0, 148, 1, 3)), (dict(head=7, begin=100, n=4000, token0=3968, slot=295 - 2, ctas=2), (146, 148, 8, 4100)),
                    (dict(head=2, begin=0, n=1, token0=0, slot=21, ctas=5), (10, 148, 3, 1))):
        f.update(seq=0, len=9, first=0, end=3)
        assert item(f, *size)
        assert not item(dict(f, ctas=0), *size)  # (nothing crosses)
