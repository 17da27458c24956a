"""Attention over the 4-bit cache where it can go wrong: keys that are all zero,
scores that are not numbers, queries of any size, rows beyond a chunk, sums over
long contexts.  The plain forms and the tolerances are test_gpu_kv_q4's unless a
test states its own."""
from __future__ import annotations

import numpy as np
import pytest

import memvanta_b200 as mv
from test_gpu_kv_q4 import attention64, check_attention, randn, random_cache, scattered

pytestmark = pytest.mark.gpu
TYPES = ["float32", "float16", "bfloat16"]
# (head_dim, kv heads, query heads) whose 150 rows go through the tensor cores
PROMPTS = [(64, 8, 16), (128, 8, 8), (256, 8, 8)]


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def i32(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------ keys of zero

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,H,heads", PROMPTS)
@pytest.mark.parametrize("which", ["all heads", "one head"])
def test_prefill_over_keys_of_zero(cuda, dtype, hd, H, heads, which):
    """Zero keys give every score 0 and the mean of the values, whatever the
    queries: rows of zeros, of 2^-9 and of 2^-120 among normal ones."""
    import torch
    page, rows, past = 16, 150, 30
    T = rows + past
    ctx = np.arange(past + 1, T + 1, dtype=np.int32)
    t, total = scattered([T], page, 90)
    kp, ks, vp, vs = random_cache(total, H, page, hd, 91)
    q = randn((rows, heads, hd), 92, dtype)
    mine = slice(None) if which == "all heads" else slice(0, heads // H)
    ks[:, slice(None) if which == "all heads" else slice(0, 1)] = 0
    q[0::4, mine] = 0
    q[1::4, mine] *= 2.0 ** -9
    q[2::4, mine] *= 2.0 ** -120 if dtype != "float16" else 2.0 ** -14
    got = mv.paged_attn_q4_prefill(q, kp, vp, ks, vs, dev(t), i32([0, rows]), rows, dev(ctx), T)
    want, bound = attention64(q, kp, ks, vp, vs, t, [0] * rows, ctx, page, hd ** -0.5)
    check_attention(got, want, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,H,heads", PROMPTS)
def test_prefill_small_queries_over_missing_tiles(cuda, dtype, hd, H, heads):
    """128 tokens one after the other on pages that do not exist are left out,
    for queries of 2^-10 and of zero too, and rows that end before them are as
    they are."""
    import torch
    page, T, rows = 16, 300, 150
    ctx = np.r_[np.arange(1, 91), np.arange(T - 59, T + 1)].astype(np.int32)
    t, total = scattered([T], page, 93)
    kp, ks, vp, vs = random_cache(total, H, page, hd, 94)
    q = randn((rows, heads, hd), 95, dtype, 2.0 ** -10)
    q[::5] = 0
    gone = range(4, 12)
    holes = t.copy()
    holes[0, list(gone)] = [-1, 2 ** 31 - 1, total, -2 ** 31] * 2
    got = mv.paged_attn_q4_prefill(q, kp, vp, ks, vs, dev(holes), i32([0, rows]), rows, dev(ctx), T)
    there = np.array([p for p in range(-(-T // page)) if p not in gone])
    inside = np.array([sum(min(page, max(0, c - page * p)) for p in there) for c in ctx])
    want, bound = attention64(q, kp, ks, vp, vs, t[:, there], [0] * rows, inside, page, hd ** -0.5)
    check_attention(got, want, bound)
