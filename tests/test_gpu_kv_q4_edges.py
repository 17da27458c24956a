"""Attention over the 4-bit cache where it can go wrong: keys that are all zero,
scores that are not numbers, queries of any size, rows beyond a chunk, sums over
long contexts.  The plain forms and the tolerances are test_gpu_kv_q4's unless a
test states its own."""
from __future__ import annotations

import numpy as np
import pytest

import memvanta_b200 as mv
from test_gpu_kv_q4 import attention64, check_attention, layout_index, randn, random_cache, scattered, tdtype, values64

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


# ------------------------------------------------- scores that are no numbers

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("route,n,heads,H,hd,ctx", [
    ("cluster", 2, 8, 2, 128, 700), ("runs, joined", 1, 16, 8, 128, 9000), ("runs, whole", 300, 8, 4, 64, 40),
    ("many runs, joined", 130, 8, 8, 128, 1500)])
def test_decode_nan_query_gives_nan(cuda, dtype, route, n, heads, H, hd, ctx):
    """A NaN in one head's query is a NaN in all of its output, and in no other
    head's, however the context is split."""
    import torch
    t, total = scattered([ctx] * n, 64, 96)
    kp, ks, vp, vs = random_cache(total, H, 64, hd, 97)
    q = randn((n, heads, hd), 98, dtype)
    args = (kp, vp, ks, vs, dev(t), i32([ctx] * n), ctx)
    clean = mv.paged_attn_q4(q, *args)
    rows = sorted({0, n // 2, n - 1})
    for r in rows:
        q[r, 1, 7] = float("nan")
    got = mv.paged_attn_q4(q, *args)
    others = torch.tensor([r for r in range(n) if r not in rows], dtype=torch.long, device=cuda)
    assert torch.isfinite(clean).all() and torch.equal(got[others], clean[others])
    heads_left = [h for h in range(heads) if h != 1]
    want, bound = attention64(q[rows], kp, ks, vp, vs, t[rows], range(len(rows)), [ctx] * len(rows), 64, hd ** -0.5)
    assert got[rows][:, 1].isnan().all()
    check_attention(got[rows][:, heads_left], want[:, heads_left], bound[:, heads_left])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,ctx", [(128, 1), (128, 33), (128, 705), (64, 65), (256, 17), (128, 8993), (64, 20481)])
def test_decode_nan_key_alone_in_its_stage(cuda, dtype, hd, ctx):
    """The last token of a context, the first of its stage, with a NaN key."""
    import torch
    heads, H, page = 4, 2, 16
    t, total = scattered([ctx], page, 99)
    kp, ks, vp, vs = random_cache(total, H, page, hd, 100)
    ks[int(t[0, (ctx - 1) // page]), 1, (ctx - 1) % page, 0] = float("nan")
    q = randn((1, heads, hd), 101, dtype)
    got = mv.paged_attn_q4(q, kp, vp, ks, vs, dev(t), i32([ctx]), ctx)
    assert got[0, 2:].isnan().all() and torch.isfinite(got[0, :2]).all()
    chunk = mv.paged_attn_q4_prefill(q, kp, vp, ks, vs, dev(t), i32([0, 1]), 1, i32([ctx]), ctx)
    assert chunk[0, 2:].isnan().all() and torch.isfinite(chunk[0, :2]).all()


# ------------------------------------------------------------- rows and routes

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,max_q", [(300, 200), (300, 100), (20, 7)])
def test_prefill_rows_past_max_q_are_zeros(cuda, dtype, rows, max_q):
    """In large chunks and in small ones."""
    import torch
    heads, H, hd, page = 8, 8, 128, 16
    chunks = [rows, 3, rows]
    starts = np.concatenate([[0], np.cumsum(chunks)]).astype(np.int32)
    ctx = np.concatenate([np.arange(1, n + 1) for n in chunks]).astype(np.int32)
    t, total = scattered(chunks, page, 102)
    kp, ks, vp, vs = random_cache(total, H, page, hd, 103)
    q = randn((len(ctx), heads, hd), 104, dtype)
    seq = np.repeat(np.arange(3), chunks)
    got = mv.paged_attn_q4_prefill(q, kp, vp, ks, vs, dev(t), dev(starts), max_q, dev(ctx), rows)
    want, bound = attention64(q, kp, ks, vp, vs, t, seq, ctx, page, hd ** -0.5)
    past = dev(np.arange(len(ctx)) - starts[seq] >= max_q)
    assert not got[past].any()
    check_attention(got[~past], want[~past], bound[~past])


def test_a_long_chunk_beside_single_rows_keeps_its_bits(cuda):
    """A chunk that is large enough for the tensor cores goes through them beside
    63 sequences of a single row too: its rows' bits are those of the chunk alone,
    where the row-by-row kernel's differ."""
    import torch
    heads, H, hd, page, rows, n = 8, 8, 128, 32, 600, 64
    need = [rows] + [50 + i for i in range(1, n)]
    t, total = scattered(need, page, 105)
    kp, ks, vp, vs = random_cache(total, H, page, hd, 106)
    q = randn((rows + n - 1, heads, hd), 107)
    ctx = np.r_[np.arange(1, rows + 1), need[1:]].astype(np.int32)
    starts = np.r_[0, rows + np.arange(n)].astype(np.int32)
    alone = mv.paged_attn_q4_prefill(q[:rows], kp, vp, ks, vs, dev(t[:1]), i32([0, rows]), rows, dev(ctx[:rows]), rows)
    got = mv.paged_attn_q4_prefill(q, kp, vp, ks, vs, dev(t), dev(starts), rows, dev(ctx), rows)
    by_row = mv.paged_attn_q4(q[:rows], kp, vp, ks, vs, dev(np.repeat(t[:1], rows, 0)), dev(ctx[:rows]), rows)
    assert not torch.equal(by_row, alone)
    assert torch.equal(got[:rows], alone)
    seq = np.r_[np.zeros(rows, int), np.arange(1, n)]
    want, bound = attention64(q, kp, ks, vp, vs, t, seq, ctx, page, hd ** -0.5)
    check_attention(got, want, bound)


# ------------------------------------------------- sums over long contexts
#
# Values of one sign, so that an output is a sum that only grows, and its error
# of one direction shows in the mean over many outputs, where the rounding of
# the outputs does not.  The tensor cores take up to 1e-7 of such a running sum
# off at every MMA: 1e-3 after 262,144 tokens, several units in the last place of
# fp16.  With a rounded total every 1,000 MMAs half of 1e-4 is left on average.

# Keys of one scale: scores of a standard deviation of about 1, so that an output
# is a sum over many tokens.

def long_cache(hd, H, T, page, seed):
    t, total = scattered([T], page, seed)
    kp, ks, vp, vs = random_cache(total, H, page, hd, seed + 1)
    return t, kp, ks.fill_(0.4), vp, vs


def one_sided(*args):
    t, kp, ks, vp, vs = long_cache(*args)
    return t, kp, ks, vp | 0x88, vs.abs()  # nibbles 8 .. 15: values of 0 to 7 scales


def mean_off(got, q, ctx, t, kp, ks, vp, vs, page):
    """Mean over the outputs of (got - want) / want, zeros for zeros apart; rows of
    one sequence."""
    import torch
    rows, heads, hd = q.shape
    H, T = kp.shape[1], int(max(ctx))
    pg = dev(t[0, :-(-T // page)].astype(np.int64))
    past = torch.arange(T, device="cuda") >= i32(list(ctx))[:, None]
    off = []
    for h in range(heads):
        g = h // (heads // H)
        k = values64(kp[pg, g], ks[pg, g]).reshape(-1, hd)[:T]
        v = values64(vp[pg, g], vs[pg, g]).reshape(-1, hd)[:T]
        s = (q[:, h].double() @ k.T * hd ** -0.5).masked_fill(past, -float("inf"))
        want = torch.softmax(s, -1) @ v
        assert not got[:, h][want == 0].any()
        off.append(((got[:, h].double() - want) / torch.where(want == 0, 1.0, want)).mean())
    return float(torch.stack(off).mean())


def far_off(got, q, ctx, t, kp, ks, vp, vs, page):
    """Relative error of the outputs, root mean square; rows of one sequence."""
    import torch
    heads, hd, H, T = q.shape[1], q.shape[2], kp.shape[1], int(max(ctx))
    pg = dev(t[0, :-(-T // page)].astype(np.int64))
    past = torch.arange(T, device="cuda") >= i32(list(ctx))[:, None]
    off = size = 0.0
    for h in range(heads):
        k, v = (values64(p[pg, h // (heads // H)], s[pg, h // (heads // H)]).reshape(-1, hd)[:T]
                for p, s in ((kp, ks), (vp, vs)))
        w = torch.softmax((q[:, h].double() @ k.T * hd ** -0.5).masked_fill(past, -float("inf")), -1) @ v
        off += float(((got[:, h].double() - w) ** 2).sum())
        size += float((w ** 2).sum())
    return (off / size) ** 0.5


@pytest.mark.parametrize("H,heads,hd,n,T", [(1, 8, 64, 3, 90_001), (4, 4, 64, 1, 700), (2, 16, 256, 2, 40_003),
                                            (8, 8, 256, 20, 3000), (8, 56, 128, 2, 30_011), (8, 32, 128, 64, 2000)])
def test_decode_fp32_loses_no_bits(cuda, H, heads, hd, n, T):
    """As test_decode_long_sums_are_rounded, and with its bound, whatever the group,
    the head size, the route and the length."""
    page = 128
    t, kp, ks, vp, vs = long_cache(hd, H, T, page, 126)
    q = randn((n, heads, hd), 128, "float32", 0.6)
    got = mv.paged_attn_q4(q, kp, vp, ks, vs, dev(np.repeat(t, n, 0)), i32([T] * n), T)
    assert far_off(got, q, [T] * n, t, kp, ks, vp, vs, page) <= 1.5e-6


@pytest.mark.parametrize("dtype,heads,hd", [("float16", 8, 128), ("float16", 8, 64), ("bfloat16", 2, 128),
                                            ("float16", 2, 256)])
def test_decode_long_half_sums_are_rounded(cuda, dtype, heads, hd):
    """As many units as the GPU holds warps, and more, so that one warp walks
    262,144 tokens: 32,768 MMAs."""
    import torch
    H, page, T, n = heads // 2, 128, 262_144, 2000 // (heads // 2)
    t, kp, ks, vp, vs = one_sided(hd, H, T, page, 108)
    q = randn((n, heads, hd), 110, dtype, 0.5)
    got = mv.paged_attn_q4(q, kp, vp, ks, vs, dev(np.repeat(t, n, 0)), i32([T] * n), T)
    some = list(range(0, n, n // 50))
    noise = 1e-5 if dtype == "float16" else 4e-5  # of the outputs' rounding, over 50 x heads x hd outputs
    assert abs(mean_off(got[some], q[some], [T] * len(some), t, kp, ks, vp, vs, page)) <= 5e-5 + noise


@pytest.mark.parametrize("dtype,heads,H,hd,rows", [("float16", 16, 8, 64, 150), ("float16", 8, 8, 128, 150),
                                                   ("float16", 8, 4, 128, 2400), ("bfloat16", 8, 8, 128, 150),
                                                   ("float16", 8, 8, 256, 150)])
def test_prefill_long_half_sums_are_rounded(cuda, dtype, heads, H, hd, rows):
    """Chunks at the end of 262,144 tokens (one and two query tiles to a CTA),
    some rows ending far before."""
    import torch
    page, T = 128, 262_144
    ctx = np.arange(T - rows + 1, T + 1, dtype=np.int32)
    ctx[::7] = 1 + np.arange(len(ctx[::7])) * 761
    t, kp, ks, vp, vs = one_sided(hd, H, T, page, 111)
    q = randn((rows, heads, hd), 113, dtype, 0.5)
    got = mv.paged_attn_q4_prefill(q, kp, vp, ks, vs, dev(t), i32([0, rows]), rows, dev(ctx), T)
    some = [r for r in range(0, rows, max(1, rows // 60)) if ctx[r] > T - rows]
    noise = 1e-5 if dtype == "float16" else 4e-5
    assert abs(mean_off(got[some], q[some], ctx[some], t, kp, ks, vp, vs, page)) <= 5e-5 + noise
    some = list(range(0, rows, 7))[:40]
    assert abs(mean_off(got[some], q[some], ctx[some], t, kp, ks, vp, vs, page)) <= 5e-5 + 2 * noise
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("route", ["decode", "prompt"])
@pytest.mark.parametrize("x0", [7.0, 7.875])
def test_half_weights_are_rounded_not_cut(cuda, route, x0):
    """64 tokens of score 0 and value 0, then one whose weight 2^x is just above, or
    just below, a power of two: outputs w v / (64 + 2^x), w of 11 bits.  Rounded, w
    is off by at most 2^-11 either way, which leaves nothing in the mean over 1,776
    rows (a hundred steps of w) and 7 values; the outputs' rounding leaves 2e-6."""
    import torch
    n, hd, page, T, heads = 1776, 64, 128, 65, 1
    kp, vp = (torch.full((1, 1, page, hd // 2), 0x88, dtype=torch.uint8, device=cuda) for _ in range(2))
    ks, vs = (torch.zeros((1, 1, page, hd // 32), dtype=torch.bfloat16, device=cuda) for _ in range(2))
    ks[0, 0, 64] = vs[0, 0, 64] = 1
    kp[0, 0, 64, 0] = 0x99  # dimensions 0 and 1: 1, the others 0
    values = 1 + torch.arange(hd, device=cuda) % 7
    byte, shift = layout_index(hd)
    vp[0, 0, 64] = 0
    vp[0, 0, 64].index_add_(0, dev(byte).long(), ((values + 8) << dev(shift)).to(torch.uint8))
    assert torch.equal(values64(vp, vs)[0, 0, 64], values.double())
    q = torch.zeros((n, heads, hd), dtype=torch.float16, device=cuda)
    q[:, 0, 0] = x0
    q[:, 0, 1] = torch.arange(n, device=cuda) * ((0.1375 if x0 == 7 else 0.09) / n)
    scale = float(np.float32(np.log(2)))
    pages = (kp, vp, ks, vs)
    if route == "decode":
        got = mv.paged_attn_q4(q, *pages, torch.zeros((n, 1), dtype=torch.int32, device=cuda), i32([T] * n), T, scale)
    else:
        got = mv.paged_attn_q4_prefill(q, *pages, torch.zeros((1, 1), dtype=torch.int32, device=cuda), i32([0, n]), n,
                                       i32([T] * n), T, scale)
    p = torch.exp(scale * (q[:, 0, 0].double() + q[:, 0, 1].double()))[:, None]
    want = p * values / (64 + p)
    off = got[:, 0].double() / want - 1
    assert float(off.abs().max()) <= 2.0 ** -11 + 2.0 ** -11 + 2e-6
    assert abs(float(off.mean())) <= 2e-5


@pytest.mark.parametrize("hd,H,heads", PROMPTS)
def test_prefill_row_of_one_token_is_its_value(cuda, hd, H, heads):
    """fp32 queries: the weight goes in as two parts of 11 bits (2^-22 of it may
    be lost), their products' sum is cut once (2^-23), and divided by the weight;
    three roundings."""
    import torch
    page, rows = 16, 150
    t, total = scattered([rows], page, 114)
    kp, ks, vp, vs = random_cache(total, H, page, hd, 115)
    ctx = np.arange(1, rows + 1, dtype=np.int32)
    ctx[::3] = 1
    q = randn((rows, heads, hd), 116)
    got = mv.paged_attn_q4_prefill(q, kp, vp, ks, vs, dev(t), i32([0, rows]), rows, dev(ctx), rows)
    want = values64(vp[int(t[0, 0]), :, 0], vs[int(t[0, 0]), :, 0]).repeat_interleave(heads // H, 0)
    assert bool(((got[::3].double() - want).abs() <= (2.0 ** -22 + 2.0 ** -23 + 3 * 2.0 ** -24) * want.abs()).all())


@pytest.mark.parametrize("hd,H,heads", PROMPTS)
def test_prefill_long_fp32_sums_are_rounded(cuda, hd, H, heads):
    """A tile's eight MMAs of first parts are cut (2^-24 of the sum each at most,
    half of that on average, over the half of the tile's sum that is there on
    average), its total is rounded; factors of 22 bits and the exponentials as
    for decode steps: 1.2e-7 + 2.4e-7 + 2.4e-7, and as much again for scores."""
    import torch
    page, T, rows = 128, 30_000, 150
    t, kp, ks, vp, vs = long_cache(hd, H, T, page, 117)
    ctx = np.arange(T - rows + 1, T + 1, dtype=np.int32)
    q = randn((rows, heads, hd), 119, "float32", 0.6)
    got = mv.paged_attn_q4_prefill(q, kp, vp, ks, vs, dev(t), i32([0, rows]), rows, dev(ctx), T)
    assert far_off(got, q, ctx, t, kp, ks, vp, vs, page) <= 1.5e-6


# ---------------------------------------------------------- queries of any size

@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("e", [116, 90, -90])
def test_queries_of_any_size(cuda, dtype, e):
    """Queries of 2^e over keys of 2^-e: scores as of 1 over 1."""
    import torch
    heads, H, hd, page, T, rows = 8, 8, 128, 16, 200, 150
    t, total = scattered([T], page, 120)
    kp, ks, vp, vs = random_cache(total, H, page, hd, 121)
    ks = (ks.double() * 2.0 ** -e).bfloat16()
    q = (randn((rows, heads, hd), 122, dtype).double() * 2.0 ** e).to(tdtype(dtype))
    ctx = np.arange(T - rows + 1, T + 1, dtype=np.int32)
    want, bound = attention64(q, kp, ks, vp, vs, t, [0] * rows, ctx, page, hd ** -0.5)
    got = mv.paged_attn_q4_prefill(q, kp, vp, ks, vs, dev(t), i32([0, rows]), rows, dev(ctx), T)
    check_attention(got, want, bound)
    got = mv.paged_attn_q4(q, kp, vp, ks, vs, dev(np.repeat(t, rows, 0)), dev(ctx), T)
    check_attention(got, want, bound)


def test_decode_value_scales_that_grow_along_the_context(cuda):
    """By 2^40 from the first token to the last, and the other way round."""
    import torch
    heads, H, hd, page, ctx = 4, 2, 64, 16, 1000
    t, total = scattered([ctx], page, 123)
    kp, ks, vp, vs = random_cache(total, H, page, hd, 124)
    q = randn((1, heads, hd), 125)
    for a, b in ((-20, 20), (20, -20)):
        grow = torch.ones((total, page), dtype=torch.float64, device=cuda)
        pages = -(-ctx // page)
        grow[dev(t[0, :pages].astype(np.int64))] = 2.0 ** torch.linspace(a, b, pages * page, dtype=torch.float64,
                                                                       device=cuda).view(pages, page)
        vs2 = (vs.double() * grow[:, None, :, None]).bfloat16()
        got = mv.paged_attn_q4(q, kp, vp, ks, vs2, dev(t), i32([ctx]), ctx)
        want, bound = attention64(q, kp, ks, vp, vs2, t, [0], [ctx], page, hd ** -0.5)
        check_attention(got, want, bound)


# ------------------------------------------------------------------ scratch

@pytest.mark.parametrize("how", ["called", "captured first"])
def test_scratch_leaves_the_default_pool_alone(cuda, how):
    """A process that never called mv.init: an attention call that takes scratch
    leaves the device's default memory pool as the process had it, and may be the
    first call of all inside a graph capture."""
    import subprocess
    import sys
    code = """
import sys
import torch
from cuda.bindings import runtime as rt
import memvanta_b200 as mv
how, attr = sys.argv[1], rt.cudaMemPoolAttr.cudaMemPoolAttrReleaseThreshold
torch.cuda.init()
err, pool = rt.cudaDeviceGetDefaultMemPool(0)
threshold = lambda: int(rt.cudaMemPoolGetAttribute(pool, attr)[1])
before = threshold()
T, H, hd = 20000, 8, 128
kp, vp, ks, vs = mv.kv_pools(mv.KV_Q4_0, -(-T // 16), 16, H, hd)
kp.random_(0, 256), vp.random_(0, 256), ks.fill_(0.1), vs.fill_(0.1)
q = torch.randn((1, H, hd), device="cuda")
args = (q, kp, vp, ks, vs, torch.arange(kp.shape[0], dtype=torch.int32, device="cuda")[None],
        torch.tensor([T], dtype=torch.int32, device="cuda"), T)
torch.cuda.synchronize()
if how == "called":
    got = mv.paged_attn_q4(*args)
else:
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = mv.paged_attn_q4(*args)
    g.replay()
torch.cuda.synchronize()
assert torch.equal(got, mv.paged_attn_q4(*args)) and got.abs().sum() > 0
assert threshold() == before, (threshold(), before)
"""
    done = subprocess.run([sys.executable, "-c", code, how], cwd=__file__.rsplit("/tests/", 1)[0], timeout=300,
                          capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-2000:]
