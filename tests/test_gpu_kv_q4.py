"""Rotary positions, the append of rotated keys and values to the paged cache,
and attention over the 4-bit cache, against plain implementations in 64 bits.

Tolerances of the attention tests, from the arithmetic.  A score is a sum of
head_dim products held in fp32: its error is at most (head_dim + 8) 2^-24 +
2^-21 (22 bits of a float32 query's factors) times A = scale sum |q_i k_i|.  A
weight exp(s - m) is then off by twice that, relatively, and the output, a sum
of T weighted values over a sum of T weights in fp32, by (4 E + 2 (T + 64) 2^-24 + 2^-20)
sum p |v|, E the largest score error of the row.  For half-precision queries the
weights may be rounded to 11 bits, and the output is rounded to its type once."""
from __future__ import annotations

import numpy as np
import pytest

import memvanta_b200 as mv
from memvanta_b200 import _lib

pytestmark = pytest.mark.gpu

ROUND = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def tdtype(name):
    import torch
    return getattr(torch, name)


def randn(shape, seed, dtype="float32", scale=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(tdtype(dtype))


# ------------------------------------------------------- plain forms, 64 bits

def rotate64(x, cos, sin, pos, rot, layout):
    import torch
    y = x.double().clone()
    c, s = cos.double()[pos.long()][:, None], sin.double()[pos.long()][:, None]
    i = torch.arange(rot // 2, device=x.device)
    a, b = (i, i + rot // 2) if layout == mv.ROPE_HALF else (2 * i, 2 * i + 1)
    x0, x1 = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = x0 * c - x1 * s, x0 * s + x1 * c
    return y


def held32(x):
    """(nibbles, scales as bf16 values, 32-bit numpy) of the 4-bit blocks of x
    [.., hd], by the header's rule in float32 arithmetic."""
    import torch
    b = np.ascontiguousarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    most = np.take_along_axis(b, np.argmax(np.abs(b), -1)[..., None], -1)
    d = torch.from_numpy(most / np.float32(-8)).bfloat16().float().numpy()
    with np.errstate(divide="ignore"):
        inv = np.where(d == 0, np.float32(0), np.float32(1) / d)
    n = np.clip(np.floor(b * inv + np.float32(8.5)), 0, 15).astype(np.uint8)
    return n.reshape(x.shape), d[..., 0]


def layout_index(hd):
    """(byte, shift) of every dimension of a packed row."""
    d = np.arange(hd)
    word = d % 32 // 8 * (hd // 32) + d // 32
    return word * 4 + d % 8 // 2, d % 2 * 4


def values64(pages, scales):
    """Pools [..][hd/2], [..][hd/32] -> values [..][hd] in 64 bits (torch)."""
    import torch
    hd = pages.shape[-1] * 2
    byte, shift = layout_index(hd)
    n = (pages[..., torch.from_numpy(byte).to(pages.device)].int() >> torch.from_numpy(shift).to(pages.device)) & 15
    return (n.double() - 8) * scales.double().repeat_interleave(32, -1)


def random_cache(n_pages, H, page, hd, seed):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for _ in range(2):
        out.append(torch.randint(0, 256, (n_pages, H, page, hd // 2), generator=g, device="cuda", dtype=torch.uint8))
        d = 0.15 * torch.exp(torch.randn((n_pages, H, page, hd // 32), generator=g, device="cuda"))
        sign = torch.randint(0, 2, d.shape, generator=g, device="cuda") * 2 - 1
        out.append((d * sign).bfloat16())
    return out  # kp, ks, vp, vs


def scattered(need, page, seed, spare=3):
    """Block table over scattered pages; entries that no token reaches point nowhere."""
    rng = np.random.default_rng(seed)
    pages = [-(-n // page) for n in need]
    total = sum(pages) + spare
    perm = rng.permutation(total).astype(np.int32)
    t = np.full((len(need), max(max(pages), 1) + 1), -7, np.int32)
    t[:, -1] = 2 ** 31 - 1
    at = 0
    for i, p in enumerate(pages):
        t[i, :p] = perm[at:at + p]
        at += p
    return t, total


def attention64(q, kp, ks, vp, vs, table, seq, ctx, page, scale):
    """(out, bound of its fp32 error without the output's rounding) by row."""
    import torch
    rows, heads, hd = q.shape
    H = kp.shape[1]
    out = torch.zeros((rows, heads, hd), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    weights = 0.0 if q.dtype == torch.float32 else 2.0 ** -10
    for r in range(rows):
        T = int(ctx[r])
        if T <= 0:
            continue
        pg = torch.from_numpy(table[seq[r], :-(-T // page)].astype(np.int64)).to(q.device)
        k = values64(kp[pg], ks[pg]).permute(1, 0, 2, 3).reshape(H, -1, hd)[:, :T]
        v = values64(vp[pg], vs[pg]).permute(1, 0, 2, 3).reshape(H, -1, hd)[:, :T]
        k, v = (x.repeat_interleave(heads // H, 0) for x in (k, v))
        qr = q[r].double()[:, None]
        p = torch.softmax((qr * k).sum(-1) * scale, -1)
        A = ((qr * k).abs().sum(-1) * scale).amax(-1)
        E = ((hd + 8) * 2.0 ** -24 + 2.0 ** -21) * A
        out[r] = (p[..., None] * v).sum(1)
        bound[r] = ((4 * E + 2 * (T + 64) * 2.0 ** -24 + 2.0 ** -20 + weights)[:, None] * (p[..., None] * v.abs()).sum(1))
    return out, bound


def check_attention(got, want, bound):
    import torch
    name = str(got.dtype).split(".")[-1]
    tol = bound + want.abs() * ROUND[name] + 1e-30
    if name == "float16":
        tol = tol + 2.0 ** -25  # subnormal outputs
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert bool((off <= tol).all()), float((off / tol).max())


# ------------------------------------------------------------------- rotary

@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("hd,rot", [(128, 128), (128, 32), (64, 64), (256, 64), (80, 40), (6, 2), (128, 90)])
def test_rope_apply(cuda, dtype, hd, rot, layout):
    import torch
    rows, heads, n_pos = 5, 3, 5000
    cos, sin = mv.rope_table(rot, n_pos)
    pos = torch.tensor([0, 1, 4999, 1234, 77], dtype=torch.int32, device=cuda)
    x = randn((rows, heads, hd), 1, dtype)
    got = mv.rope_apply(x, cos, sin, pos, layout=layout)
    want = rotate64(x, cos, sin, pos, rot, layout)
    # two products and a sum in fp32, then one rounding to the type
    size = rotate64(x.abs(), cos.abs(), -sin.abs(), pos, rot, layout).abs() + x.double().abs()
    assert bool(((got.double() - want).abs() <= 3 * 2.0 ** -24 * size + ROUND[dtype] * want.abs() + 2.0 ** -25).all())
    assert torch.equal(got[..., rot:], x[..., rot:])
    # other strides, and in place: the same bits
    wide = torch.full((rows, heads + 2, hd + 3), 7.0, dtype=x.dtype, device=cuda)
    view = wide[:, 1:1 + heads, 1:1 + hd]
    view.copy_(x)
    mv.rope_apply(view, cos, sin, pos, layout=layout, out=view)
    assert torch.equal(view, got)
    assert bool((wide[:, 0] == 7).all() and (wide[:, -1] == 7).all() and (wide[..., 0] == 7).all()
                and (wide[..., hd + 1:] == 7).all())
    by_head = x.transpose(0, 1).contiguous().transpose(0, 1)  # [heads][rows][hd] in memory
    assert torch.equal(mv.rope_apply(by_head, cos, sin, pos, layout=layout), got)


def test_rope_apply_gives_mv_ropes_bits(cuda):
    import torch
    rows, heads, hd = 7, 32, 128
    cos, sin = mv.rope_table(hd, 300)
    pos = torch.randint(0, 300, (rows,), device=cuda, dtype=torch.int32)
    x = randn((rows, heads, hd), 2)
    want, k = x.reshape(rows, -1).clone(), randn((rows, 8 * hd), 3)
    mv.rope(want, heads, k, 8, hd, cos, sin, pos)
    assert torch.equal(mv.rope_apply(x, cos, sin, pos).reshape(rows, -1), want)


def test_rope_rows_outside_the_table_are_zero(cuda):
    import torch
    cos, sin = mv.rope_table(64, 10)
    pos = torch.tensor([-1, 9, 10, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32, device=cuda)
    y = mv.rope_apply(randn((5, 2, 64), 4), cos, sin, pos)
    assert not y[[0, 2, 3, 4]].any() and y[1].all()


@pytest.mark.parametrize("kind", ["none", "linear", "yarn", "bands", "factors"])
def test_rope_table(cuda, kind):
    import torch
    rot, n_pos, theta, factor, orig = 96, 20000, 500000.0, 8.0, 4096.0
    i = np.arange(rot // 2, dtype=np.float64)
    inv = theta ** (-2 * i / rot)
    mul, kw = 1.0, {}
    if kind == "linear":
        inv, kw = inv / factor, dict(scaling=mv.ROPE_SCALE_LINEAR, factor=factor)
    elif kind == "yarn":
        dim = lambda b: rot * np.log(orig / (b * 2 * np.pi)) / (2 * np.log(theta))  # noqa: E731
        lo, hi = max(np.floor(dim(32.0)), 0), min(np.ceil(dim(1.0)), rot - 1)
        ramp = np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
        inv, mul = inv / factor * ramp + inv * (1 - ramp), 0.1 * np.log(factor) + 1
        kw = dict(scaling=mv.ROPE_SCALE_YARN, factor=factor, orig_ctx=orig)
    elif kind == "bands":
        turns = orig * inv / (2 * np.pi)
        keep = np.clip((turns - 1) / (4 - 1), 0, 1)
        inv = inv / factor * (1 - keep) + inv * keep
        kw = dict(scaling=mv.ROPE_SCALE_BANDS, factor=factor, orig_ctx=orig, beta_fast=4.0, beta_slow=1.0)
    elif kind == "factors":
        f = np.linspace(1, 40, rot // 2).astype(np.float32)
        inv, kw = inv / f, dict(freq_factors=torch.from_numpy(f).to(cuda))
    cos, sin = mv.rope_table(rot, n_pos, theta, **kw)
    a = np.arange(n_pos)[:, None] * inv
    # half an ulp of the fp32 result, and a double angle's own error (2^-50 of 20000)
    for got, want in ((cos, np.cos(a) * mul), (sin, np.sin(a) * mul)):
        off = np.abs(got.cpu().numpy().astype(np.float64) - want)
        assert np.all(off <= np.abs(want) * 2.0 ** -24 * 1.0001 + 1e-10)


# ------------------------------------------------------------------- append

def append_setup(rows, H, hd, page, seed, need=(300, 41, 9)):
    import torch
    rng = np.random.default_rng(seed)
    t, total = scattered(need, page, seed)
    seq = rng.integers(0, len(need), rows).astype(np.int32)
    # distinct slots
    pos = np.zeros(rows, np.int32)
    for s in range(len(need)):
        at = np.flatnonzero(seq == s)[:need[s]]
        seq[np.flatnonzero(seq == s)[need[s]:]] = 0
        pos[at] = rng.permutation(need[s])[:len(at)]
    pairs, keep = set(), []
    for r in range(rows):
        keep.append((seq[r], pos[r]) not in pairs)
        pairs.add((seq[r], pos[r]))
    keep = np.array(keep)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    return t, total, seq[keep], pos[keep], dev


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("H,hd,rot,page,layout", [(8, 128, 128, 16, 0), (1, 64, 64, 1, 1), (3, 64, 16, 13, 0),
                                                  (2, 256, 128, 128, 1), (5, 96, 10, 7, 0), (1, 32, 0, 4, 0)])
def test_append_q4(cuda, dtype, H, hd, rot, page, layout):
    """Stored nibbles and scales, word for word, and the values read back."""
    import torch
    t, total, seq, pos, dev = append_setup(60, H, hd, page, 5)
    rows = len(seq)
    cos, sin = mv.rope_table(rot, 300) if rot else (None, None)
    qkv = randn((rows, 4 * H + 2 * H, hd), 6, dtype)  # one projection's row: strided heads
    q, k, v = qkv[:, :4 * H], qkv[:, 4 * H:5 * H], qkv[:, 5 * H:]
    pools = mv.kv_pools(mv.KV_Q4_0, total, page, H, hd)
    for p in pools:
        p.view(torch.uint8).fill_(0xA5)
    q_out = mv.rope_kv_append(mv.KV_Q4_0, q, k, v, cos, sin, dev(pos), dev(t), page, *pools, seq=dev(seq),
                              layout=layout)
    if rot:
        assert torch.equal(q_out, mv.rope_apply(q, cos, sin, dev(pos), layout=layout))
        k32 = mv.rope_apply(k.float(), cos, sin, dev(pos), layout=layout)  # fp32: what the quantiser sees
    else:
        assert torch.equal(q_out, q)
        k32 = k.float()
    byte, shift = layout_index(hd)
    touched = np.zeros((total, page), bool)
    for x, pages, scales in ((k32, pools[0], pools[2]), (v.float(), pools[1], pools[3])):
        n, d = held32(x.cpu().numpy())
        pages_h, scales_h = pages.cpu().numpy(), scales.float().cpu().numpy()
        for r in range(rows):
            pg, slot = t[seq[r], pos[r] // page], pos[r] % page
            touched[pg, slot] = True
            assert np.array_equal((pages_h[pg, :, slot][:, byte] >> shift) & 15, n[r])
            assert np.array_equal(scales_h[pg, :, slot], d[r])
        # nothing else was written
        assert (pages_h.transpose(0, 2, 1, 3)[~touched] == 0xA5).all()
        read = mv.kv_read(mv.KV_Q4_0, pages, scales, dev(pos), dev(t), page, H, hd, seq=dev(seq))
        assert np.array_equal(read.cpu().numpy(), (n.astype(np.float32) - 8) * np.repeat(d, 32, -1))


@pytest.mark.parametrize("kv_type", [0, 1, 2, 3])
@pytest.mark.parametrize("rot", [0, 64])
def test_append_other_types_give_mv_kv_appends_bits(cuda, kv_type, rot):
    import torch
    H, hd, page = 4, 64, 13
    t, total, seq, pos, dev = append_setup(50, H, hd, page, 7)
    rows = len(seq)
    k, v = randn((rows, H, hd), 8), randn((rows, H, hd), 9)
    cos, sin = mv.rope_table(hd, 300) if rot else (None, None)
    got, want = (mv.kv_pools(kv_type, total, page, H, hd) for _ in range(2))
    none = mv.rope_kv_append(kv_type, None, k, v, cos, sin, dev(pos), dev(t), page, *got, seq=dev(seq))
    assert none is None
    k2, dummy = k.reshape(rows, -1).clone(), randn((rows, hd), 1)
    if rot:
        mv.rope(dummy, 1, k2, H, hd, cos, sin, dev(pos))
    mv.kv_append(kv_type, k2, v.reshape(rows, -1), dev(pos), dev(t), t.shape[1], page, want[0], want[1], want[2],
                 want[3], seq=dev(seq))
    for g, w, x in zip(got, want, (k2, v, None, None)):
        if kv_type == mv.KV_F16 and x is not None:
            # rounded to nearest even; mv_kv_append's conversion loses a carry
            # into an odd exponent (1.9999 -> 1), as the reference's does
            at = [torch.from_numpy(t[seq, pos // page]).long(), torch.from_numpy(pos % page).long()]
            assert torch.equal(g[at[0].cuda(), at[1].cuda()], x.view(rows, H, hd).half())
        else:
            assert g is None and w is None or torch.equal(g, w)
    # read back: the stored values
    sc = {0: None, 1: None}.get(kv_type, got[2])
    read = mv.kv_read(kv_type, got[0], sc, dev(pos), dev(t), page, H, hd, seq=dev(seq))
    step = {0: 0.0, 1: 2.0 ** -11, 2: 1 / 254.0, 3: 1 / 254.0}[kv_type]
    top = k2.view(rows, H * hd).abs().amax(-1).view(rows, 1, 1) if kv_type >= 2 else k2.view(rows, H, hd).abs()
    assert bool(((read - k2.view(rows, H, hd)).abs() <= top * step * 1.001 + 1e-7).all())


def test_append_skips_and_special_blocks(cuda):
    import torch
    H, hd, page = 2, 64, 8
    table = torch.tensor([[1, 0, 9], [2, -1, 3]], dtype=torch.int32, device=cuda)
    seq = torch.tensor([0, 0, 0, 1, 1, 2, -1, 0, 1], dtype=torch.int32, device=cuda)
    pos = torch.tensor([0, -1, 16, 8, 3, 0, 0, 24, 2 ** 31 - 1], dtype=torch.int32, device=cuda)
    pools = mv.kv_pools(mv.KV_Q4_0, 4, page, H, hd)
    k, v = randn((9, H, hd), 10), randn((9, H, hd), 11)
    k[0, 0, 3], k[0, 1, 40] = float("nan"), float("inf")
    v[0, 0] = 0.0
    v[0, 1, :32] = 1e-38
    v[0, 1, 32:] = torch.tensor([2.5, -2.5] * 16)  # equal magnitudes: the first one's sign
    mv.rope_kv_append(mv.KV_Q4_0, None, k, v, None, None, pos, table, page, *pools, seq=seq)
    stored = [(1, 0), (2, 3)]  # rows 0 and 4; page 9 and -1, sequences 2 and -1, far positions: skipped
    for p in pools:
        u = p.view(torch.uint8).reshape(4, H, page, -1).clone()
        for pg, slot in stored:
            u[pg, :, slot] = 0
        assert not u.any()
    got = [mv.kv_read(mv.KV_Q4_0, p, s, pos, table, page, H, hd, seq=seq) for p, s in
           ((pools[0], pools[2]), (pools[1], pools[3]))]
    assert got[0][0, 0, :32].isnan().all() and not got[0][0, 0, 32:].isnan().any()
    assert got[0][0, 1, 32:].isnan().all() and not got[0][0, 1, :32].isnan().any()
    assert not got[1][0, 0].any() and not got[1][0, 1, :32].any()
    assert torch.equal(got[1][0, 1, 32:], torch.tensor([2.5, -2.1875] * 16, device=cuda))
    skipped = [1, 2, 3, 5, 6, 7, 8]
    assert not got[0][skipped].any() and not got[1][skipped].any()
    assert torch.equal(got[1][4].cpu(), torch.from_numpy(
        (held32(v[4].cpu().numpy())[0].astype(np.float32) - 8) * np.repeat(held32(v[4].cpu().numpy())[1], 32, -1)))


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,H,hd,page", [(8, 8, 128, 16), (32, 8, 128, 13), (8, 1, 64, 1), (14, 2, 256, 100),
                                             (3, 1, 64, 64), (40, 2, 128, 128), (16, 1, 128, 32)])
def test_decode(cuda, heads, H, hd, page, dtype):
    import torch
    ctx = [1, 0, 2, 15, 16, 17, 63, 64, 65, 333, 1025, 7]
    t, total = scattered(ctx, page, 20)
    kp, ks, vp, vs = random_cache(total, H, page, hd, 21)
    q = randn((len(ctx), heads, hd), 22, dtype, 1.5)
    got = mv.paged_attn_q4(q, kp, vp, ks, vs, torch.from_numpy(t).cuda(),
                           torch.tensor(ctx, dtype=torch.int32, device=cuda), 1025)
    want, bound = attention64(q, kp, ks, vp, vs, t, list(range(len(ctx))), ctx, page, hd ** -0.5)
    check_attention(got, want, bound)
    assert not got[1].any()


@pytest.mark.parametrize("n_seq,heads,H,hd,ctx", [(1, 8, 8, 128, 9000), (1, 8, 1, 64, 30011), (2, 16, 2, 256, 5000),
                                                  (70, 4, 4, 64, 700)])
def test_decode_long(cuda, n_seq, heads, H, hd, ctx):
    """Long contexts, whose work is split over many CTAs, twice: equal bits."""
    import torch
    page = 64
    lens = [ctx] + [ctx * (i * 7 % 10) // 10 for i in range(1, n_seq)]
    t, total = scattered(lens, page, 23)
    kp, ks, vp, vs = random_cache(total, H, page, hd, 24)
    q = randn((n_seq, heads, hd), 25, "float32", 1.2)
    args = (q, kp, vp, ks, vs, torch.from_numpy(t).cuda(), torch.tensor(lens, dtype=torch.int32, device=cuda), ctx)
    got = mv.paged_attn_q4(*args)
    want, bound = attention64(q, kp, ks, vp, vs, t, list(range(n_seq)), lens, page, hd ** -0.5)
    check_attention(got, want, bound)
    assert torch.equal(got, mv.paged_attn_q4(*args))


@pytest.mark.parametrize("n_seq,heads,H,hd,longest,dtype", [
    (1, 2, 1, 128, 1, "float32"), (2, 8, 4, 128, 130, "float16"), (5, 24, 8, 128, 1200, "bfloat16"),
    (27, 9, 3, 64, 700, "float32"), (55, 4, 4, 256, 90, "float16"), (110, 4, 1, 128, 300, "float32"),
    (100, 4, 4, 128, 60, "bfloat16"), (150, 3, 3, 64, 260, "float32"), (1, 20, 1, 256, 4000, "bfloat16")])
def test_decode_few_and_many_units(cuda, n_seq, heads, H, hd, longest, dtype):
    """From one (sequence, kv head) to more than the GPU holds at once: contexts
    of no token (and fewer), of one, and up to the longest in between."""
    import torch
    rng = np.random.default_rng(n_seq)
    ctx = rng.integers(1, longest + 1, n_seq).astype(np.int32)
    ctx[0] = longest
    if n_seq > 1:
        ctx[n_seq // 2], ctx[-1] = 0, 1
    if n_seq > 4:
        ctx[3] = -5
    page = 13
    t, total = scattered(np.maximum(ctx, 0), page, 80)
    kp, ks, vp, vs = random_cache(total, H, page, hd, 81)
    q = randn((n_seq, heads, hd), 82, dtype, 1.5)
    args = (q, kp, vp, ks, vs, torch.from_numpy(t).cuda(), torch.from_numpy(ctx).cuda(), longest)
    got = mv.paged_attn_q4(*args)
    want, bound = attention64(q, kp, ks, vp, vs, t, range(n_seq), ctx, page, hd ** -0.5)
    check_attention(got, want, bound)
    assert not got[torch.from_numpy(ctx <= 0).cuda()].any()
    assert torch.equal(got, mv.paged_attn_q4(*args))


def test_decode_long_sums_are_rounded(cuda):
    """The tensor cores cut their running sums; 120,000 tokens are 70 MMAs to a
    warp.  Rounded totals every 32: half of 32 cuts of at most 2^-24 of the sum on
    average, 9.5e-7, two factors of 22 bits, 2.4e-7, and the exponentials' 2^-22."""
    import torch
    H, hd, page, T = 8, 128, 128, 120_000
    t, total = scattered([T], page, 83)
    kp, ks, vp, vs = random_cache(total, H, page, hd, 84)
    q = randn((1, H, hd), 85, "float32", 0.6)
    got = mv.paged_attn_q4(q, kp, vp, ks, vs, torch.from_numpy(t).cuda(),
                           torch.tensor([T], dtype=torch.int32, device=cuda), T).double()
    pg = torch.from_numpy(t[0, :-(-T // page)].astype(np.int64)).cuda()
    off = size = 0.0
    for h in range(H):
        k = values64(kp[pg, h], ks[pg, h]).reshape(-1, hd)[:T]
        v = values64(vp[pg, h], vs[pg, h]).reshape(-1, hd)[:T]
        want = torch.softmax(k @ q[0, h].double() * hd ** -0.5, 0) @ v
        off += float(((got[0, h] - want) ** 2).sum())
        size += float((want ** 2).sum())
    assert (off / size) ** 0.5 <= 1.5e-6


def test_decode_garbage_past_the_context(cuda):
    """NaN scales, wild pages and stale nibbles past ctx_len change nothing; a
    page that does not exist is left out; max_ctx cuts."""
    import torch
    heads, H, hd, page, n = 8, 2, 128, 16, 4
    t, total = scattered([100] * n, page, 26)
    kp, ks, vp, vs = random_cache(total, H, page, hd, 27)
    q = randn((n, heads, hd), 28, "float32", 2.0)
    ctx = torch.tensor([37, 1, 96, 100], dtype=torch.int32, device=cuda)
    want = mv.paged_attn_q4(q, kp, vp, ks, vs, torch.from_numpy(t).cuda(), ctx, 100)
    ks2, vs2, t2 = ks.clone(), vs.clone(), t.copy()
    for r, c in enumerate(ctx.tolist()):
        for i in range(100 // page + 1):
            first = max(0, min(page, c - i * page))
            for s in (ks2, vs2):
                s[t[r, i], :, first:] = float("nan") if r % 2 else float("inf")
    t2[0, 3:] = -1
    t2[1, 1:] = total
    got = mv.paged_attn_q4(q, kp, vp, ks2, vs2, torch.from_numpy(t2).cuda(), ctx, 100)
    assert torch.equal(got, want)
    # a hole in the middle, and a cut at max_ctx
    t3 = t.copy()
    t3[2, 1] = -1
    got = mv.paged_attn_q4(q, kp, vp, ks, vs, torch.from_numpy(t3).cuda(), ctx, 96)
    keep = np.r_[0:16, 32:96]
    k = values64(kp[t[2, :6].tolist()], ks[t[2, :6].tolist()]).permute(1, 0, 2, 3).reshape(H, 96, hd)[:, keep]
    v = values64(vp[t[2, :6].tolist()], vs[t[2, :6].tolist()]).permute(1, 0, 2, 3).reshape(H, 96, hd)[:, keep]
    p = torch.softmax((q[2].double().view(H, 4, 1, hd) * k[:, None]).sum(-1) * hd ** -0.5, -1)
    assert float((got[2].double().view(H, 4, hd) - (p[..., None] * v[:, None]).sum(2)).abs().max()) < 1e-5
    w2, b2 = attention64(q[3:], kp, ks, vp, vs, t, [3], [96], page, hd ** -0.5)
    check_attention(got[3:], w2, b2)


def test_decode_scales_of_any_size(cuda):
    """Value and key scales from 2^-60 to 2^60: relative accuracy is kept."""
    import torch
    heads, H, hd, page, ctx = 4, 2, 64, 16, 200
    t, total = scattered([ctx], page, 29)
    kp, ks, vp, vs = random_cache(total, H, page, hd, 30)
    q = randn((1, heads, hd), 31)
    for e in (-60, -20, 20, 60):
        vs2 = (vs.double() * 2.0 ** e).bfloat16()
        ks2, q2 = (ks.double() * 2.0 ** -e).bfloat16(), q * 2.0 ** e
        got = mv.paged_attn_q4(q2, kp, vp, ks2, vs2, torch.from_numpy(t).cuda(),
                               torch.tensor([ctx], dtype=torch.int32, device=cuda), ctx)
        want, bound = attention64(q2, kp, ks2, vp, vs2, t, [0], [ctx], page, hd ** -0.5)
        check_attention(got, want, bound)
    # scales that grow along the context by 2^40
    grow = torch.from_numpy(2.0 ** np.linspace(-20, 20, total * page)).cuda().view(total, 1, page, 1)
    order = torch.argsort(torch.from_numpy(t[0, :-(-ctx // page)]).cuda())
    vs2 = (vs.double() * grow).bfloat16()
    got = mv.paged_attn_q4(q, kp, vp, ks, vs2, torch.from_numpy(t).cuda(),
                           torch.tensor([ctx], dtype=torch.int32, device=cuda), ctx)
    want, bound = attention64(q, kp, ks, vp, vs2, t, [0], [ctx], page, hd ** -0.5)
    check_attention(got, want, bound)
    assert order.numel()


def test_decode_nan_and_infinite_scores_propagate(cuda):
    import torch
    heads, H, hd, page = 2, 2, 64, 16
    t, total = scattered([40], page, 32)
    kp, ks, vp, vs = random_cache(total, H, page, hd, 33)
    ks[t[0, 1], 0, 3] = float("nan")
    vs[t[0, 2], 1, 5, 1] = float("nan")
    got = mv.paged_attn_q4(randn((1, heads, hd), 34), kp, vp, ks, vs, torch.from_numpy(t).cuda(),
                           torch.tensor([40], dtype=torch.int32, device=cuda), 40)
    assert got[0, 0].isnan().all()
    assert got[0, 1, 32:].isnan().all() and torch.isfinite(got[0, 1, :32]).all()


def test_attention_strides_scale_and_stream(cuda):
    import torch
    heads, H, hd, page, n = 8, 4, 64, 16, 6
    ctx = [50, 3, 99, 0, 17, 64]
    t, total = scattered(ctx, page, 35)
    kp, ks, vp, vs = random_cache(total, H, page, hd, 36)
    wide = randn((n, heads + 2 * H, hd), 37)
    q = wide[:, :heads]
    ctx_t, table = torch.tensor(ctx, dtype=torch.int32, device=cuda), torch.from_numpy(t).cuda()
    out = torch.full((n, heads + 1, hd), 5.0, device=cuda)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = mv.paged_attn_q4(q, kp, vp, ks, vs, table, ctx_t, 99, scale=0.3, out=out[:, :heads], stream=side)
    side.synchronize()
    want, bound = attention64(q, kp, ks, vp, vs, t, list(range(n)), ctx, page, 0.3)
    check_attention(got, want, bound)
    assert bool((out[:, heads] == 5).all())
    # captured in a graph and replayed on other inputs
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            mv.paged_attn_q4(q, kp, vp, ks, vs, table, ctx_t, 99, scale=0.3, out=out[:, :heads], stream=side)
        wide.mul_(-0.5)
        g.replay()
    side.synchronize()
    want, bound = attention64(q, kp, ks, vp, vs, t, list(range(n)), ctx, page, 0.3)
    check_attention(out[:, :heads], want, bound)


def test_offsets_past_32_bits(cuda):
    """Pools of 4.5 GB: the pages used lie past 2^32 bytes."""
    import torch
    heads, H, hd, page, ctx = 4, 1, 256, 64, 100
    n_pages = (9 << 29) // (H * page * hd // 2)
    kp, vp = (torch.empty((n_pages, H, page, hd // 2), dtype=torch.uint8, device=cuda) for _ in range(2))
    ks, vs = (torch.empty((n_pages, H, page, hd // 32), dtype=torch.bfloat16, device=cuda) for _ in range(2))
    t = np.array([[n_pages - 1, n_pages - 3]], np.int32)
    table = torch.from_numpy(t).cuda()
    k, v = randn((ctx, H, hd), 38), randn((ctx, H, hd), 39)
    pos = torch.arange(ctx, dtype=torch.int32, device=cuda)
    mv.rope_kv_append(mv.KV_Q4_0, None, k, v, None, None, pos, table, page, kp, vp, ks, vs)
    q = randn((1, heads, hd), 40)
    got = mv.paged_attn_q4(q, kp, vp, ks, vs, table, torch.tensor([ctx], dtype=torch.int32, device=cuda), ctx)
    idx = [int(x) for x in t[0]]
    want, bound = attention64(q, kp[idx], ks[idx], vp[idx], vs[idx], np.array([[0, 1]]), [0], [ctx], page, hd ** -0.5)
    check_attention(got, want, bound)
    again = mv.paged_attn_q4_prefill(q, kp, vp, ks, vs, table, torch.tensor([0, 1], dtype=torch.int32, device=cuda), 1,
                                     torch.tensor([ctx], dtype=torch.int32, device=cuda), ctx)
    check_attention(again, want, bound)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,H,hd,page", [(4, 4, 128, 16), (8, 2, 128, 13), (7, 1, 64, 128), (4, 2, 256, 32),
                                             (20, 1, 64, 1)])
def test_prefill(cuda, heads, H, hd, page, dtype):
    """Chunks of several sequences: causal rows, one of a single row, one of none."""
    import torch
    chunks = [(70, 0), (1, 200), (0, 0), (33, 129), (130, 1)]
    starts = np.concatenate([[0], np.cumsum([n for n, _ in chunks])]).astype(np.int32)
    ctx = np.concatenate([np.arange(p + 1, p + n + 1) for n, p in chunks]).astype(np.int32)
    seq = np.concatenate([[i] * n for i, (n, _) in enumerate(chunks)]).astype(int)
    t, total = scattered([n + p for n, p in chunks], page, 41)
    kp, ks, vp, vs = random_cache(total, H, page, hd, 42)
    q = randn((len(ctx), heads, hd), 43, dtype, 1.3)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    got = mv.paged_attn_q4_prefill(q, kp, vp, ks, vs, dev(t), dev(starts), 130, dev(ctx), int(ctx.max()))
    want, bound = attention64(q, kp, ks, vp, vs, t, seq, ctx, page, hd ** -0.5)
    check_attention(got, want, bound)


def test_prefill_rows_of_any_length(cuda):
    """ctx_len need not be causal: rows with none, one, and all tokens in turn."""
    import torch
    heads, H, hd, page, T = 4, 2, 128, 16, 300
    ctx = np.array([0, T, 1, 0, 128, 129, 127, T - 1] * 9, np.int32)
    t, total = scattered([T], page, 44)
    kp, ks, vp, vs = random_cache(total, H, page, hd, 45)
    q = randn((len(ctx), heads, hd), 46)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    got = mv.paged_attn_q4_prefill(q, kp, vp, ks, vs, dev(t), dev(np.array([0, len(ctx)], np.int32)), len(ctx),
                                   dev(ctx), T)
    want, bound = attention64(q, kp, ks, vp, vs, t, [0] * len(ctx), ctx, page, hd ** -0.5)
    check_attention(got, want, bound)
    assert not got[torch.from_numpy(ctx == 0).cuda()].any()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,H,hd,page,chunks", [
    (8, 8, 64, 16, [(40, 100), (1, 3), (0, 0), (29, 0), (300, 7)]),
    (12, 4, 128, 13, [(200, 0), (30, 500), (127, 1)]),
    (10, 5, 128, 64, [(129, 130)]),
    (7, 7, 256, 1, [(90, 60), (64, 0)]),
    (12, 6, 256, 128, [(260, 1)]),
    (130, 1, 64, 32, [(70, 70)]),
    (33, 3, 64, 7, [(200, 1)])])
def test_prefill_of_many_rows(cuda, heads, H, hd, page, chunks, dtype):
    """Chunks large enough for the tensor-core kernel in every type and head_dim,
    with groups that leave tile rows over and that take more than one tile."""
    import torch
    starts = np.concatenate([[0], np.cumsum([n for n, _ in chunks])]).astype(np.int32)
    ctx = np.concatenate([np.arange(p + 1, p + n + 1) for n, p in chunks]).astype(np.int32)
    seq = np.concatenate([[i] * n for i, (n, _) in enumerate(chunks)]).astype(int)
    t, total = scattered([n + p for n, p in chunks], page, 61)
    kp, ks, vp, vs = random_cache(total, H, page, hd, 62)
    q = randn((len(ctx), heads, hd), 63, dtype, 1.3)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    args = (q, kp, vp, ks, vs, dev(t), dev(starts), max(n for n, _ in chunks), dev(ctx), int(ctx.max()))
    got = mv.paged_attn_q4_prefill(*args)
    want, bound = attention64(q, kp, ks, vp, vs, t, seq, ctx, page, hd ** -0.5)
    check_attention(got, want, bound)
    assert torch.equal(got, mv.paged_attn_q4_prefill(*args))


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("hd,H,heads", [(64, 8, 16), (128, 8, 8), (256, 8, 8)])
def test_prefill_of_many_rows_of_any_length(cuda, hd, H, heads, dtype):
    """No order among the rows' lengths, rows of no token among them, a table
    with pages that are missing (their tokens do not count), rows past the last
    chunk and rows before the first (zeros)."""
    import torch
    page, T, rows = 16, 300, 150
    rng = np.random.default_rng(64)
    ctx = rng.choice([0, 0, 1, 2, 63, 64, 65, 127, 128, 129, 255, T - 1, T], size=rows).astype(np.int32)
    ctx[:3] = 0, T, 1
    t, total = scattered([T], page, 65)
    kp, ks, vp, vs = random_cache(total, H, page, hd, 66)
    q = randn((rows, heads, hd), 67, dtype)
    holes = t.copy()
    holes[0, [1, 7, 8, 18]] = [-1, 2 ** 31 - 1, total, -2 ** 31]
    starts = np.array([4, rows - 5], np.int32)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    got = mv.paged_attn_q4_prefill(q, kp, vp, ks, vs, dev(holes), dev(starts), rows, dev(ctx), T)
    # the tokens of the pages that are there, as a cache of their own
    there = np.array([p for p in range(-(-T // page)) if p not in (1, 7, 8, 18)])
    inside = np.array([sum(min(page, max(0, c - page * p)) for p in there) for c in ctx])
    want, bound = attention64(q, kp, ks, vp, vs, t[:, there], [0] * rows, inside, page, hd ** -0.5)
    used = np.zeros(rows, bool)
    used[4:rows - 5] = True
    keep = torch.from_numpy(used & (inside > 0)).cuda()
    check_attention(got[keep], want[keep], bound[keep])
    assert not got[~keep].any()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_prefill_of_many_rows_with_garbage_past_the_context(cuda, dtype):
    """NaN and infinite scales in the tokens that a row does not reach leave it
    as it is, inside its tile and in the pages after; a row that reaches a value
    block of NaN has NaN in that block's dimensions."""
    import torch
    hd, H, heads, page, T, cut = 128, 8, 8, 16, 256, 150
    ctx = np.arange(T - 120 + 1, T + 1, dtype=np.int32)  # 137 .. 256
    t, total = scattered([T], page, 68)
    kp, ks, vp, vs = random_cache(total, H, page, hd, 69)
    q = randn((len(ctx), heads, hd), 70, dtype)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    args = (dev(t), dev(np.array([0, len(ctx)], np.int32)), len(ctx), dev(ctx), T)
    want, bound = attention64(q, kp, ks, vp, vs, t, [0] * len(ctx), ctx, page, hd ** -0.5)
    # token `cut` and all later ones
    for token in range(cut, T):
        pg, o = int(t[0, token // page]), token % page
        vs[pg, :, o, 1] = float("nan")
        if token > cut:
            ks[pg, :, o] = float("nan") if token % 2 else float("inf")
            vs[pg, :, o] = float("inf") if token % 3 else float("nan")
    got = mv.paged_attn_q4_prefill(q, kp, vp, ks, vs, *args)
    clean = torch.from_numpy(ctx <= cut).cuda()
    check_attention(got[clean], want[clean], bound[clean])
    one = got[torch.from_numpy(ctx == cut + 1).cuda()][0]
    assert one[:, 32:64].isnan().all()
    rest = torch.cat([one[:, :32], one[:, 64:]], -1)
    row = int(np.flatnonzero(ctx == cut + 1)[0])
    w, b = (torch.cat([x[row][:, :32], x[row][:, 64:]], -1) for x in (want, bound))
    check_attention(rest[None], w[None], b[None])
    assert got[torch.from_numpy(ctx > cut + 1).cuda()].isnan().all()


def test_large_and_small_chunks_agree(cuda):
    """The same rows as one large chunk, in small ones, and one by one."""
    import torch
    hd, H, heads, page, T = 128, 8, 32, 32, 400
    ctx = np.arange(T - 100 + 1, T + 1, dtype=np.int32)
    t, total = scattered([T], page, 71)
    kp, ks, vp, vs = random_cache(total, H, page, hd, 72)
    q = randn((100, heads, hd), 73)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    want, bound = attention64(q, kp, ks, vp, vs, t, [0] * 100, ctx, page, hd ** -0.5)
    for n in (100, 10, 1):
        got = torch.cat([mv.paged_attn_q4_prefill(q[i:i + n], kp, vp, ks, vs, dev(t),
                                                  dev(np.array([0, n], np.int32)), n, dev(ctx[i:i + n]), T)
                         for i in range(0, 100, n)])
        check_attention(got, want, bound)


# ----------------------------------------------------------------- refusals

def test_refusals(cuda):
    import torch
    H, hd, page = 2, 64, 16
    pools = mv.kv_pools(mv.KV_Q4_0, 4, page, H, hd)
    table = torch.zeros((1, 4), dtype=torch.int32, device=cuda)
    one = torch.ones(1, dtype=torch.int32, device=cuda)
    q = randn((1, 4, hd), 50)
    cos, sin = mv.rope_table(hd, 8)

    def refused(code, fn, *a, **k):
        with pytest.raises(mv.MemVantaError) as e:
            fn(*a, **k)
        assert e.value.code == code, e.value

    I, U = _lib.MV_ERR_INVALID, _lib.MV_ERR_UNSUPPORTED
    refused(U, mv.rope_apply, q.double(), cos, sin, one)
    refused(I, mv.rope_apply, q, cos, sin, one.long())
    refused(I, mv.rope_apply, q, cos, sin, one, layout=2)
    refused(I, mv.rope_apply, q[..., :32], cos, sin, one)
    refused(I, mv.rope_apply, q, cos.half(), sin, one)
    refused(I, mv.rope_table, 63, 4)
    refused(I, mv.rope_table, 64, 4, 1.0)
    refused(I, mv.rope_table, 64, 4, scaling=mv.ROPE_SCALE_YARN, factor=2.0)
    refused(I, mv.rope_table, 64, 4, scaling=9)
    refused(I, mv.rope_kv_append, mv.KV_Q4_0, None, q[:, :2], q[:, :3], None, None, one, table, page, *pools)
    refused(I, mv.rope_kv_append, mv.KV_Q4_0, None, q[:, :2], q[:, :2], None, None, one, table, page, *pools[:2])
    refused(U, mv.rope_kv_append, 5, None, q[:, :2], q[:, :2], None, None, one, table, page, *pools)
    refused(I, mv.rope_kv_append, mv.KV_Q4_0, None, q[:, :2], q[:, :2], None, None, one, table, 0, *pools)
    odd = randn((1, 2, 48), 51)
    refused(I, mv.rope_kv_append, mv.KV_Q4_0, None, odd, odd, None, None, one, table, page, *pools)
    refused(I, mv.paged_attn_q4, randn((1, 3, hd), 52), *pools[:2], *pools[2:], table, one, 4)
    refused(I, mv.paged_attn_q4, randn((2, 4, hd), 52), *pools[:2], *pools[2:], table, one, 4)
    refused(I, mv.paged_attn_q4, q, pools[0], pools[1], pools[2][:2], pools[3], table, one, 4)
    refused(I, mv.paged_attn_q4, q, *pools, table, one, 4, scale=-1.0)
    refused(I, mv.paged_attn_q4, randn((1, 4, 128), 53), *pools, table, one, 4)
    p96 = mv.kv_pools(mv.KV_Q4_0, 4, page, H, 96)
    refused(U, mv.paged_attn_q4, randn((1, 4, 96), 53), *p96, table, one, 4)
    refused(I, mv.paged_attn_q4_prefill, q, *pools, table, torch.zeros(2, dtype=torch.int32, device=cuda), 2, one, 4)
    torch.cuda.synchronize()


def test_empty_calls(cuda):
    import torch
    pools = mv.kv_pools(mv.KV_Q4_0, 4, 16, 2, 64)
    none = torch.zeros(0, dtype=torch.int32, device=cuda)
    q = torch.empty((0, 4, 64), device=cuda)
    cos, sin = mv.rope_table(64, 8)
    assert mv.rope_apply(q, cos, sin, none).shape == q.shape
    assert mv.rope_kv_append(mv.KV_Q4_0, q, q[:, :2], q[:, :2], cos, sin, none,
                             torch.zeros((1, 4), dtype=torch.int32, device=cuda), 16, *pools).shape == q.shape
    assert mv.paged_attn_q4(q, *pools, torch.zeros((0, 4), dtype=torch.int32, device=cuda), none, 4).shape == q.shape
    torch.cuda.synchronize()
