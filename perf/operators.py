"""Cases of the operators around a long-context paged KV cache: rotary positions, the append of rotated
keys and of values to the cache, and attention over the cache held in 4 bits.

``run`` computes them in elementary torch operations (``own`` false) or through memvanta_b200's entry
points (``own`` true).  A cache in 4 bits is held as its entry points define it: per page and kv head the
tokens' rows of head_dim / 2 bytes, and one bfloat16 scale for 32 dimensions.  A row's 32-bit words are
ordered [4][head_dim / 32]: word (t, b) holds dimensions 32 b + 8 t .. + 7, the lowest nibble first; nibble
n of a block of scale d stands for (n - 8) d.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
GOLDEN = 0.6180339887498949


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one decode step's queries of 64 sequences, 7B heads, the half layout: latency counts
        dict(name="rope_decode_64", op="rope", type="f32", rows=64, heads=32, hd=128, rot=128, layout="half",
             n_pos=8192),
        # a long prompt's queries with a quarter of each head rotated in interleaved pairs, an odd row count
        dict(name="rope_prompt_partial", op="rope", type="bf16", rows=8191, heads=32, hd=128, rot=32,
             layout="interleaved", n_pos=16384),
        # decode of 64 sequences into the 4-bit cache, 16-token pages, the queries rotated in the same call
        dict(name="append_q4_decode_64", op="append", kv="q4", type="f32", rows=64, heads=32, kv_heads=8, hd=128,
             rot=128, layout="half", page=16, chunk=1, start=700),
        # a 7B prompt chunk of 4093 rows into the 4-bit cache, 128-token pages
        dict(name="append_q4_prompt", op="append", kv="q4", type="f32", rows=4093, heads=32, kv_heads=32, hd=128,
             rot=128, layout="half", page=128, chunk=4093, start=1000),
        # a prompt chunk of half-precision activations into an F16 cache, half of each head rotated, interleaved
        dict(name="append_f16_prompt", op="append", kv="f16", type="f16", rows=2048, heads=32, kv_heads=8, hd=128,
             rot=64, layout="interleaved", page=64, chunk=2048, start=77),
        # one sequence's decode step with 7B heads at the bench's context: latency counts
        dict(name="decode_one_768", op="decode", type="f32", seqs=1, heads=32, kv_heads=32, hd=128, page=128,
             lo=768, hi=768),
        # one sequence at the end of a 131072-token context, grouped heads
        dict(name="decode_one_131k", op="decode", type="f32", seqs=1, heads=32, kv_heads=8, hd=128, page=128,
             lo=131071, hi=131071),
        # 64 sequences of 64..768 tokens in scattered 16-token pages, 7B heads (the paged attention benchmark)
        dict(name="decode_64_ragged", op="decode", type="f32", seqs=64, heads=32, kv_heads=32, hd=128, page=16,
             lo=64, hi=768),
        # 48 sequences of very different lengths, small heads, half-precision activations, a page size of 13
        dict(name="decode_48_hd64", op="decode", type="f16", seqs=48, heads=64, kv_heads=8, hd=64, page=13,
             lo=1, hi=16384),
        # the bench's 512-token prompt, 7B heads, float32 activations
        dict(name="prompt_512", op="prompt", type="f32", seqs=1, rows=512, heads=32, kv_heads=32, hd=128, page=128,
             past=0),
        # a 2048-row chunk of a prompt after 14336 cached tokens, grouped heads, bfloat16 activations
        dict(name="prompt_chunk_16k", op="prompt", type="bf16", seqs=1, rows=2048, heads=32, kv_heads=8, hd=128,
             page=64, past=14336),
        # chunks of 7 sequences of different lengths in one call, large heads
        dict(name="prompt_7_hd256", op="prompt", type="f16", seqs=7, rows=331, heads=16, kv_heads=4, hd=256,
             page=16, past=1500),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "decode", "decode", "prompt", "prompt"])
    t = rng.choice(["f32", "f32", "f16", "bf16"])
    hd = rng.choice([64, 128, 128, 256])
    kv_heads, group = rng.choice([(32, 1), (8, 1), (8, 4), (8, 8), (4, 4), (2, 8), (1, 16), (4, 7)])
    page = rng.choice([13, 16, 16, 32, 64, 100, 128])
    if op in ("rope", "append"):
        rot = rng.choice([hd, hd, hd // 2, hd // 4])
        layout = rng.choice(["half", "interleaved"])
        rows = _log(rng, 1, 8191 * 32 * 128 // (kv_heads * group * hd) if op == "rope" else 4093)
        if op == "rope":
            return dict(op="rope", type=t, rows=min(rows, 16384), heads=kv_heads * group, hd=hd, rot=rot,
                        layout=layout, n_pos=16384)
        rows = min(rows, 4093 * 32 * 128 // (kv_heads * max(group, 3) * hd))
        chunk = rng.choice([1, rows])
        return dict(op="append", kv=rng.choice(["q4", "q4", "f16"]), type=t, rows=rows, heads=kv_heads * group,
                    kv_heads=kv_heads, hd=hd, rot=rot, layout=layout, page=page, chunk=chunk,
                    start=rng.randint(0, 1500))
    if op == "decode":
        cells = 131071 * 8 * 128 // (kv_heads * hd)  # cached (sequence, token) pairs of the largest listed case
        seqs = _log(rng, 1, 128)
        hi = _log(rng, 1, min(131071, max(1, cells // seqs)))
        return dict(op="decode", type=t, seqs=seqs, heads=kv_heads * group, kv_heads=kv_heads, hd=hd, page=page,
                    lo=rng.choice([hi, max(1, hi // 16)]), hi=hi)
    heads = kv_heads * group
    seqs = rng.choice([1, 1, 3, 6])
    rows = _log(rng, 2, 1500 // seqs)
    past = rng.choice([0, _log(rng, 1, max(1, min(12000, 500_000_000 // (heads * hd * seqs * rows) * 16)))])
    return dict(op="prompt", type=t, seqs=seqs, rows=rows, heads=heads, kv_heads=kv_heads, hd=hd, page=page, past=past)


def lengths(case):
    """Cached tokens of each sequence: spread over lo..hi by the golden ratio, the longest first."""
    lo, hi = case["lo"], case["hi"]
    return [hi] + [lo + int((hi - lo) * ((i * GOLDEN) % 1.0) ** 2) for i in range(1, case["seqs"])]


def chunks(case):
    """(rows, past) of each sequence of a prompt case: the first has them whole, the others parts of them."""
    n, past = case["rows"], case["past"]
    return [(n, past)] + [(max(1, int(n * ((i * GOLDEN) % 1.0))), int(past * ((i * 0.37) % 1.0)))
                          for i in range(1, case["seqs"])]


# ----------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _tables(rot, n_pos):
    """cos and sin [n_pos][rot / 2], the base frequencies stretched fourfold below a wavelength ramp."""
    i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    inv = 500000.0 ** (-2.0 * i / rot)
    turns = inv * 2048 / (2 * math.pi)
    keep = ((turns - 1) / 31).clamp(0, 1)
    inv = inv * (keep + (1 - keep) / 4)
    a = torch.arange(n_pos, device="cuda", dtype=torch.float64)[:, None] * inv
    return a.cos().float(), a.sin().float()


def _cache(g, n_pages, kv_heads, page, hd):
    """One 4-bit pool and its scales: nibbles of a rounded normal distribution, scales of many sizes."""
    n = n_pages * kv_heads * page
    parts = []
    for at in range(0, n, 1 << 18):
        m = min(1 << 18, n - at)
        q = (torch.randn((2, m, hd // 2), generator=g, device="cuda") * 2.9 + 8).round().clamp(0, 15).to(torch.uint8)
        parts.append(q[0] | (q[1] << 4))
    pool = torch.cat(parts).view(n_pages, kv_heads, page, hd // 2)
    d = 0.3 * torch.exp(0.4 * torch.randn((n_pages, kv_heads, page, hd // 32), generator=g, device="cuda"))
    sign = torch.randint(0, 2, d.shape, generator=g, device="cuda") * 2 - 1
    return pool, (d * sign).to(torch.bfloat16)


def _table_of(g, need, page):
    """A block table [len(need)][pages] over scattered pages, and the number of pages."""
    pages = [(n + page - 1) // page for n in need]
    order = torch.randperm(sum(pages), generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((len(need), max(max(pages), 1)), dtype=torch.int32, device="cuda")
    at = 0
    for i, p in enumerate(pages):
        table[i, :p] = order[at:at + p]
        at += p
    return table, at


def prepare(case, seed):
    g, t = _gen(seed), TYPES[case["type"]]
    hd, heads = case["hd"], case["heads"]
    randn = lambda *s: torch.randn(s, generator=g, device="cuda").to(t)  # noqa: E731
    if case["op"] == "rope":
        cos, sin = _tables(case["rot"], case["n_pos"])
        pos = torch.randint(0, case["n_pos"], (case["rows"],), generator=g, device="cuda", dtype=torch.int32)
        x = randn(case["rows"], heads, hd)
        return dict(case=case, x=x, cos=cos, sin=sin, pos=pos, out=torch.empty_like(x))
    H, page = case["kv_heads"], case["page"]
    if case["op"] == "append":
        rows, chunk, start = case["rows"], case["chunk"], case["start"]
        n = rows // chunk
        first = [start + (i * 131) % 517 for i in range(n)]
        table, n_pages = _table_of(g, [f + chunk for f in first], page)
        seq = torch.arange(n, device="cuda", dtype=torch.int32).repeat_interleave(chunk)
        pos = (torch.tensor(first, device="cuda")[:, None] + torch.arange(chunk, device="cuda")).reshape(-1).int()
        cos, sin = _tables(case["rot"], max(first) + chunk)
        # q, k and v as a projection leaves them: one row of all heads
        qkv = randn(rows, heads + 2 * H, hd)
        s = dict(case=case, q=qkv[:, :heads], k=qkv[:, heads:heads + H], v=qkv[:, heads + H:], cos=cos, sin=sin,
                 pos=pos, seq=seq, table=table, q_out=torch.empty((rows, heads, hd), dtype=t, device="cuda"))
        if case["kv"] == "q4":
            s["kp"] = torch.zeros((n_pages, H, page, hd // 2), dtype=torch.uint8, device="cuda")
            s["ks"] = torch.zeros((n_pages, H, page, hd // 32), dtype=torch.bfloat16, device="cuda")
            s["vp"], s["vs"] = torch.zeros_like(s["kp"]), torch.zeros_like(s["ks"])
        else:
            s["kp"] = torch.zeros((n_pages, page, H, hd), dtype=torch.float16, device="cuda")
            s["vp"], s["ks"], s["vs"] = torch.zeros_like(s["kp"]), None, None
        return s
    if case["op"] == "decode":
        need = lengths(case)
        ctx = torch.tensor(need, dtype=torch.int32, device="cuda")
        rows, more = case["seqs"], dict(max_ctx=max(need))
    else:
        parts = chunks(case)
        need = [n + p for n, p in parts]
        ctx = torch.cat([torch.arange(p + 1, p + n + 1, dtype=torch.int32) for n, p in parts]).cuda()
        starts = [0]
        for n, _ in parts:
            starts.append(starts[-1] + n)
        rows = starts[-1]
        more = dict(q_start=torch.tensor(starts, dtype=torch.int32, device="cuda"), max_q=max(n for n, _ in parts),
                    max_ctx=max(need))
    table, n_pages = _table_of(g, need, page)
    kp, ks = _cache(g, n_pages, H, page, hd)
    vp, vs = _cache(g, n_pages, H, page, hd)
    q = (torch.randn((rows, heads, hd), generator=g, device="cuda") * 1.5).to(t)
    return dict(case=case, q=q, kp=kp, vp=vp, ks=ks, vs=vs, table=table, ctx=ctx, out=torch.empty_like(q), **more)


# ------------------------------------------------------------------ passes

def run(s):
    c = s["case"]
    return (_run_own if own else _run_plain)(s, c)


def _run_own(s, c):
    import memvanta_b200 as mv

    if c["op"] == "decode":
        return mv.paged_attn_q4(s["q"], s["kp"], s["vp"], s["ks"], s["vs"], s["table"], s["ctx"], s["max_ctx"],
                                out=s["out"])
    if c["op"] == "prompt":
        return mv.paged_attn_q4_prefill(s["q"], s["kp"], s["vp"], s["ks"], s["vs"], s["table"], s["q_start"],
                                        s["max_q"], s["ctx"], s["max_ctx"], out=s["out"])
    layout = mv.ROPE_HALF if c["layout"] == "half" else mv.ROPE_INTERLEAVED
    if c["op"] == "rope":
        return mv.rope_apply(s["x"], s["cos"], s["sin"], s["pos"], layout=layout, out=s["out"])
    kv = mv.KV_Q4_0 if c["kv"] == "q4" else mv.KV_F16
    q = mv.rope_kv_append(kv, s["q"], s["k"], s["v"], s["cos"], s["sin"], s["pos"], s["table"], c["page"], s["kp"],
                          s["vp"], s["ks"], s["vs"], seq=s["seq"], layout=layout, q_out=s["q_out"])
    if c["kv"] != "q4":
        return q, s["kp"], s["vp"]
    # what is held in 4 bits, as the values it stands for
    read = lambda p, d: mv.kv_read(kv, p, d, s["pos"], s["table"], c["page"], c["kv_heads"], c["hd"],  # noqa: E731
                                   seq=s["seq"], dtype=torch.float16)
    return q, read(s["kp"], s["ks"]), read(s["vp"], s["vs"])


def _rotate(x, cos, sin, pos, rot, layout):
    """x [rows, heads, hd] in 32 bits with the first rot dimensions of each head rotated."""
    co, si = cos[pos.long()][:, None], sin[pos.long()][:, None]
    r, rest = x[..., :rot], x[..., rot:]
    x0, x1 = (r[..., :rot // 2], r[..., rot // 2:]) if layout == "half" else (r[..., 0::2], r[..., 1::2])
    y0, y1 = x0 * co - x1 * si, x0 * si + x1 * co
    y = torch.cat((y0, y1), -1) if layout == "half" else torch.stack((y0, y1), -1).flatten(-2)
    return torch.cat((y, rest), -1)


def _quantise(x):
    """x [rows, heads, hd] in 32 bits -> packed bytes [.., hd / 2] and bfloat16 scales [.., hd / 32]."""
    b = x.unflatten(-1, (-1, 32))
    most = b.gather(-1, b.abs().argmax(-1, keepdim=True))
    d = (most / -8).to(torch.bfloat16)
    inv = torch.where(d == 0, 0.0, 1.0 / d.float())
    n = (b * inv + 8.5).floor().clamp(0, 15).to(torch.uint8)
    n = n.unflatten(-1, (4, 4, 2)).transpose(-4, -3)  # [.., 4 words, blocks, 4 bytes, 2 nibbles]
    return (n[..., 0] | (n[..., 1] << 4)).flatten(-3), d.squeeze(-1)


def _values(p, d):
    """Packed bytes [.., hd / 2] and scales [.., hd / 32] -> values [.., hd] in 32 bits."""
    n = torch.stack((p & 15, p >> 4), -1).unflatten(-2, (4, -1, 4)).transpose(-4, -3)
    return ((n.flatten(-3).float() - 8) * d.float()[..., None]).flatten(-2)


def _run_plain(s, c):
    f = lambda k: s[k].float()  # noqa: E731
    if c["op"] == "rope":
        s["out"].copy_(_rotate(f("x"), s["cos"], s["sin"], s["pos"], c["rot"], c["layout"]))
        return s["out"]
    page = s["case"]["page"]
    if c["op"] == "append":
        q = _rotate(f("q"), s["cos"], s["sin"], s["pos"], c["rot"], c["layout"]).to(s["q"].dtype)
        k = _rotate(f("k"), s["cos"], s["sin"], s["pos"], c["rot"], c["layout"])
        pos, seq = s["pos"].long(), s["seq"].long()
        pages, slot = s["table"][seq, pos // page].long(), pos % page
        if c["kv"] != "q4":
            s["kp"][pages, slot] = k.half()
            s["vp"][pages, slot] = f("v").half()
            return q, s["kp"], s["vp"]
        out = [q]
        (s["kp"][pages, :, slot], s["ks"][pages, :, slot]) = _quantise(k)
        (s["vp"][pages, :, slot], s["vs"][pages, :, slot]) = _quantise(f("v"))
        out.append(_values(s["kp"][pages, :, slot], s["ks"][pages, :, slot]).half())
        out.append(_values(s["vp"][pages, :, slot], s["vs"][pages, :, slot]).half())
        return tuple(out)
    H, G, hd, T = c["kv_heads"], c["heads"] // c["kv_heads"], c["hd"], s["max_ctx"]
    tok = torch.arange(T, device="cuda")
    pages, slot = s["table"][:, tok // page].long(), (tok % page).expand(s["table"].shape[0], T)
    k = _values(s["kp"][pages, :, slot], s["ks"][pages, :, slot]).permute(0, 2, 3, 1)  # [seq, H, hd, T]
    v = _values(s["vp"][pages, :, slot], s["vs"][pages, :, slot]).transpose(1, 2)      # [seq, H, T, hd]
    if c["op"] == "decode":
        q = f("q").view(-1, H, G, hd)
        ctx = s["ctx"].view(-1, 1, 1, 1)
    else:
        # rows padded to max_q for each sequence; ctx 0 in the padding
        n = s["q_start"].diff()
        at = s["q_start"][:-1, None] + torch.arange(s["max_q"], device="cuda")
        inside = torch.arange(s["max_q"], device="cuda") < n[:, None]
        at = torch.where(inside, at, 0).long()
        q = f("q")[at].view(-1, s["max_q"], H, G, hd).permute(0, 2, 3, 1, 4).flatten(2, 3)
        ctx = torch.where(inside, s["ctx"][at], 0)[:, None, None, :, None]
        ctx = ctx.expand(-1, 1, G, -1, 1).flatten(2, 3)
    p = (q * (1 / math.sqrt(hd))) @ k
    p = p.masked_fill_(tok >= ctx, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top > -math.inf, top, 0)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / torch.where(total > 0, total, 1)
    if c["op"] == "decode":
        return o.reshape(s["q"].shape).to(s["q"].dtype)
    o = o.unflatten(2, (G, -1)).permute(0, 3, 1, 2, 4).reshape(-1, s["max_q"], H * G, hd)
    return o[inside].to(s["q"].dtype)


# -------------------------------------------------------------------- work

def work(case):
    hd, heads, e = case["hd"], case["heads"], SIZE[case["type"]]
    if case["op"] == "rope":
        n = case["rows"] * heads * hd
        # x in, out written, the cos and sin rows of the positions
        return {"bytes": 2 * n * e + case["rows"] * (case["rot"] * 4 + 4),
                "flops": case["rows"] * heads * case["rot"] * 3}
    H = case["kv_heads"]
    row4 = H * (hd // 2 + hd // 32 * 2)  # one token's keys or values in 4 bits
    if case["op"] == "append":
        rows = case["rows"]
        n = rows * (2 * heads + 2 * H) * hd * e + rows * (case["rot"] * 4 + 12)
        # q4: the rows written, read back, and their values in half precision
        n += 2 * rows * (2 * row4 + H * hd * 2) if case["kv"] == "q4" else 2 * rows * H * hd * 2
        return {"bytes": n, "flops": rows * ((heads + H) * case["rot"] * 3 + 2 * H * hd * 3)}
    if case["op"] == "decode":
        cells, rows, tokens = sum(lengths(case)), case["seqs"], sum(lengths(case))
    else:
        parts = chunks(case)
        cells = sum(n * p + n * (n + 1) // 2 for n, p in parts)
        rows, tokens = sum(n for n, _ in parts), sum(n + p for n, p in parts)
    return {"bytes": 2 * tokens * row4 + 2 * rows * heads * hd * e, "flops": 4 * cells * heads * hd}


# ------------------------------------------------------------ in 64 bits

def _exact_rotate(x, cos, sin, pos, rot, layout):
    """Each pair as a complex number times cos + i sin."""
    y = x.double().clone()
    i = torch.arange(rot // 2, device="cuda")
    a, b = (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
    turn = torch.complex(cos.double(), sin.double())[pos.long()][:, None]
    z = torch.complex(y[..., a], y[..., b]) * turn
    y[..., a], y[..., b] = z.real, z.imag
    return y


def _exact_values(p, d, hd):
    """Value of each dimension from the byte and the half-byte where it lies."""
    dim = torch.arange(hd, device="cuda")
    word = (dim % 32) // 8 * (hd // 32) + dim // 32
    n = (p[..., word * 4 + dim % 8 // 2].int() >> (dim % 2 * 4)) & 15
    return (n.double() - 8) * d.double()[..., dim // 32]


def _exact_held(x):
    """x in 64 bits as the 4-bit blocks stand for it."""
    out = torch.zeros_like(x)
    for b in range(x.shape[-1] // 32):
        blk = x[..., 32 * b:32 * b + 32]
        hi, lo = blk.amax(-1, keepdim=True), blk.amin(-1, keepdim=True)
        most = torch.where(hi >= -lo, hi, lo)
        d = (most / -8).float().bfloat16().double()
        n = torch.floor(blk / torch.where(d == 0, 1.0, d) + 8.5).clamp(0, 15)
        out[..., 32 * b:32 * b + 32] = (n - 8) * d
    return out


def exact(case, seed):
    s, c = prepare(case, seed), case
    hd, heads = c["hd"], c["heads"]
    if c["op"] == "rope":
        return _exact_rotate(s["x"], s["cos"], s["sin"], s["pos"], c["rot"], c["layout"])
    page, H = c["page"], c["kv_heads"]
    G = heads // H
    if c["op"] == "append":
        q = _exact_rotate(s["q"], s["cos"], s["sin"], s["pos"], c["rot"], c["layout"])
        k = _exact_rotate(s["k"], s["cos"], s["sin"], s["pos"], c["rot"], c["layout"])
        if c["kv"] == "q4":
            return q, _exact_held(k), _exact_held(s["v"].double())
        at = s["table"].long()[s["seq"].long(), s["pos"].long() // page] * page + s["pos"].long() % page
        pools = [torch.zeros((s["kp"].shape[0] * page, H, hd), dtype=torch.float64, device="cuda") for _ in range(2)]
        pools[0][at], pools[1][at] = k, s["v"].double()
        return q, pools[0].view(s["kp"].shape), pools[1].view(s["vp"].shape)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    starts = list(range(c["seqs"] + 1)) if c["op"] == "decode" else s["q_start"].tolist()
    ctx = s["ctx"].tolist()
    for i in range(c["seqs"]):
        a, z = starts[i], starts[i + 1]
        T = max(ctx[a:z])
        pg = s["table"][i, :(T + page - 1) // page].long()
        keep = torch.arange(T, device="cuda") < s["ctx"][a:z, None]  # [rows, T]
        for h in range(H):
            k = _exact_values(s["kp"][pg, h].flatten(0, 1)[:T], s["ks"][pg, h].flatten(0, 1)[:T], hd)
            v = _exact_values(s["vp"][pg, h].flatten(0, 1)[:T], s["vs"][pg, h].flatten(0, 1)[:T], hd)
            for j in range(h * G, h * G + G):
                e = (s["q"][a:z, j].double() @ k.T) / math.sqrt(hd)
                e = torch.softmax(e.masked_fill(~keep, -math.inf), -1)
                out[a:z, j] = e @ v
    return out
