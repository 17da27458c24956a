"""Refusals of the rotary, append, read and 4-bit attention entry points: every
check is made on the host, before anything is launched (no GPU needed).
"""
from __future__ import annotations

import ctypes as C

import pytest

import memvanta_b200 as mv
from memvanta_b200 import _lib

BUF = (C.c_uint8 * 4096)()
AT = (C.addressof(BUF) + 15) // 16 * 16  # 16-byte aligned; never read
OK, INVALID, UNSUPPORTED = _lib.MV_OK, _lib.MV_ERR_INVALID, _lib.MV_ERR_UNSUPPORTED


def call(name, args, **change):
    assert set(change) <= set(args), change
    return getattr(mv.load(), name)(*{**args, **change}.values())


TABLE = dict(rot=64, n_pos=16, theta=1e4, kind=0, factor=1.0, orig=0.0, fast=32.0, slow=1.0, attn=0.0, factors=None,
             cos=AT, sin=AT, stream=None)
APPLY = dict(type=0, x=AT, xs=256, xh=128, out=AT, os=256, oh=128, rows=4, heads=2, hd=128, rot=64, layout=0, cos=AT,
             sin=AT, n_pos=16, pos=AT, stream=None)
APPEND = dict(kv=4, type=0, q=AT, qs=256, qh=128, qo=AT, qos=256, qoh=128, heads=2, k=AT, ks=128, kh=128, v=AT, vs=128,
              vh=128, kv_heads=1, rows=4, hd=128, rot=64, layout=0, cos=AT, sin=AT, n_pos=16, seq=None, pos=AT,
              table=AT, n_seq=1, max_pages=4, page=16, n_pages=4, kp=AT, vp=AT, ksc=AT, vsc=AT, stream=None)
READ = dict(kv=4, pages=AT, scales=AT, kv_heads=1, hd=128, rows=4, seq=None, pos=AT, table=AT, n_seq=1, max_pages=4,
            page=16, n_pages=4, type=0, out=AT, stream=None)
DECODE = dict(type=0, q=AT, qs=256, n_seq=2, heads=2, kv_heads=1, hd=128, kp=AT, vp=AT, ksc=AT, vsc=AT, table=AT,
              max_pages=4, page=16, n_pages=4, ctx=AT, max_ctx=64, scale=0.0, out=AT, os=256, stream=None)
PREFILL = dict(type=0, q=AT, qs=256, n_q=2, heads=2, kv_heads=1, hd=128, kp=AT, vp=AT, ksc=AT, vsc=AT, table=AT,
               n_seq=1, max_pages=4, page=16, n_pages=4, q_start=AT, max_q=2, ctx=AT, max_ctx=64, scale=0.0, out=AT,
               os=256, stream=None)


@pytest.mark.parametrize("name,args,change,want", [
    ("mv_rope_table", TABLE, dict(rot=63), INVALID),
    ("mv_rope_table", TABLE, dict(kind=9), INVALID),
    ("mv_rope_table", TABLE, dict(cos=None), INVALID),
    ("mv_rope_apply", APPLY, dict(type=2), UNSUPPORTED),
    ("mv_rope_apply", APPLY, dict(rot=130), INVALID),
    ("mv_rope_apply", APPLY, dict(rot=33), INVALID),
    ("mv_rope_apply", APPLY, dict(layout=2), INVALID),
    ("mv_rope_apply", APPLY, dict(cos=None), INVALID),
    ("mv_rope_apply", APPLY, dict(os=512), INVALID),  # in place with other strides
    ("mv_rope_apply", APPLY, dict(pos=None), INVALID),
    ("mv_rope_apply", APPLY, dict(rows=2 ** 31), INVALID),
    ("mv_rope_apply", APPLY, dict(rows=0, x=None, pos=None), OK),
    ("mv_rope_kv_append", APPEND, dict(kv=5), UNSUPPORTED),
    ("mv_rope_kv_append", APPEND, dict(type=8), UNSUPPORTED),
    ("mv_rope_kv_append", APPEND, dict(hd=80, rot=64), INVALID),  # whole blocks
    ("mv_rope_kv_append", APPEND, dict(ksc=None), INVALID),
    ("mv_rope_kv_append", APPEND, dict(kp=AT + 4), INVALID),
    ("mv_rope_kv_append", APPEND, dict(k=None), INVALID),
    ("mv_rope_kv_append", APPEND, dict(q=None), INVALID),
    ("mv_rope_kv_append", APPEND, dict(page=0), INVALID),
    ("mv_rope_kv_append", APPEND, dict(table=None), INVALID),
    ("mv_rope_kv_append", APPEND, dict(kv_heads=0), INVALID),
    ("mv_rope_kv_append", APPEND, dict(rows=0, k=None, table=None), OK),
    ("mv_kv_read", READ, dict(type=2), UNSUPPORTED),
    ("mv_kv_read", READ, dict(kv=-1), UNSUPPORTED),
    ("mv_kv_read", READ, dict(out=AT + 2), INVALID),
    ("mv_kv_read", READ, dict(scales=None), INVALID),
    ("mv_kv_read", READ, dict(rows=0, out=None), OK),
    ("mv_paged_attn_q4", DECODE, dict(hd=96), UNSUPPORTED),
    ("mv_paged_attn_q4", DECODE, dict(heads=3, kv_heads=2), INVALID),
    ("mv_paged_attn_q4", DECODE, dict(type=8), UNSUPPORTED),
    ("mv_paged_attn_q4", DECODE, dict(n_pages=0), INVALID),
    ("mv_paged_attn_q4", DECODE, dict(n_pages=2 ** 31, page=16), INVALID),
    ("mv_paged_attn_q4", DECODE, dict(scale=-1.0), INVALID),
    ("mv_paged_attn_q4", DECODE, dict(scale=float("nan")), INVALID),
    ("mv_paged_attn_q4", DECODE, dict(q=None), INVALID),
    ("mv_paged_attn_q4", DECODE, dict(ctx=None), INVALID),
    ("mv_paged_attn_q4", DECODE, dict(n_seq=0, q=None), OK),
    ("mv_paged_attn_q4_prefill", PREFILL, dict(hd=32), UNSUPPORTED),
    ("mv_paged_attn_q4_prefill", PREFILL, dict(q_start=None), INVALID),
    ("mv_paged_attn_q4_prefill", PREFILL, dict(ctx=None), INVALID),
    ("mv_paged_attn_q4_prefill", PREFILL, dict(vsc=AT + 8), INVALID),
    ("mv_paged_attn_q4_prefill", PREFILL, dict(n_q=0, q=None), OK)])
def test_c_entry_points_refuse(name, args, change, want):
    assert len(args) == len(_lib.SIGNATURES[name][1])
    rc = call(name, args, **change)
    assert rc == want, mv.load().mv_last_error()
    if want != OK:
        assert mv.load().mv_last_error()
