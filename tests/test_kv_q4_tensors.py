"""The rotary, append, read and 4-bit attention calls refuse tensors that are not
on the current GPU (no GPU needed: every refusal comes before anything else is done)."""
from __future__ import annotations

import pytest

import memvanta_b200 as mv
from memvanta_b200 import _lib

ROWS, HEADS, H, HD, PAGE, PAGES = 3, 4, 2, 64, 16, 5


class At:
    """A tensor as another, on GPU `device`."""

    def __init__(self, tensor, device):
        self._tensor, self._device = tensor, device

    def get_device(self):
        return self._device

    def __getattr__(self, name):
        return getattr(self._tensor, name)


def calls():
    """(call, its tensors by name, its other arguments)."""
    import torch
    f, i = (lambda *s: torch.zeros(s)), (lambda *s: torch.zeros(s, dtype=torch.int32))
    tables = dict(cos_t=f(8, HD // 2), sin_t=f(8, HD // 2))
    pages = lambda: torch.zeros((PAGES, H, PAGE, HD // 2), dtype=torch.uint8)  # noqa: E731
    scales = lambda: torch.zeros((PAGES, H, PAGE, HD // 32), dtype=torch.bfloat16)  # noqa: E731
    pools = dict(k_pages=pages(), v_pages=pages(), k_scales=scales(), v_scales=scales())
    return [
        (mv.rope_apply, dict(x=f(ROWS, HEADS, HD), **tables, pos=i(ROWS), out=f(ROWS, HEADS, HD)), {}),
        (mv.rope_kv_append, dict(q=f(ROWS, HEADS, HD), k=f(ROWS, H, HD), v=f(ROWS, H, HD), **tables, pos=i(ROWS),
                                 block_table=i(1, PAGES), **pools, seq=i(ROWS), q_out=f(ROWS, HEADS, HD)),
         dict(kv_type=mv.KV_Q4_0, page=PAGE)),
        (mv.kv_read, dict(pages=pages(), scales=scales(), pos=i(ROWS), block_table=i(1, PAGES), seq=i(ROWS),
                          out=f(ROWS, H, HD)), dict(kv_type=mv.KV_Q4_0, page=PAGE, n_head_kv=H, head_dim=HD)),
        (mv.paged_attn_q4, dict(q=f(ROWS, HEADS, HD), **pools, block_table=i(ROWS, PAGES), ctx_len=i(ROWS),
                                out=f(ROWS, HEADS, HD)), dict(max_ctx=PAGES * PAGE)),
        (mv.paged_attn_q4_prefill, dict(q=f(ROWS, HEADS, HD), **pools, block_table=i(1, PAGES), q_start=i(2),
                                        ctx_len=i(ROWS), out=f(ROWS, HEADS, HD)),
         dict(max_ctx=PAGES * PAGE, max_q=ROWS)),
    ]


def refused(call, **args):
    with pytest.raises(mv.MemVantaError, match="current GPU") as e:
        call(**args)
    assert e.value.code == _lib.MV_ERR_INVALID


@pytest.mark.parametrize("n", range(5))
def test_tensors_on_the_host_or_on_another_gpu_are_refused(n, monkeypatch):
    monkeypatch.setattr(mv, "_current_device", lambda: 0)
    call, tensors, rest = calls()[n]
    refused(call, **tensors, **rest)
    here = {k: At(t, 0) for k, t in tensors.items()}
    for name, t in tensors.items():
        refused(call, **{**here, name: At(t, -1)}, **rest)
        refused(call, **{**here, name: At(t, 1)}, **rest)


def test_rope_table_refuses_factors_on_the_host(monkeypatch):
    import torch
    monkeypatch.setattr(mv, "_current_device", lambda: 0)
    refused(mv.rope_table, rot_dim=8, n_pos=4, freq_factors=torch.ones(4), device="cpu")
