"""LlamaModel over the 4-bit cache at the end of a long context: its rotary
angles.  One layer, so that the last token's logits follow from every token's
own key and value; frequencies of 1 to 1/2, where an angle rounded to fp32 is off
by up to 2^-8 at 131,071."""
from __future__ import annotations

import numpy as np
import pytest

import memvanta_b200 as mv
from memvanta_b200 import gguf
from test_gpu_model_q4 import held4

N = 131_072
SHAPE = gguf.LlamaShape(n_layer=1, n_embd=128, n_head=2, n_head_kv=1, n_ff=128, vocab=256, n_ctx=N, rms_eps=1e-6,
                        rope_theta=2.0, layer_type=gguf.F32, embd_type=gguf.F32, output_type=gguf.F32)


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    """A GGUF file with q, k and v weights 8 times as large (scores of a standard
    deviation of 3), and its tensors in 64 bits."""
    path = str(tmp_path_factory.mktemp("q4") / "long.gguf")
    gguf.write_random_llama(path, SHAPE, seed=5)
    _, infos = gguf.read_tensor_infos(path)
    raw = np.memmap(path, np.uint8, mode="r+")
    w = {}
    for i in infos:
        x = np.frombuffer(raw[i.offset:i.offset + i.nbytes].tobytes(), np.float32).copy()
        if i.name.startswith("blk.0.attn_") and i.name[11] in "qkv":
            x *= 8
            raw[i.offset:i.offset + i.nbytes] = x.view(np.uint8)
        w[i.name] = x.astype(np.float64).reshape([i.rows, i.cols] if len(i.dims) > 1 else [-1])
    raw.flush()
    return path, w


def last_logits(w, tokens, angles, noise=0.0):
    """Logits of the last token, the cache quantised by the formulas."""
    hd, h = 64, 32
    norm = lambda x, name: x / np.sqrt(np.mean(x * x, -1, keepdims=True) + SHAPE.rms_eps) * w[name]  # noqa: E731
    n = norm(w["token_embd.weight"], "blk.0.attn_norm.weight")
    q, k, v = ((n @ w[f"blk.0.attn_{a}.weight"].T)[tokens] for a in "qkv")
    c, s = np.cos(angles), np.sin(angles)
    turn = lambda x, c, s: np.concatenate([x[..., :h] * c - x[..., h:] * s,  # noqa: E731
                                           x[..., :h] * s + x[..., h:] * c], -1)
    k, q = turn(k, c, s), turn(q[-1].reshape(2, hd), c[-1], s[-1])
    if noise:
        rng = np.random.default_rng(1)
        k, v = (y * (1 + noise * rng.standard_normal(y.shape)) for y in (k, v))
    k, v = held4(k), held4(v)
    sc = q @ k.T / np.sqrt(hd)
    e = np.exp(sc - sc.max(1, keepdims=True))
    out = e / e.sum(1, keepdims=True) @ v
    x = w["token_embd.weight"][tokens[-1]] + w["blk.0.attn_output.weight"] @ out.reshape(-1)
    n = norm(x, "blk.0.ffn_norm.weight")
    g, u = (w[f"blk.0.ffn_{a}.weight"] @ n for a in ("gate", "up"))
    x = x + w["blk.0.ffn_down.weight"] @ (g / (1 + np.exp(-g)) * u)
    return w["output.weight"] @ norm(x, "output_norm.weight")


@pytest.fixture(scope="module")
def expected(model):
    """(tokens, logits with exact angles, with fp32's, with exact ones and fp32's noise on keys and values)"""
    tokens = np.random.default_rng(2).integers(0, SHAPE.vocab, N).astype(np.int32)
    inv = SHAPE.rope_theta ** (-np.arange(32) / 32)
    exact = np.arange(N)[:, None] * inv
    rounded = (np.arange(N, dtype=np.float32)[:, None] * inv.astype(np.float32)).astype(np.float64)
    w = model[1]
    return tokens, last_logits(w, tokens, exact), last_logits(w, tokens, rounded), last_logits(w, tokens, exact, 3e-6)


def test_what_the_angles_can_be_told_by(expected):
    """Rounded angles move the logits by a hundred times what fp32's noise does."""
    _, exact, rounded, near = expected
    assert np.max(np.abs(rounded - exact)) >= 50 * np.max(np.abs(near - exact))


@pytest.mark.gpu
def test_angles_at_the_end_of_a_long_context(cuda, model, expected):
    tokens, exact, rounded, _ = expected
    m = mv.LlamaModel(model[0], ctx_override=N, kv_page_tokens=64, kv_type=mv.KV_Q4_0)
    try:
        m.prefill(tokens[:-1], 512, False)
        got = m.forward(int(tokens[-1]))
    finally:
        m.close()
    assert np.max(np.abs(got - exact)) <= np.max(np.abs(rounded - exact)) / 8
