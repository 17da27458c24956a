"""LlamaModel over the 4-bit cache (kv_type=KV_Q4_0) against the same model in
64 bits with the cache quantised by the formulas, and against itself by its
three routes: a prompt, one token at a time, a batch of sequences.
"""
from __future__ import annotations

import ctypes as C
import dataclasses
import os
import tempfile

import numpy as np
import pytest

import memvanta_b200 as mv
from memvanta_b200 import gguf

FULL = gguf.LlamaShape(n_layer=2, n_embd=512, n_head=8, n_head_kv=4, n_ff=768, vocab=512, n_ctx=512, rms_eps=1e-6,
                       rope_theta=10000.0, layer_type=gguf.F32, embd_type=gguf.F32, output_type=gguf.F32)
MID = gguf.LlamaShape(n_layer=3, n_embd=1024, n_head=8, n_head_kv=4, n_ff=1536, vocab=1024, n_ctx=512, rms_eps=1e-6,
                      rope_theta=10000.0, output_type=gguf.Q4_0)


@pytest.fixture(scope="module")
def tmp():
    with tempfile.TemporaryDirectory() as d:
        yield d


def written(tmp, name, shape, seed):
    path = os.path.join(tmp, name)
    if not os.path.exists(path):
        gguf.write_random_llama(path, shape, seed=seed)
    return path


def bf16(x):
    """Nearest bf16 (ties to even) of float32 values."""
    b = np.asarray(x, np.float32).view(np.uint32)
    return ((b + 0x7fff + ((b >> 16) & 1)) & 0xffff0000).astype(np.uint32).view(np.float32)


def held4(x):
    """What the 4-bit cache holds of rows x [.., 32 k]."""
    b = np.asarray(x, np.float32).reshape(-1, 32)
    mx = b[np.arange(len(b)), np.argmax(np.abs(b), axis=1)]
    d = bf16(mx / np.float32(-8))
    inv = np.divide(np.float32(1), d, out=np.zeros_like(d), where=d != 0)
    n = np.clip(np.floor(b * inv[:, None] + np.float32(8.5)), 0, 15)
    return ((n - 8).astype(np.float64) * d[:, None]).reshape(np.shape(x))


class Model64:
    """The decoder with F32 weights, one token after another, in 64 bits."""

    def __init__(self, path, shape, quantise=True, noise=0.0):
        self.s, self.hold = shape, held4 if quantise else (lambda x: np.asarray(x, np.float64))
        _, infos = gguf.read_tensor_infos(path)
        raw = np.memmap(path, np.uint8)
        self.w = {i.name: np.frombuffer(raw[i.offset:i.offset + i.nbytes].tobytes(), np.float32).astype(np.float64)
                  .reshape([i.rows, i.cols] if len(i.dims) > 1 else [-1]) for i in infos}
        self.k, self.v = ([[] for _ in range(shape.n_layer)] for _ in range(2))
        self.rng, self.noise = np.random.default_rng(1), noise

    def norm(self, x, name):
        return x / np.sqrt(np.mean(x * x) + self.s.rms_eps) * self.w[name]

    def rope(self, x, pos):
        h = x.shape[1] // 2
        a = pos * self.s.rope_theta ** (-np.arange(h) / h)
        c, s, lo, hi = np.cos(a), np.sin(a), x[:, :h], x[:, h:]
        return np.concatenate([lo * c - hi * s, lo * s + hi * c], axis=1)

    def forward(self, token):
        s, w = self.s, self.w
        hd, G, pos = s.n_embd // s.n_head, s.n_head // s.n_head_kv, len(self.k[0])
        x = w["token_embd.weight"][token].copy()
        for i in range(s.n_layer):
            p = f"blk.{i}."
            n = self.norm(x, p + "attn_norm.weight")
            q, k, v = ((w[p + f"attn_{a}.weight"] @ n).reshape(-1, hd) for a in "qkv")
            k, v = self.rope(k, pos), v
            if self.noise:
                k, v = (y * (1 + self.noise * self.rng.standard_normal(y.shape)) for y in (k, v))
            self.k[i].append(self.hold(k))
            self.v[i].append(self.hold(v))
            K, V = np.stack(self.k[i]).repeat(G, 1), np.stack(self.v[i]).repeat(G, 1)
            sc = np.einsum("hd,thd->ht", self.rope(q, pos), K) / np.sqrt(hd)
            e = np.exp(sc - sc.max(1, keepdims=True))
            att = np.einsum("ht,thd->hd", e / e.sum(1, keepdims=True), V)
            x = x + w[p + "attn_output.weight"] @ att.reshape(-1)
            n = self.norm(x, p + "ffn_norm.weight")
            g, u = (w[p + f"ffn_{a}.weight"] @ n for a in ("gate", "up"))
            x = x + w[p + "ffn_down.weight"] @ (g / (1 + np.exp(-g)) * u)
        return w["output.weight"] @ self.norm(x, "output_norm.weight")


# A key or value that lies within its fp32 error of a rounding boundary may be
# held one step apart from the 64-bit model's, and the next layer's with it: the
# logits then move by up to 2.5e-3 of their largest (taken on the CPU, with
# noise of fp32's size on every key and value), whereas dropping the
# quantisation moves them by 0.07 to 0.14.  The tolerance stands between, and
# test_tolerance_and_what_it_can_see holds it there.
TOL64 = 1.5e-2


def test_tolerance_and_what_it_can_see(tmp):
    path = written(tmp, "full.gguf", FULL, 31)
    prompt = np.random.default_rng(3).integers(0, FULL.vocab, size=40)
    runs = [Model64(path, FULL), Model64(path, FULL, noise=3e-6), Model64(path, FULL, quantise=False)]
    held, near, plain = ([m.forward(int(t)) for t in prompt] for m in runs)
    for a, b, c in zip(held[1:], near[1:], plain[1:]):
        assert np.max(np.abs(a - b)) <= TOL64 / 4 * np.max(np.abs(a))
    assert max(np.max(np.abs(a - c)) / np.max(np.abs(a)) for a, c in zip(held, plain)) > 4 * TOL64


@pytest.mark.gpu
def test_model_follows_the_64_bit_model(cuda, tmp):
    """Prompt chunks (one by one, a few, and enough for the tensor cores),
    then decode steps; page 13 ends inside every tile."""
    path = written(tmp, "full.gguf", FULL, 31)
    prompt = np.random.default_rng(4).integers(0, FULL.vocab, size=330).astype(np.int32)
    ref = Model64(path, FULL)
    m = mv.LlamaModel(path, ctx_override=512, kv_page_tokens=13, kv_type=mv.KV_Q4_0)
    try:
        at = 0
        for n in (1, 2, 7, 170, 150):
            got = m.prefill(prompt[at:at + n], 256).copy()
            want = [ref.forward(int(t)) for t in prompt[at:at + n]][-1]
            at += n
            assert m.position() == at
            assert np.max(np.abs(got - want)) <= TOL64 * np.max(np.abs(want)), (at, n)
        for step in range(6):
            tok = int(np.argmax(want))
            got, want = m.forward(tok).copy(), ref.forward(tok)
            assert np.max(np.abs(got - want)) <= TOL64 * np.max(np.abs(want)), step
        kvd = FULL.n_head_kv * 64
        tokens = -(-m.position() // 13) * 13
        assert m.kv_bytes_allocated() == 2 * FULL.n_layer * tokens * (kvd // 2 + kvd // 32 * 2)
        m.reset()
        again = m.prefill(prompt[:1], 1).copy()
        first = Model64(path, FULL).forward(int(prompt[0]))
        assert np.max(np.abs(again - first)) <= TOL64 * np.max(np.abs(first))
    finally:
        m.close()


@pytest.mark.gpu
def test_long_prompt_in_chunks(cuda, tmp):
    """A prompt of several merged chunks, which overlap on two streams."""
    shape = dataclasses.replace(FULL, n_ctx=1400)
    path = written(tmp, "long.gguf", shape, 33)
    prompt = np.random.default_rng(8).integers(0, shape.vocab, size=1300).astype(np.int32)
    ref = Model64(path, shape)
    m = mv.LlamaModel(path, ctx_override=1400, kv_page_tokens=64, kv_type=mv.KV_Q4_0)
    try:
        got = m.prefill(prompt, 128).copy()
        want = [ref.forward(int(t)) for t in prompt][-1]
        assert np.max(np.abs(got - want)) <= TOL64 * np.max(np.abs(want))
        for _ in range(3):
            tok = int(np.argmax(want))
            got, want = m.forward(tok).copy(), ref.forward(tok)
            assert np.max(np.abs(got - want)) <= TOL64 * np.max(np.abs(want))
    finally:
        m.close()


@pytest.mark.gpu
def test_many_sequences(cuda, tmp):
    """A set of 70 sequences against the 64-bit model, a few of them at a time."""
    path = written(tmp, "full.gguf", FULL, 31)
    rng = np.random.default_rng(9)
    prompts = [rng.integers(0, FULL.vocab, size=1 + 3 * i % 50).astype(np.int32) for i in range(70)]
    steps = rng.integers(0, FULL.vocab, size=(4, 70)).astype(np.int32)
    m = mv.LlamaModel(path, ctx_override=128, kv_page_tokens=16, kv_type=mv.KV_Q4_0)
    try:
        S = m.open_sequences(70, 64)
        try:
            for i, p in enumerate(prompts):
                S.prefill(i, p, 32)
            got = [S.forward(t).copy() for t in steps]
        finally:
            S.close()
    finally:
        m.close()
    for i in (0, 1, 17, 40, 69):
        ref = Model64(path, FULL)
        for t in prompts[i]:
            ref.forward(int(t))
        for k in range(4):
            want = ref.forward(int(steps[k, i]))
            assert np.max(np.abs(got[k][i] - want)) <= TOL64 * np.max(np.abs(want)), (i, k)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 128])
def test_batched_and_single_decode_agree(cuda, tmp, page):
    """Q4_0 weights: a set's prompts are the model's bit for bit; the steps
    split the cache otherwise, so a Q8 activation may round the other way (a
    step of 1/127 in some of 1024 inputs of a projection: 1e-3 of the logits'
    size, taken 20 times)."""
    path = written(tmp, "mid.gguf", MID, 32)
    m = mv.LlamaModel(path, ctx_override=512, kv_page_tokens=page, kv_type=mv.KV_Q4_0)
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, MID.vocab, size=n).astype(np.int32) for n in (1, 33, 150, 260)]
    forced = rng.integers(0, MID.vocab, size=(6, len(prompts))).astype(np.int32)
    try:
        ref = []
        for i, p in enumerate(prompts):
            m.reset()
            ref.append([m.prefill(p, 128).copy()] + [m.forward(int(forced[k, i])).copy() for k in range(6)])
        S = m.open_sequences(len(prompts), 300)
        try:
            for i, p in enumerate(prompts):
                assert np.array_equal(S.prefill(i, p, 128), ref[i][0]), i
            for k in range(6):
                got = S.forward(forced[k]).copy()
                for i in range(len(prompts)):
                    want = ref[i][k + 1]
                    assert np.max(np.abs(got[i] - want)) <= 2e-2 * np.max(np.abs(want)), (k, i)
        finally:
            S.close()
        # the same calls give the same bits
        m.reset()
        assert np.array_equal(m.prefill(prompts[-1], 128), ref[-1][0])
        assert np.array_equal(m.forward(int(forced[0, -1])), ref[-1][1])
    finally:
        m.close()


@pytest.mark.gpu
def test_generate_follows_the_steps(cuda, tmp):
    path = written(tmp, "mid.gguf", MID, 32)
    m = mv.LlamaModel(path, ctx_override=256, kv_page_tokens=16, kv_type=mv.KV_Q4_0)
    try:
        prompt = np.random.default_rng(6).integers(0, MID.vocab, size=20).astype(np.int32)
        m.prefill(prompt[:-1], 64, False)
        toks, cur = [], int(prompt[-1])
        for _ in range(10):
            cur = int(np.argmax(m.forward(cur)))
            toks.append(cur)
        assert m.generate(prompt.tolist(), 10) == toks
        m.reset()
        m.prefill(prompt[:-1], 64, False)
        assert list(m.generate_greedy(int(prompt[-1]), 10)) == toks
    finally:
        m.close()


@pytest.mark.gpu
def test_refusals(cuda, tmp):
    path = written(tmp, "mid.gguf", MID, 32)
    h = C.c_void_p()
    lib = mv._lib.load()
    assert lib.mv_model_open_tp(path.encode(), 128, 16, mv.KV_Q4_0, 0, 2, 64, C.byref(h)) == mv._lib.MV_ERR_UNSUPPORTED
    assert not h.value
    with pytest.raises(mv.MemVantaError, match="unknown KV cache type"):
        mv.LlamaModel(path, ctx_override=128, kv_page_tokens=16, kv_type=5)
    m = mv.LlamaModel(path, ctx_override=8, kv_page_tokens=16, kv_type=mv.KV_Q4_0)
    try:
        with pytest.raises(mv.MemVantaError, match="context exhausted"):
            m.prefill(list(range(9)), 4)
        m.prefill(list(range(8)), 4)
        with pytest.raises(mv.MemVantaError, match="context exhausted"):
            m.forward(1)
    finally:
        m.close()
