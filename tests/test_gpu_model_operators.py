"""Models whose layers norm their query and key heads or use differential
attention (optional GGUF tensors attn_q_norm, attn_k_norm, attn_diff_lambda,
attn_diff_norm): le_embed_ids against the same forward in 64 bits from the
model's F32 tensors, within the parity bar of the plain models (cosine >=
0.99999, largest difference 2e-3)."""
import math

import numpy as np
import pytest

from llm_embed_b200 import synth
from llm_embed_b200.embed import LE_EINVAL, Embedder, HParams, LlmEmbedError

pytestmark = pytest.mark.gpu


def spec_of(qk_norm, diff_attn, **kw):
    return synth.ModelSpec(layers=2, vocab=2048, seed=31, eps=1e-6, embd_type=synth.GGML_F32,
                           weight_types=(synth.GGML_F32,) * 5, qk_norm=qk_norm, diff_attn=diff_attn, **kw)


def layernorm(x, w, b, eps):
    x = x - x.mean(1, keepdims=True)
    return x / np.sqrt((x * x).mean(1, keepdims=True) + eps) * w + b


def rms(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def softmax(s):
    p = np.exp(s - s.max(-1, keepdims=True))
    return p / p.sum(-1, keepdims=True)


def gelu(v):
    t = 0.7978845608 * v * (1 + 0.044715 * v * v)
    r = np.where(np.abs(t) > 4.97, np.sign(t), t * (27 + t * t) / (27 + 9 * t * t))
    return 0.5 * v * (1 + r)


def forward64(path, spec, ids):
    """One sequence's embedding."""
    _, tensors = synth.read_gguf(path)

    def w(name):
        _, dims, data = tensors[name]
        a = np.frombuffer(data, np.float32).astype(np.float64)
        return a.reshape(dims[1], dims[0]) if len(dims) > 1 else a

    H, h, d, L, eps = spec.hidden, spec.heads, spec.hidden // spec.heads, len(ids), float(np.float32(spec.eps))
    x = layernorm(w("token_embd.weight")[ids] + w("token_types.weight")[0], w("token_embd_norm.weight"),
                  w("token_embd_norm.bias"), eps)
    angle = np.arange(L)[:, None] * spec.rope_base ** (-np.arange(0, d, 2) / d)
    cos, sin = np.cos(angle)[:, None], np.sin(angle)[:, None]

    def rotate(u):
        out = np.empty_like(u)
        a, b = u[..., 0::2], u[..., 1::2]
        out[..., 0::2], out[..., 1::2] = a * cos - b * sin, a * sin + b * cos
        return out

    for i in range(spec.layers):
        p = f"blk.{i}."
        q, k, v = np.split(x @ w(p + "attn_qkv.weight").T, 3, 1)
        q, k = q.reshape(L, h, d), k.reshape(L, h, d)
        if spec.qk_norm:
            q, k = rms(q, w(p + "attn_q_norm.weight"), eps), rms(k, w(p + "attn_k_norm.weight"), eps)
        q, k = rotate(q), rotate(k)
        maps = softmax(np.einsum("ihd,jhd->hij", q, k) / math.sqrt(d))
        if spec.diff_attn:
            lam = w(p + "attn_diff_lambda.weight")
            init = 0.8 - 0.6 * math.exp(-0.3 * i)
            lam = math.exp(lam[0] @ lam[1]) - math.exp(lam[2] @ lam[3]) + init
            o = np.einsum("hij,jhd->ihd", maps[0::2] - lam * maps[1::2], v.reshape(L, h // 2, 2 * d))
            o = (1 - init) * rms(o, w(p + "attn_diff_norm.weight"), eps)
        else:
            o = np.einsum("hij,jhd->ihd", maps, v.reshape(L, h, d))
        x = layernorm(x + o.reshape(L, H) @ w(p + "attn_output.weight").T, w(p + "attn_output_norm.weight"),
                      w(p + "attn_output_norm.bias"), eps)
        f = (gelu(x @ w(p + "ffn_gate.weight").T) * (x @ w(p + "ffn_up.weight").T)) @ w(p + "ffn_down.weight").T
        x = layernorm(x + f, w(p + "layer_output_norm.weight"), w(p + "layer_output_norm.bias"), eps)
    e = x.mean(0)
    return e / np.linalg.norm(e)


@pytest.mark.parametrize("qk_norm,diff_attn", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("lens", [[8], [5, 3, 8], [30, 1, 17], [60, 64, 9, 33], [130, 100, 70, 300], [16] * 40 + [128] * 4])
def test_model_with_operators(model_path, qk_norm, diff_attn, lens):
    """Every GEMM path (a few tokens, small and large batches) and attention
    kernel; replayed calls give the same bits."""
    spec = spec_of(qk_norm, diff_attn)
    path = model_path(spec)
    ids, offs = synth.make_ids(lens, seed=7, vocab=spec.vocab)
    e = Embedder.Load(path)
    try:
        got = e.EmbedIDs(ids, offs)
        for _ in range(2):
            assert np.array_equal(e.EmbedIDs(ids, offs), got)
        e.sync()
    finally:
        e.Close()
    for s in sorted({0, 1 % len(lens), len(lens) - 1}):
        ref = forward64(path, spec, ids[offs[s]:offs[s + 1]])
        cos = float(got[s] @ ref / np.linalg.norm(got[s]))
        assert cos >= 0.99999 and np.abs(got[s] - ref).max() <= 2e-3, (s, cos, np.abs(got[s] - ref).max())


def test_tensors_come_together_and_fit(model_path):
    """One of a pair missing, or of another size, is refused at load."""
    spec = spec_of(True, True)
    kv, tensors = synth.read_gguf(model_path(spec))
    hp = HParams(n_layers=spec.layers, hidden=spec.hidden, ffn=spec.ffn, heads=spec.heads, context_length=spec.context,
                 ln_eps=spec.eps, rope_base=spec.rope_base)

    def load(change):
        ts = {n: (t, list(dims), bytes(b)) for n, (t, dims, b) in tensors.items()}
        change(ts)
        Embedder.LoadTensors([(n, *x) for n, x in ts.items()], hp).Close()

    load(lambda ts: None)
    for name in ("attn_q_norm", "attn_k_norm", "attn_diff_lambda", "attn_diff_norm"):
        key = f"blk.1.{name}.weight"

        def short(ts):
            t, dims, b = ts[key]
            ts[key] = (t, [dims[0] - 1] + dims[1:], b)

        for change in (lambda ts: ts.pop(key), short):
            with pytest.raises(LlmEmbedError) as err:
                load(change)
            assert err.value.code == LE_EINVAL


def embed_tensors(ts, spec, ids, offs):
    hp = HParams(n_layers=spec.layers, hidden=spec.hidden, ffn=spec.ffn, heads=spec.heads, context_length=spec.context,
                 ln_eps=spec.eps, rope_base=spec.rope_base)
    e = Embedder.LoadTensors([(n, *x) for n, x in ts.items()], hp)
    try:
        return e.EmbedIDs(ids, offs)
    finally:
        e.Close()


@pytest.mark.parametrize("size,bias", [("row", True), ("row", False), ("head", True)])
def test_norms_of_another_kind_are_not_read(model_path, size, bias):
    """Norms of whole query and key rows, or with a bias, are another operator
    than the heads' norm: a model that has them gives what it does without, as
    in the reference, which knows no such tensors."""
    spec = spec_of(False, False)
    _, tensors = synth.read_gguf(model_path(spec))
    ids, offs = synth.make_ids([30, 1, 17], seed=7, vocab=spec.vocab)
    ts = {n: (t, list(dims), bytes(b)) for n, (t, dims, b) in tensors.items()}
    want = embed_tensors(ts, spec, ids, offs)
    n = spec.hidden if size == "row" else spec.hidden // spec.heads
    for i in range(spec.layers):
        for name in ("attn_q_norm", "attn_k_norm"):
            ts[f"blk.{i}.{name}.weight"] = (synth.GGML_F32, [n], np.full(n, 1.5, np.float32).tobytes())
            if bias:
                ts[f"blk.{i}.{name}.bias"] = (synth.GGML_F32, [n], np.full(n, 0.5, np.float32).tobytes())
    assert np.array_equal(embed_tensors(ts, spec, ids, offs), want)


@pytest.mark.parametrize("dims,fits", [([64, 4], True), ([256], True), ([4, 64], False), ([128, 2], False)])
def test_lambda_layout(model_path, dims, fits):
    """The learned weights are four vectors of head_dim one after another; the
    same number of values in another layout is refused."""
    spec = spec_of(False, True)
    _, tensors = synth.read_gguf(model_path(spec))
    ids, offs = synth.make_ids([9], seed=7, vocab=spec.vocab)
    ts = {n: (t, list(d), bytes(b)) for n, (t, d, b) in tensors.items()}
    want = embed_tensors(ts, spec, ids, offs)
    for i in range(spec.layers):
        t, _, b = ts[f"blk.{i}.attn_diff_lambda.weight"]
        ts[f"blk.{i}.attn_diff_lambda.weight"] = (t, dims, b)
    if fits:
        assert np.array_equal(embed_tensors(ts, spec, ids, offs), want)
    else:
        with pytest.raises(LlmEmbedError) as err:
            embed_tensors(ts, spec, ids, offs)
        assert err.value.code == LE_EINVAL
