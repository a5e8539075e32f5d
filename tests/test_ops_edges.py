"""The stand-alone operators (llm_embed_b200.ops) at the ends of their ranges:
rows further apart than 32 bits count, weights of millions of rows, scores of
minus infinity, and sizes that are refused.

Rows far apart give the bits of the same rows packed.  The wide weight's
products are sums of at most 64 small integers, exact in float32.  Attention
has the tolerance of test_ops.py.
"""
import os
import subprocess
import sys

import numpy as np
import pytest

from llm_embed_b200 import ops
from test_ops import INIT, check_diff, diff64, expect_einval, gen, lambdas, make_diff, make_f8, run_diff, stream

gpu = pytest.mark.gpu
FAR = 1 << 27  # elements between rows: row 16 begins past 2^31, row 32 past 2^32
ROWS = 40


@pytest.fixture(scope="module")
def far():
    """bfloat16 [ROWS][FAR], columns from 32768 on never touched."""
    import torch
    x = torch.empty(ROWS * FAR, device="cuda", dtype=torch.bfloat16)
    yield x
    del x
    torch.cuda.empty_cache()


def columns(far, first, n, dtype=None):
    """Columns first .. first + n of every row."""
    x = far if dtype is None else far.view(dtype)
    return x.as_strided((ROWS, n), (FAR * far.element_size() // x.element_size(), 1), first)


@gpu
@pytest.mark.parametrize("d,rot", [(64, 64), (80, 24)])
def test_qk_norm_rows_far_apart(far, d, rot):
    import torch
    h = 3
    x = torch.randn(ROWS, h * d, device="cuda", generator=gen(d)).bfloat16()
    pos = torch.arange(ROWS, device="cuda", dtype=torch.int32)
    r = ops.Rope(ROWS, rot, pairing="half")
    want = torch.empty_like(x)
    r.qk_norm_device("bf16", ROWS, h, 0, d, x.data_ptr(), 0, pos.data_ptr(), want.data_ptr(), 0, stream=stream())
    q, k, out = (columns(far, 1024 * i, h * d) for i in range(3))
    q.copy_(x)
    k.copy_(x)
    r.qk_norm_device("bf16", ROWS, h, h, d, q.data_ptr(), k.data_ptr(), pos.data_ptr(), out.data_ptr(), k.data_ptr(),
                     q_stride=FAR, k_stride=FAR, q_out_stride=FAR, k_out_stride=FAR, stream=stream())
    r.sync()
    assert torch.equal(out, want) and torch.equal(k, want)
    r.close()


@gpu
@pytest.mark.parametrize("m", [5, 20, ROWS])
def test_product_rows_far_apart(far, m):
    import torch
    n, k = 200, 272
    w8, ws = make_f8(n, k, 2)
    w = ops.F8Weight(w8.data_ptr(), ws.data_ptr(), n, k)
    x = torch.randn(m, k, device="cuda", generator=gen(m)).bfloat16()
    work = torch.empty(w.workspace_bytes(m, "bf16"), device="cuda", dtype=torch.uint8)
    args = dict(d_work=work.data_ptr(), work_bytes=work.numel(), stream=stream())
    want = torch.empty(m, n, device="cuda", dtype=torch.bfloat16)
    w.matmul_device(x.data_ptr(), m, want.data_ptr(), "bf16", "bf16", **args)
    fx, fy = columns(far, 0, k)[:m], columns(far, 1024, n)[:m]
    fx.copy_(x)
    w.matmul_device(fx.data_ptr(), m, fy.data_ptr(), "bf16", "bf16", ldx=FAR, ldy=FAR, **args)
    w.sync()
    assert torch.equal(fy, want)
    # Rows that are quantised already.
    q = torch.empty(m, k, device="cuda", dtype=torch.uint8)
    s = torch.empty(-(-k // 128), m, device="cuda")
    ops.f8_quantize_device(fx.data_ptr(), "bf16", m, k, q.data_ptr(), s.data_ptr(), ldx=FAR, stream=stream())
    fq = columns(far, 8192, k, torch.uint8)[:m]
    fq.copy_(q)
    fy.zero_()
    w.matmul_device(fq.data_ptr(), m, fy.data_ptr(), "e4m3", "bf16", ldx=2 * FAR, ldy=FAR, d_x_scales=s.data_ptr(),
                    stream=stream())
    w.sync()
    assert torch.equal(fy, want)
    w.close()


@gpu
@pytest.mark.parametrize("lens", [[30, 10], [3, 0, 37]])
def test_diff_attention_rows_far_apart(far, lens):
    import torch
    h, d = 2, 64
    q, k, v, offs, t = make_diff(lens, h, h, d, "bf16", 8)
    lam, _ = lambdas(h, d, True, 3)
    a = ops.DiffAttention(h, h, d, lam, INIT, np.ones(2 * d, np.float32))
    o = torch.from_numpy(offs).cuda()
    parts = [columns(far, 1024 * i, 2 * h * d) for i in range(4)]
    for p, x in zip(parts, (q, k, v)):
        p.copy_(x)
    for hint in (0, 1, 40, 100):
        want = run_diff(a, q, k, v, offs, t, h, d, "bf16", hint)
        parts[3].zero_()
        a.run_device("bf16", *(p.data_ptr() for p in parts[:3]), o.data_ptr(), len(lens), t, hint, parts[3].data_ptr(),
                     q_stride=FAR, k_stride=FAR, v_stride=FAR, out_stride=FAR, stream=stream())
        a.sync()
        assert torch.equal(parts[3], want)
    a.close()


@gpu
def test_weight_of_millions_of_rows():
    """More blocks of 128 rows than a grid's second dimension has."""
    import torch
    n, k = 65535 * 128 + 300, 16
    g = np.random.default_rng(1)
    rows = np.exp2(g.integers(-1, 2, (999, k))).astype(np.float32) * g.choice([-1, 1], (999, k))
    w = ops.F8Weight.from_float(np.resize(rows.astype(np.float32), (n, k)))
    q, s = w.read()
    assert s.shape == (65538, 1) and (s == 2.0 ** -7).all()  # largest 2: 2 / 2^-7 = 256, 2 / 2^-8 > 448
    for m in (3, 40):
        x = torch.from_numpy(g.integers(-2, 3, (m, k)).astype(np.float32)).cuda()
        y = torch.empty(m, n, device="cuda")
        work = torch.empty(w.workspace_bytes(m, "f32"), device="cuda", dtype=torch.uint8)
        w.matmul_device(x.data_ptr(), m, y.data_ptr(), "f32", "f32", d_work=work.data_ptr(), work_bytes=work.numel(),
                        stream=stream())
        w.sync()
        for first in (0, n // 2, n - 999):
            ref = x.cpu().numpy().astype(np.float64) @ rows[(first + np.arange(999)) % 999].T
            assert np.array_equal(y[:, first:first + 999].cpu().numpy(), ref)
        del y
    w.close()


@gpu
@pytest.mark.parametrize("n,dead", [(60, 30), (120, 64), (120, 100), (300, 130), (300, 299)])
def test_diff_attention_scores_of_minus_infinity(n, dead):
    """Keys whose score is -inf have weight 0, also where they fill the first
    blocks; a row of nothing else is NaN."""
    import torch
    h, d = 2, 64
    q, k, v, offs, t = make_diff([n, n] + 8 * [1], h, h, d, "f16", n)  # short on average
    dead2 = slice(n, 2 * n)
    q[:, 0] = 1  # head 0, map 1
    k[:dead, 0] = float("-inf")
    k[dead2, 2 * d] = float("-inf")  # the second sequence's head 1: every key
    q[:, 2 * d] = 1
    lam, val = lambdas(h, d, True, 2)
    a = ops.DiffAttention(h, h, d, lam, INIT, None)
    ref, mag = diff64(q, k, v, offs.tolist(), h, h, d, val, INIT, None, 0)
    assert torch.isfinite(ref[:n]).all() and torch.isnan(ref[dead2, 1]).all()
    for hint in (0, 1, n):
        out = run_diff(a, q, k, v, offs, t, h, d, "f16", hint).reshape(ref.shape)
        assert torch.isnan(out[dead2, 1]).all()
        check_diff(out[:n], ref[:n], mag[:n], "f16")
        check_diff(out[n:, 0], ref[n:, 0], mag[n:, 0], "f16")
        check_diff(out[2 * n:], ref[2 * n:], mag[2 * n:], "f16")
    a.sync()
    a.close()


def test_sizes_that_are_refused():
    """Beyond 32 bits (a C int would cut them) and beyond what the kernels count."""
    w, s = np.zeros(16, np.uint8), np.ones(1, np.float32)
    big = 1 << 30
    for n, k in ((1 << 32) + 1, 16), (1, (1 << 32) + 16), (big + 1, 16), (1, big + 16):
        expect_einval(lambda: ops.F8Weight(w.ctypes.data, s.ctypes.data, n, k))
    expect_einval(lambda: ops.F8Weight.from_float(np.zeros(16, np.float32)))
    expect_einval(lambda: ops.F8Weight.from_float(np.zeros((1, 1, 16), np.float32)))
    for m, k in ((1 << 32) + 1, 16), (1, (1 << 32) + 16), (big + 1, 16), (1, big + 1):
        expect_einval(lambda: ops.f8_quantize_device(64, "f16", m, k, 64, 64))
    expect_einval(lambda: ops.f8_quantize_device(64, "f16", 1, 16, 64, 64, dev=1 << 32))
    expect_einval(lambda: ops.Rope((1 << 32) + 1, 64))
    expect_einval(lambda: ops.Rope(16, (1 << 32) + 64))
    expect_einval(lambda: ops.DiffAttention((1 << 32) + 1, 1, 64, np.zeros((4, 64), np.float32), 0.8))


@gpu
def test_rows_and_sequences_that_are_refused():
    w8, ws = make_f8(32, 64, 1)
    w = ops.F8Weight(w8.data_ptr(), ws.data_ptr(), 32, 64)
    for m in ((1 << 30) + 1, 1 << 32, -1):
        expect_einval(lambda: w.workspace_bytes(m, "f16"))
        expect_einval(lambda: w.matmul_device(w8.data_ptr(), m, w8.data_ptr(), d_work=w8.data_ptr(), work_bytes=1 << 50))
    w.close()
    a = ops.DiffAttention(2, 1, 64, np.zeros((4, 64), np.float32), INIT)
    p = w8.data_ptr()
    for nseq in ((1 << 30) + 1, 1 << 32):
        expect_einval(lambda: a.run_device("f16", p, p, p, p, nseq, 2, 0, p, stream=stream()))
    a.close()


FIRST_CALLS = """
import numpy as np, torch
from llm_embed_b200 import ops
t, h, d = %d, 2, 64
W = 2 * h * d
g = torch.Generator("cuda").manual_seed(1)
x = torch.randn(t, W, device="cuda", generator=g).half()
w = ops.F8Weight.from_float(np.random.default_rng(1).standard_normal((3 * W, W)).astype(np.float32) / 16)
rope, att = ops.Rope(t, d), ops.DiffAttention(h, h, d, np.zeros((4, d), np.float32), 0.5)
pos = torch.arange(t, device="cuda", dtype=torch.int32)
offs = torch.tensor([0, t // 2, t], device="cuda", dtype=torch.int32)
work = torch.empty(w.workspace_bytes(t, "f16"), device="cuda", dtype=torch.uint8)
qkv, out = (torch.zeros(t, n, device="cuda", dtype=torch.float16) for n in (3 * W, W))
q8, s8 = torch.zeros(t, W, device="cuda", dtype=torch.uint8), torch.zeros(2, t, device="cuda")

def layer(s):
    ops.f8_quantize_device(x.data_ptr(), "f16", t, W, q8.data_ptr(), s8.data_ptr(), stream=s)
    w.matmul_device(x.data_ptr(), t, qkv.data_ptr(), d_work=work.data_ptr(), work_bytes=work.numel(), stream=s)
    q, k, v = (qkv.data_ptr() + 2 * W * i for i in range(3))
    rope.qk_norm_device("f16", t, 2 * h, 2 * h, d, q, k, pos.data_ptr(), q, k, 3 * W, 3 * W, 3 * W, 3 * W, stream=s)
    att.run_device("f16", q, k, v, offs.data_ptr(), 2, t, %d, out.data_ptr(), 3 * W, 3 * W, 3 * W, stream=s)

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):  # the process's first call of each
    layer(torch.cuda.current_stream().cuda_stream)
graph.replay()
torch.cuda.synchronize()
got = [y.clone() for y in (q8, s8, qkv, out)]
for y in (q8, s8, qkv, out):
    y.zero_()
layer(ops.LEGACY_STREAM)
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, (q8, s8, qkv, out))) and float(out.abs().max()) > 0
# Other sequences in the same graph: offsets are read at each replay.
offs.copy_(torch.tensor([0, 1, t]))
graph.replay()
torch.cuda.synchronize()
got = out.clone()
layer(ops.LEGACY_STREAM)
torch.cuda.synchronize()
assert torch.equal(got, out)
for hnd in (w, rope, att):
    hnd.sync()
print("same")
"""


@gpu
@pytest.mark.parametrize("t,hint", [(6, 6), (50, 64), (100, 128), (700, 0)])
def test_first_calls_of_a_process_are_captured(t, hint):
    """A graph that holds the first call of every operator, replayed on other
    offsets; in a process of its own, whose kernels are not loaded yet."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS % (t, hint)], cwd=root, capture_output=True, text=True,
                       timeout=300, env=dict(os.environ, PYTHONPATH=root))
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]
