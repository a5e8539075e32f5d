"""The stand-alone operators (llm_embed_b200.ops) against their formulas in 64
bits, at the sizes, strides and values where they can go wrong, and their
refusals.

Tolerances, with half steps h = finfo(type).eps / 2 of the result's type:
- quantiser: none, its bytes and scales are defined exactly;
- product: operands are exact, so a result is off by its float32 sums (at most
  one step of 2^-23 of the sum of magnitudes for each of its K + K/128 additions)
  and the rounding to the result's type (h of the value);
- norm and rotation: the sum of squares has 13 roundings (half of that in its
  root), the reciprocal root two steps, the products five: 16 * 2^-24 of a
  value, of a pair's length after the rotation (at most sqrt 2 times the
  largest), so 24 * 2^-24 of the head vector's largest result, 2 more for the
  table, and h of the value;
- differential attention: weights P are rounded to the operands' type (h
  each).  Scores are float32 sums of d products, off by at most d 2^-24 of
  their sum of magnitudes (about 10 here after the division by sqrt d), which
  moves a weight and its map's sum by 2^-14.6 each; the exponent's argument
  and ex2.approx add less than 2^-18.  So both maps' results are off by at
  most (h + 2^-13) of sum_j P_j |v_j|; then the rounding of the result.  The norm divides by the row's root mean square, which scales the
  same error and adds its own part of it (sum over the row).
"""
import ctypes as C
import math
import threading

import numpy as np
import pytest

from llm_embed_b200 import ops
from llm_embed_b200.embed import LE_EINVAL, LlmEmbedError

gpu = pytest.mark.gpu
INIT = 0.8 - 0.6 * math.exp(-1.5)


def T(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def half_step(name):
    import torch
    return torch.finfo(T(name)).eps / 2


def stream():
    import torch
    return torch.cuda.current_stream().cuda_stream or ops.LEGACY_STREAM


def gen(seed):
    import torch
    return torch.Generator("cuda").manual_seed(seed)


# ------------------------------------------------------------- quantiser --

def quantise64(x):
    """The definition, in 64 bits: (values/scale rounded to e4m3, scales [blocks][m])."""
    import torch
    x = x.double()
    m, k = x.shape
    kb = -(-k // 128)
    b = torch.nn.functional.pad(x, (0, kb * 128 - k)).view(m, kb, 128)
    top = b.abs().amax(2)
    _, e = torch.frexp(top)  # top = f 2^e, f in [1/2, 1)
    e = e.to(torch.int64) - 9 + (top > torch.ldexp(torch.full_like(top, 0.875), e)).long()
    e = torch.where(top == 0, torch.zeros_like(e), e.clamp(min=-126))
    s = ((e + 1023) << 52).view(torch.float64)
    s = torch.where(torch.isfinite(top), s, float("nan"))
    u = b / s[:, :, None]
    _, ue = torch.frexp(u.abs().clamp(min=2.0 ** -6))
    step = ((ue.long() - 4 + 1023) << 52).view(torch.float64)
    q = torch.round(u / step) * step
    return q.view(m, kb * 128)[:, :k], s.t()


def same(a, b):
    """Equal values, NaN (a block with an infinity, as fp16 rows may hold) equal to NaN."""
    import torch
    nan = torch.isnan(b)
    return torch.equal(torch.isnan(a), nan) and torch.equal(a[~nan], b[~nan])


def run_quantise(x, name, ldx=0):
    import torch
    m, k = x.shape
    q = torch.full((m + 1, k), 0x55, dtype=torch.uint8, device="cuda")
    s = torch.full((-(-k // 128), m), -7.0, device="cuda")
    ops.f8_quantize_device(x.data_ptr(), name, m, k, q.data_ptr(), s.data_ptr(), ldx=ldx or x.stride(0),
                           stream=stream())
    torch.cuda.synchronize()
    assert (q[m] == 0x55).all()  # the row behind the last
    return q[:m].view(torch.float8_e4m3fn).double(), s.double()


@gpu
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 16), (3, 127), (5, 130), (7, 768), (130, 1000), (33, 4096), (2000, 4096)])
def test_quantise(name, m, k):
    import torch
    x = (torch.randn(m, k, device="cuda", generator=gen(m + k)) * torch.exp(
        4 * torch.randn(m, 1, device="cuda", generator=gen(k)))).to(T(name))
    q, s = run_quantise(x, name)
    rq, rs = quantise64(x)
    assert same(s, rs) and same(q, rq)


@gpu
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad,shift", [(8, 0), (3, 0), (8, 1)])
def test_quantise_strides(name, pad, shift):
    """Rows inside wider ones, aligned and not."""
    import torch
    wide = torch.randn(9, 384 + pad + shift, device="cuda", generator=gen(3)).to(T(name))
    x = wide[:, shift:shift + 384]
    q, s = run_quantise(x, name)
    rq, rs = quantise64(x)
    assert same(s, rs) and same(q, rq)


@gpu
@pytest.mark.parametrize("k", [128, 131])
def test_quantise_borders(k):
    """Largest values at 448 times a power of two and next to it, zeros,
    subnormal and huge values, ties, infinities and NaN."""
    import torch
    rows = []
    for top in (448.0, np.nextafter(np.float32(448), np.float32(1e9)), np.nextafter(np.float32(448), np.float32(0)),
                1.0, 2.0 ** -126, 2.0 ** -140, 3.0e38, 448 * 2.0 ** 100, 448 * 2.0 ** -120, 0.0):
        r = np.float32(top) * np.linspace(-1, 1, k).astype(np.float32)
        r[0] = top
        rows.append(r)
    ties = np.zeros(k, np.float32)  # scale 1: halfway between neighbours
    ties[:6] = [448, 17, 19, 2.0 ** -10, 3 * 2.0 ** -10, -17]
    rows.append(ties)
    for bad in (np.inf, -np.inf, np.nan):
        r = np.ones(k, np.float32)
        r[5] = bad
        rows.append(r)
    x = torch.from_numpy(np.stack(rows)).cuda()
    q, s = run_quantise(x, "f32")
    rq, rs = quantise64(x)
    assert torch.equal(torch.isnan(s), torch.isnan(rs)) and torch.isnan(s).any()
    assert torch.equal(s.nan_to_num(-1), rs.nan_to_num(-1))
    good = ~torch.isnan(rs).any(0)
    assert torch.equal(q[good], rq[good])
    assert torch.isnan(q[:, :128] * s[0][:, None])[torch.isnan(s[0])].all()


@gpu
@pytest.mark.parametrize("n,k", [(1, 16), (130, 272), (256, 768)])
def test_quantise_weight(n, k):
    """from_float: blocks of 128 x 128 by the same rule; read returns them."""
    import torch
    w = torch.randn(n, k, generator=torch.Generator().manual_seed(n)).numpy() * 0.03
    f = ops.F8Weight.from_float(w)
    q, s = f.read()
    f.close()
    nb, kb = s.shape
    assert (nb, kb) == (-(-n // 128), -(-k // 128))
    for i in range(nb):
        for j in range(kb):
            b = torch.from_numpy(w[128 * i:128 * i + 128, 128 * j:128 * j + 128])
            rq, rs = quantise64(torch.nn.functional.pad(b, (0, 128 - b.shape[1], 0, 0)).reshape(1, -1).abs().amax()
                                .view(1, 1))
            assert s[i, j] == rs.item()
            got = torch.from_numpy(q[128 * i:128 * i + 128, 128 * j:128 * j + 128].copy()).view(torch.float8_e4m3fn)
            assert torch.equal(got.float(), (b / s[i, j]).to(torch.float8_e4m3fn).float())


# --------------------------------------------------------------- product --

def make_f8(n, k, seed):
    import torch
    w8 = (100 * torch.randn(n, k, device="cuda", generator=gen(seed))).clamp(-448, 448).to(torch.float8_e4m3fn)
    ws = 0.001 * (0.5 + torch.rand(-(-n // 128), -(-k // 128), device="cuda", generator=gen(seed + 1)))
    return w8, ws


def product64(x, w8, ws):
    """(y, sum of magnitudes) in 64 bits from the quantised x."""
    import torch
    q, s = quantise64(x)
    return product64_q(q, s, w8, ws)


def product64_q(q, s, w8, ws):
    import torch
    n, k = w8.shape
    cols = torch.arange(k, device="cuda") // 128
    a = q * s.t()[:, cols]
    b = w8.double() * ws.double()[torch.arange(n, device="cuda") // 128][:, cols]
    return a @ b.t(), a.abs() @ b.abs().t()


def check_product(y, ref, mag, k, yt):
    import torch
    tol = (k + k // 128 + 4) * 2.0 ** -23 * mag + half_step(yt) * ref.abs() * 1.01 + 1e-30
    tol = tol + (2.0 ** -25 if yt == "f16" else 0)  # half a step of fp16's subnormals
    bad = ((y.double() - ref).abs() > tol)
    assert not bad.any(), (int(bad.sum()), float(((y.double() - ref).abs() / tol).max()))


def run_product(w, x, n, xt, yt, ldy=0, scales=None, m=None, s=None):
    import torch
    m = x.shape[0]
    ldy = ldy or n
    y = torch.full((m + 1, ldy), -3.0, device="cuda", dtype=T(yt))
    work = torch.full((max(16, w.workspace_bytes(m, xt)),), 0x7F, device="cuda", dtype=torch.uint8)
    w.matmul_device(x.data_ptr(), m, y.data_ptr(), xt, yt, ldx=x.stride(0), ldy=ldy,
                    d_x_scales=0 if scales is None else scales.data_ptr(), d_work=work.data_ptr(),
                    work_bytes=work.numel(), stream=s or stream())
    torch.cuda.synchronize()
    assert (y[m] == -3).all() and (y[:, n:] == -3).all()
    return y[:m, :n]


PRODUCTS = [(1, 16, 1), (1, 768, 2304), (2, 144, 17), (7, 128, 130), (8, 4096, 128), (9, 1040, 300), (16, 768, 768),
            (17, 272, 96), (31, 2000, 250), (33, 768, 2304), (64, 256, 129), (65, 768, 1000), (129, 784, 256),
            (300, 1024, 1), (257, 4096, 512), (1000, 768, 2304), (2049, 400, 776)]


@gpu
@pytest.mark.parametrize("m,k,n", PRODUCTS)
@pytest.mark.parametrize("xt,yt", [("f16", "f16"), ("bf16", "bf16"), ("f32", "f32"), ("f32", "bf16"), ("f16", "f32")])
def test_product(m, k, n, xt, yt):
    import torch
    w8, ws = make_f8(n, k, m)
    x = (torch.randn(m, k, device="cuda", generator=gen(k)) * torch.exp(
        torch.randn(m, 1, device="cuda", generator=gen(n)))).to(T(xt))
    w = ops.F8Weight(w8.data_ptr(), ws.data_ptr(), n, k)
    ref, mag = product64(x, w8, ws)
    check_product(run_product(w, x, n, xt, yt), ref, mag, k, yt)
    w.sync()
    w.close()


@gpu
@pytest.mark.parametrize("m", [1, 20, 40, 200, 700])
def test_product_of_quantised(m):
    """e4m3 activations with their scales give the bits of the float path's;
    the scales need not be powers of two."""
    import torch
    n, k = 384, 784
    w8, ws = make_f8(n, k, m)
    w = ops.F8Weight(w8.data_ptr(), ws.data_ptr(), n, k)
    x = torch.randn(m, k, device="cuda", generator=gen(m), dtype=torch.float32)
    q = torch.empty(m, k, device="cuda", dtype=torch.uint8)
    s = torch.empty(-(-k // 128), m, device="cuda")
    ops.f8_quantize_device(x.data_ptr(), "f32", m, k, q.data_ptr(), s.data_ptr(), stream=stream())
    assert torch.equal(run_product(w, x, n, "f32", "f32"), run_product(w, q, n, "e4m3", "f32", scales=s))
    s *= 1.3
    ref, mag = product64_q(q.view(torch.float8_e4m3fn).double(), s.double(), w8, ws)
    check_product(run_product(w, q, n, "e4m3", "bf16", scales=s), ref, mag, k, "bf16")
    w.close()


@gpu
@pytest.mark.parametrize("m", [5, 33, 300])
@pytest.mark.parametrize("xt", ["f32", "f16"])
@pytest.mark.parametrize("pad,shift,ldy", [(8, 0, 136), (3, 1, 131), (0, 0, 257)])
def test_product_strides(m, xt, pad, shift, ldy):
    import torch
    n, k = 130, 400
    w8, ws = make_f8(n, k, m)
    w = ops.F8Weight(w8.data_ptr(), ws.data_ptr(), n, k)
    x = torch.randn(m, k + pad + shift, device="cuda", generator=gen(m)).to(T(xt))[:, shift:shift + k]
    ref, mag = product64(x, w8, ws)
    check_product(run_product(w, x, n, xt, "f16", ldy=max(ldy, n)), ref, mag, k, "f16")
    w.close()


@gpu
@pytest.mark.parametrize("m", [6, 40, 300])
def test_product_nan_stays_in_its_row(m):
    import torch
    n, k = 256, 512
    w8, ws = make_f8(n, k, m)
    w = ops.F8Weight(w8.data_ptr(), ws.data_ptr(), n, k)
    x = torch.randn(m, k, device="cuda", generator=gen(m))
    x[1, 300] = float("nan")
    x[m - 2, 2] = float("inf")
    x[3] = 0
    y = run_product(w, x, n, "f32", "f32")
    bad = torch.isnan(y)
    assert bad[1].all() and bad[m - 2].all() and int(bad.sum()) == 2 * n
    assert (y[3] == 0).all()
    w.close()


@gpu
def test_product_numpy_weight_and_repeat():
    """The same call twice gives the same bits; a weight from host arrays."""
    import torch
    n, k = 520, 1296
    w8, ws = make_f8(n, k, 5)
    a = ops.F8Weight(w8.data_ptr(), ws.data_ptr(), n, k)
    b = ops.F8Weight(w8.view(torch.uint8).cpu().numpy(), ws.cpu().numpy(), n, k)
    q, s = b.read()
    assert np.array_equal(q, w8.view(torch.uint8).cpu().numpy()) and np.array_equal(s, ws.cpu().numpy())
    for m in (3, 30, 500):
        x = torch.randn(m, k, device="cuda", generator=gen(m)).half()
        y = run_product(a, x, n, "f16", "f32")
        for _ in range(3):
            assert torch.equal(run_product(b, x, n, "f16", "f32"), y)
    a.close()
    b.close()


@gpu
@pytest.mark.parametrize("m", [4, 600])
def test_product_two_streams_and_a_graph(m):
    """Two streams at once with workspaces of their own, and a captured call
    replayed on new inputs."""
    import torch
    n, k = 768, 768
    w8, ws = make_f8(n, k, 9)
    w = ops.F8Weight(w8.data_ptr(), ws.data_ptr(), n, k)
    xs = [torch.randn(m, k, device="cuda", generator=gen(i)).half() for i in range(2)]
    want = [run_product(w, x, n, "f16", "f16").clone() for x in xs]
    size = w.workspace_bytes(m, "f16")
    works = [torch.empty(size, device="cuda", dtype=torch.uint8) for _ in range(2)]
    ys = [torch.empty(m, n, device="cuda", dtype=torch.float16) for _ in range(2)]
    sts = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            w.matmul_device(xs[i].data_ptr(), m, ys[i].data_ptr(), d_work=works[i].data_ptr(), work_bytes=size,
                            stream=sts[i].cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(ys[0], want[0]) and torch.equal(ys[1], want[1])
    x, y = torch.zeros_like(xs[0]), torch.zeros_like(ys[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w.matmul_device(x.data_ptr(), m, y.data_ptr(), d_work=works[0].data_ptr(), work_bytes=size, stream=stream())
    for i in (0, 1, 0):
        x.copy_(xs[i])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[i])
    w.sync()
    del g
    w.close()


def expect_einval(call):
    with pytest.raises(LlmEmbedError) as e:
        call()
    assert e.value.code == LE_EINVAL, str(e.value)


def test_refusals_without_a_device():
    """Argument checks that come before any device work."""
    w = np.zeros((16, 16), np.uint8)
    s = np.ones((1, 1), np.float32)
    expect_einval(lambda: ops.F8Weight(w, s, 16, 24))
    expect_einval(lambda: ops.F8Weight(w.ctypes.data, s.ctypes.data, 16, 24))
    expect_einval(lambda: ops.F8Weight(w.ctypes.data, s.ctypes.data, 0, 16))
    expect_einval(lambda: ops.F8Weight(0, s.ctypes.data, 16, 16))
    expect_einval(lambda: ops.F8Weight(w.ctypes.data, 0, 16, 16))
    expect_einval(lambda: ops.F8Weight.from_float(np.zeros((4, 8), np.float32)))
    expect_einval(lambda: ops.f8_quantize_device(0, "f16", 1, 16, 0, 0))
    expect_einval(lambda: ops.f8_quantize_device(64, "f64", 1, 16, 64, 64))
    expect_einval(lambda: ops.f8_quantize_device(64, "e4m3", 1, 16, 64, 64))
    expect_einval(lambda: ops.f8_quantize_device(64, "f16", -1, 16, 64, 64))
    expect_einval(lambda: ops.f8_quantize_device(64, "f16", 1, 0, 64, 64))
    expect_einval(lambda: ops.f8_quantize_device(64, "f16", 1, 16, 64, 64, ldx=8))
    expect_einval(lambda: ops.f8_quantize_device(65, "f16", 1, 16, 64, 64))
    for args in ((0, 64, 1e4, "half"), (16, 63, 1e4, "half"), (16, 258, 1e4, "half"), (16, -2, 1e4, "half"),
                 (16, 64, 0.0, "half"), (16, 64, float("inf"), "half"), (16, 64, 1e4, "pairs")):
        expect_einval(lambda: ops.Rope(*args))
    lam = np.zeros((4, 64), np.float32)
    expect_einval(lambda: ops.DiffAttention(6, 4, 64, lam, 0.8))
    expect_einval(lambda: ops.DiffAttention(0, 1, 64, lam, 0.8))
    expect_einval(lambda: ops.DiffAttention(6, 6, 48, np.zeros((4, 48), np.float32), 0.8))
    expect_einval(lambda: ops.DiffAttention(6, 6, 64, lam[:3], 0.8))
    expect_einval(lambda: ops.DiffAttention(6, 6, 64, lam, 0.8, np.ones(64, np.float32)))
    expect_einval(lambda: ops.DiffAttention(6, 6, 64, lam, 0.8, None, -1.0))


@gpu
def test_product_refusals():
    import torch
    w8, ws = make_f8(32, 64, 1)
    w = ops.F8Weight(w8.data_ptr(), ws.data_ptr(), 32, 64)
    x = torch.zeros(64, 64, device="cuda", dtype=torch.float16)
    y = torch.zeros(64, 32, device="cuda", dtype=torch.float16)
    wk = torch.zeros(1 << 16, device="cuda", dtype=torch.uint8)
    a = dict(d_work=wk.data_ptr(), work_bytes=wk.numel())
    xp, yp = x.data_ptr(), y.data_ptr()
    expect_einval(lambda: w.matmul_device(xp, 64, yp))  # no workspace
    expect_einval(lambda: w.matmul_device(xp, 64, yp, d_work=wk.data_ptr(), work_bytes=100))
    expect_einval(lambda: w.matmul_device(xp, 64, yp, d_work=wk.data_ptr() + 4, work_bytes=1 << 15))
    expect_einval(lambda: w.matmul_device(xp, -1, yp, **a))
    expect_einval(lambda: w.matmul_device(0, 64, yp, **a))
    expect_einval(lambda: w.matmul_device(xp, 64, 0, **a))
    expect_einval(lambda: w.matmul_device(xp, 64, yp, "f16", "e4m3", **a))
    expect_einval(lambda: w.matmul_device(xp, 64, yp, "e4m3", "f16", **a))  # no scales
    expect_einval(lambda: w.matmul_device(xp + 1, 64, yp, **a))
    expect_einval(lambda: w.matmul_device(xp, 64, yp, ldx=63, **a))
    expect_einval(lambda: w.matmul_device(xp, 64, yp, ldy=31, **a))
    expect_einval(lambda: w.matmul_device(xp + 8, 4, yp, "e4m3", "f16", d_x_scales=wk.data_ptr(), **a))
    expect_einval(lambda: w.matmul_device(xp, 4, yp, "e4m3", "f16", ldx=72, d_x_scales=wk.data_ptr(), **a))
    w.matmul_device(0, 0, 0)  # no rows: nothing to do
    w.close()


# ----------------------------------------------------- norm and rotation --

def qk64(x, heads, d, rot, pairing, w, pos, base, eps):
    import torch
    u = x.double().reshape(x.shape[0], heads, d)
    u = u / (u.square().mean(2, keepdim=True) + eps).sqrt()
    if w is not None:
        u = u * w.double()
    if rot:
        i = torch.arange(0, rot, 2, device=x.device, dtype=torch.float64)
        a = (pos.double()[:, None] * base ** (-i / rot))[:, None]
        r = u[:, :, :rot]
        p, q = (r[..., 0::2], r[..., 1::2]) if pairing == "interleaved" else (r[..., :rot // 2], r[..., rot // 2:])
        p, q = p * a.cos() - q * a.sin(), p * a.sin() + q * a.cos()
        r = torch.stack([p, q], 3).flatten(2) if pairing == "interleaved" else torch.cat([p, q], 2)
        u = torch.cat([r, u[:, :, rot:]], 2)
    return u


def check_qk(got, ref, name):
    # As derived above; fp16's subnormals have steps of 2^-24.
    tol = (24 + 2) * 2.0 ** -24 * ref.abs().amax(2, keepdim=True) + half_step(name) * ref.abs() * 1.01
    tol = tol + (2.0 ** -25 if name == "f16" else 1e-40)
    err = (got.double().reshape(ref.shape) - ref).abs()
    assert (err <= tol).all(), float((err / tol).max())


@gpu
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("t,hq,hk,d,rot,pairing", [
    (1, 1, 1, 64, 64, "interleaved"), (8, 12, 12, 64, 64, "interleaved"), (5, 12, 12, 64, 64, "half"),
    (129, 8, 2, 128, 128, "half"), (33, 3, 1, 96, 96, "half"), (33, 3, 1, 96, 32, "interleaved"),
    (17, 5, 1, 256, 128, "half"), (21, 1, 7, 32, 16, "interleaved"), (64, 4, 4, 80, 32, "half"),
    (9, 2, 3, 72, 24, "half"), (9, 2, 3, 50, 50, "interleaved"), (7, 1, 1, 7, 4, "half"), (3, 2, 2, 1, 0, "half"),
    (40, 4, 0, 64, 0, "half"), (40, 0, 4, 64, 64, "half"), (20011, 3, 2, 64, 64, "interleaved"),
    (9001, 2, 5, 256, 256, "half")])
def test_qk_norm(name, t, hq, hk, d, rot, pairing):
    import torch
    g = gen(t + d)
    x = [torch.randn(t, max(h, 1) * d, device="cuda", generator=g) * torch.exp(
        2 * torch.randn(t, 1, device="cuda", generator=g)) for h in (hq, hk)]
    q, k = (v.to(T(name)) for v in x)
    qw, kw = (1 + 0.3 * torch.randn(d, device="cuda", generator=g) for _ in range(2))
    pos = torch.randint(0, 9000, (t,), device="cuda", generator=g, dtype=torch.int32)
    qo, ko = torch.full_like(q, 9), torch.full_like(k, 9)
    r = ops.Rope(9000, rot, 10000.0, pairing)
    r.qk_norm_device(name, t, hq, hk, d, q.data_ptr(), k.data_ptr(), pos.data_ptr(), qo.data_ptr(), ko.data_ptr(),
                     d_q_weight=qw.data_ptr(), eps=1e-6, stream=stream(), d_k_weight=0 if t % 2 else kw.data_ptr())
    r.sync()
    if hq:
        check_qk(qo, qk64(q, hq, d, rot, pairing, qw, pos, 10000.0, 1e-6), name)
    else:
        assert (qo == 9).all()
    if hk:
        check_qk(ko, qk64(k, hk, d, rot, pairing, None if t % 2 else kw, pos, 10000.0, 1e-6), name)
    else:
        assert (ko == 9).all()
    r.close()


@gpu
@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("pairing", ["interleaved", "half"])
def test_qk_norm_in_place_inside_packed_rows(name, shift, pairing):
    """Queries and keys of a packed QKV row, in place; the values and the rows
    behind the last token stay as they were."""
    import torch
    t, h, d = 77, 12, 64
    rows = torch.randn(t + 2, 3 * h * d + shift, device="cuda", generator=gen(1)).to(T(name))
    before = rows.clone()
    pos = torch.arange(t, device="cuda", dtype=torch.int32)
    q, k = rows[:t, shift:shift + h * d], rows[:t, shift + h * d:shift + 2 * h * d]
    refs = [qk64(v, h, d, d, pairing, None, pos, 1000.0, 1e-5) for v in (q, k)]
    r = ops.Rope(t, d, 1000.0, pairing)
    ld = rows.stride(0)
    r.qk_norm_device(name, t, h, h, d, q.data_ptr(), k.data_ptr(), pos.data_ptr(), q.data_ptr(), k.data_ptr(),
                     q_stride=ld, k_stride=ld, q_out_stride=ld, k_out_stride=ld, eps=1e-5, stream=stream())
    r.sync()
    check_qk(q, refs[0], name)
    check_qk(k, refs[1], name)
    assert torch.equal(rows[t:], before[t:]) and torch.equal(rows[:, shift + 2 * h * d:], before[:, shift + 2 * h * d:])
    r.close()


@gpu
def test_qk_norm_far_positions():
    """Angles at position 2^20 (float32 angles would be off by 0.06)."""
    import torch
    t, d = 64, 64
    q = torch.randn(t, d, device="cuda", generator=gen(2))
    pos = (2 ** 20 - 1 - 977 * torch.arange(t, device="cuda")).to(torch.int32)
    out = torch.empty_like(q)
    r = ops.Rope(2 ** 20, d, 10000.0, "half")
    r.qk_norm_device("f32", t, 1, 0, d, q.data_ptr(), 0, pos.data_ptr(), out.data_ptr(), 0, stream=stream())
    r.sync()
    check_qk(out, qk64(q, 1, d, d, "half", None, pos, 10000.0, 1e-6), "f32")
    r.close()


@gpu
@pytest.mark.parametrize("d", [64, 50])
def test_qk_norm_bad_positions_are_reported(d):
    """A position outside the table leaves its token's rows unwritten, the
    others right; sync reports it once."""
    import torch
    t, h = 9, 2
    q = torch.randn(t, h * d, device="cuda", generator=gen(3))
    pos = torch.arange(t, device="cuda", dtype=torch.int32)
    pos[2], pos[7] = -1, 16
    out = torch.full_like(q, 5)
    r = ops.Rope(16, d, 10000.0, "interleaved")
    r.qk_norm_device("f32", t, h, 0, d, q.data_ptr(), 0, pos.data_ptr(), out.data_ptr(), 0, stream=stream())
    with pytest.raises(LlmEmbedError) as e:
        r.sync()
    assert e.value.code == -3
    r.sync()
    ok = torch.tensor([i not in (2, 7) for i in range(t)], device="cuda")
    assert (out[~ok] == 5).all()
    check_qk(out[ok], qk64(q[ok], h, d, d, "interleaved", None, pos[ok], 10000.0, 1e-6), "f32")
    r.close()


@gpu
def test_qk_norm_zero_and_infinite_heads():
    import torch
    t, d = 3, 64
    q = torch.randn(t, 2 * d, device="cuda", generator=gen(4))
    q[0, :d] = 0
    q[1, 5] = float("nan")
    pos = torch.zeros(t, device="cuda", dtype=torch.int32)
    out = torch.empty_like(q)
    r = ops.Rope(4, d)
    r.qk_norm_device("f32", t, 2, 0, d, q.data_ptr(), 0, pos.data_ptr(), out.data_ptr(), 0, eps=0.1, stream=stream())
    r.sync()
    assert (out[0, :d] == 0).all() and torch.isnan(out[1, :d]).all()
    assert torch.isfinite(out[0, d:]).all() and torch.isfinite(out[1, d:]).all() and torch.isfinite(out[2]).all()
    r.close()


@gpu
def test_qk_norm_refusals():
    import torch
    x = torch.zeros(4, 512, device="cuda", dtype=torch.float16)
    p = torch.zeros(4, device="cuda", dtype=torch.int32)
    r = ops.Rope(8, 64)

    def call(dtype="f16", t=4, hq=2, hk=2, d=64, q=x.data_ptr(), k=x.data_ptr() + 512, pos=p.data_ptr(),
             qo=x.data_ptr(), ko=x.data_ptr() + 512, **kw):
        r.qk_norm_device(dtype, t, hq, hk, d, q, k, pos, qo, ko, stream=stream(), **kw)

    for bad in (dict(dtype="e4m3"), dict(t=-1), dict(hq=-1), dict(hk=70000), dict(d=32), dict(d=257), dict(eps=-1.0),
                dict(eps=float("nan")), dict(q=0), dict(k=0), dict(qo=0), dict(ko=0), dict(pos=0), dict(q=x.data_ptr() + 1),
                dict(q_stride=127), dict(q_stride=512), dict(pos=p.data_ptr() + 2)):
        expect_einval(lambda: call(**bad))
    call(t=0, q=0, k=0, qo=0, ko=0, pos=0)
    r.close()


# ------------------------------------------------- differential attention --

def diff64(q, k, v, offs, h, hkv, d, lam, init, nw, eps):
    """(result, sum_j of both maps' weights times |v_j|, row norm factors) in 64 bits."""
    import torch
    t = q.shape[0]
    out = torch.zeros(t, h, 2 * d, device=q.device, dtype=torch.float64)
    mag = torch.zeros_like(out)
    q, k, v = (x.double().reshape(t, -1, 2 * d) for x in (q, k, v))
    for a, b in zip(offs, offs[1:]):
        for j in range(h):
            g = j // (h // hkv)
            maps = [torch.softmax(q[a:b, j, i * d:i * d + d] @ k[a:b, g, i * d:i * d + d].t() / math.sqrt(d), 1)
                    for i in (0, 1)]
            out[a:b, j] = (maps[0] - lam[j] * maps[1]) @ v[a:b, g]
            mag[a:b, j] = (maps[0] + abs(lam[j]) * maps[1]) @ v[a:b, g].abs()
    if nw is not None:
        f = (1 - init) / (out.square().mean(2, keepdim=True) + eps).sqrt()
        # d(o f)/do: the error of o itself times f, and f's own: o (o . do) / |o|^2
        worst = mag + out.abs() * (out.abs() * mag).sum(2, keepdim=True) / out.square().sum(2, keepdim=True).clamp(
            min=1e-300)
        return out * f * nw.double(), worst * f * nw.double().abs()
    return out, mag


def make_diff(lens, h, hkv, d, name, seed, lead=0, tail=0, sharp=2.0):
    import torch
    offs = (lead + np.concatenate([[0], np.cumsum(lens)])).astype(np.int32)
    t = int(offs[-1]) + tail
    rows = torch.randn(t, (2 * h + 4 * hkv) * d, device="cuda", generator=gen(seed))
    rows[:, :2 * h * d] *= sharp
    rows = rows.to(T(name))
    q, k, v = rows.split([2 * h * d, 2 * hkv * d, 2 * hkv * d], 1)
    return q, k, v, offs, t


def lambdas(h, d, per_head, seed):
    g = np.random.default_rng(seed)
    lam = (0.15 * g.standard_normal((h if per_head else 1, 4, d))).astype(np.float32)
    val = [math.exp(float(l[0].astype(np.float64) @ l[1])) - math.exp(float(l[2].astype(np.float64) @ l[3])) + INIT
           for l in (lam if per_head else [lam[0]] * h)]
    return lam if per_head else lam[0], val


def run_diff(a, q, k, v, offs, t, h, d, name, hint=None, s=None):
    import torch
    out = torch.full((t, 2 * h * d), 7.0, device="cuda", dtype=T(name))
    o = torch.from_numpy(offs).cuda()
    hint = int(np.diff(offs).max()) if hint is None and len(offs) > 1 else hint or 0
    a.run_device(name, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), len(offs) - 1, t, hint, out.data_ptr(),
                 q_stride=q.stride(0), k_stride=k.stride(0), v_stride=v.stride(0), stream=s or stream())
    torch.cuda.synchronize()
    return out


def check_diff(out, ref, mag, name):
    err = (out.double().reshape(ref.shape) - ref).abs()
    tol = (half_step(name) + 2.0 ** -13) * mag + half_step(name) * ref.abs() * 1.01 + 2.0 ** -25
    assert torch_all(err <= tol), float((err / tol).max())


def torch_all(x):
    return bool(x.all())


DIFFS = [([1], 1, 1, 64), ([8], 6, 6, 64), ([8], 12, 4, 32), ([64], 2, 1, 64), ([65], 2, 2, 32), ([127, 128, 129], 3, 3, 64),
         ([1, 0, 5, 0, 0, 17, 63], 2, 2, 64), ([130, 1, 257, 40], 4, 2, 64), ([300, 2, 512], 2, 2, 32),
         ([1000], 2, 1, 64), ([16, 100, 31, 77, 128, 55, 90, 3] * 5, 6, 6, 64), ([513, 640, 1, 200], 2, 2, 64),
         ([2047], 1, 1, 64), ([1] * 200, 2, 2, 64), ([1500, 3], 1, 1, 32)]


@gpu
@pytest.mark.parametrize("lens,h,hkv,d", DIFFS)
@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("norm", [True, False])
def test_diff_attention(lens, h, hkv, d, name, norm):
    import torch
    q, k, v, offs, t = make_diff(lens, h, hkv, d, name, sum(lens) + d)
    per_head = h % 2 == 0
    lam, val = lambdas(h, d, per_head, d)
    nw = (1 + 0.3 * torch.randn(2 * d, generator=torch.Generator().manual_seed(1))) if norm else None
    a = ops.DiffAttention(h, hkv, d, lam, INIT, None if nw is None else nw.numpy(), 1e-5)
    out = run_diff(a, q, k, v, offs, t, h, d, name)
    a.sync()
    ref, mag = diff64(q, k, v, offs.tolist(), h, hkv, d, val, INIT, None if nw is None else nw.cuda(), 1e-5)
    check_diff(out, ref, mag, name)
    # The hint of the longest sequence chooses a kernel, not a result.
    for hint in (0, 1, 100000):
        check_diff(run_diff(a, q, k, v, offs, t, h, d, name, hint), ref, mag, name)
    a.close()


@gpu
@pytest.mark.parametrize("count,lo,hi", [(700, 1, 64), (700, 16, 128), (700, 65, 100), (700, 1, 300), (3000, 0, 9)])
@pytest.mark.parametrize("norm", [True, False])
def test_diff_attention_many_sequences(count, lo, hi, norm):
    """Many tiles per SM, short ones among them: the steps of a tile overlap
    those of the next ones, and twice gives the same bits."""
    import torch
    h, d = 6, 64
    lens = np.random.default_rng(hi).integers(lo, hi + 1, count).tolist()
    q, k, v, offs, t = make_diff(lens, h, h, d, "f16", hi)
    lam, val = lambdas(h, d, True, 3)
    nw = (1 + 0.3 * torch.randn(2 * d, generator=torch.Generator().manual_seed(1))) if norm else None
    a = ops.DiffAttention(h, h, d, lam, INIT, None if nw is None else nw.numpy(), 1e-5)
    for hint in (0, hi):
        out = run_diff(a, q, k, v, offs, t, h, d, "f16", hint)
        for _ in range(3):
            assert torch.equal(out, run_diff(a, q, k, v, offs, t, h, d, "f16", hint))
        a.sync()
        part = torch.arange(0, count, 23).tolist()
        for s in part:
            x, y = int(offs[s]), int(offs[s + 1])
            if x == y:
                continue
            ref, mag = diff64(q[x:y], k[x:y], v[x:y], [0, y - x], h, h, d, val, INIT, None if nw is None else nw.cuda(), 1e-5)
            check_diff(out[x:y], ref, mag, "f16")
    a.close()


@gpu
@pytest.mark.parametrize("lens", [[9001, 300, 4097], [16385]])
@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("sharp", [0.5, 3.0])
def test_diff_attention_long(lens, name, sharp):
    """Thousands of keys, from nearly equal weights to a few that count."""
    import torch
    h, d = 2, 64
    q, k, v, offs, t = make_diff(lens, h, 1, d, name, 11, sharp=sharp)
    lam, val = lambdas(h, d, True, 3)
    nw = torch.linspace(0.5, 1.5, 2 * d)
    a = ops.DiffAttention(h, 1, d, lam, INIT, nw.numpy(), 1e-5)
    out = run_diff(a, q, k, v, offs, t, h, d, name)
    a.sync()
    ref, mag = diff64(q, k, v, offs.tolist(), h, 1, d, val, INIT, nw.cuda(), 1e-5)
    check_diff(out, ref, mag, name)
    a.close()


@gpu
@pytest.mark.parametrize("lens", [[5], [60, 70], [200, 130], [600]])
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_diff_attention_ignores_other_rows(lens, name):
    """Rows before the first and behind the last sequence hold NaN and
    infinities: neither read into a result nor written; and a sequence of NaN
    values does not reach its neighbours."""
    import torch
    h, d = 2, 64
    q, k, v, offs, t = make_diff([*lens, 33, *lens], h, h, d, name, 4, lead=3, tail=150)
    lam, val = lambdas(h, d, False, 2)
    a = ops.DiffAttention(h, h, d, lam, INIT, None)
    mid = slice(int(offs[len(lens)]), int(offs[len(lens) + 1]))
    for x in (q, k, v):
        x[:3], x[int(offs[-1]):] = float("nan"), float("inf")
        x[mid] = float("nan")
    out = run_diff(a, q, k, v, offs, t, h, d, name)
    a.sync()
    assert (out[:3] == 7).all() and (out[int(offs[-1]):] == 7).all() and torch.isnan(out[mid]).all()
    ref, mag = diff64(q, k, v, offs.tolist(), h, h, d, val, INIT, None, 0)
    keep = torch.ones(t, dtype=torch.bool, device="cuda")
    keep[:3] = keep[int(offs[-1]):] = keep[mid] = False
    check_diff(out[keep], ref[keep], mag[keep], name)
    a.close()


@gpu
@pytest.mark.parametrize("lens", [[40, 90], [700]])
def test_diff_attention_sharp_and_growing_scores(lens):
    """Maxima that grow along the keys (every block rescales), scores far
    apart, and equal scores."""
    import torch
    h, d = 2, 64
    q, k, v, offs, t = make_diff(lens, h, h, d, "f16", 9, sharp=1.0)
    at = torch.cat([torch.arange(n, device="cuda") for n in lens])
    q[:, 0], q[:, d] = 8, 0
    k[:, 0] = (at * 0.25).half()  # head 0, map 1: the score grows by 0.25 per key
    k[:, 2 * d:3 * d] = 0         # head 1, map 1: every score is 0
    lam, val = lambdas(h, d, True, 2)
    a = ops.DiffAttention(h, h, d, lam, INIT, None)
    out = run_diff(a, q, k, v, offs, t, h, d, "f16")
    ref, mag = diff64(q, k, v, offs.tolist(), h, h, d, val, INIT, None, 0)
    # Scores reach 0.25 * 700 = 175: their float32 sums are off by up to
    # 64 * 2^-24 * 175 = 2^-10.5, which moves a weight and the sum as much.
    err = (out.double().reshape(ref.shape) - ref).abs()
    tol = (half_step("f16") + 2.0 ** -9.5) * mag + half_step("f16") * ref.abs() * 1.01 + 2.0 ** -25
    assert torch_all(err <= tol), float((err / tol).max())
    a.close()


@gpu
def test_diff_attention_bad_offsets_are_reported():
    """Offsets that leave the rows or descend: an error from sync, no access
    outside, nothing written behind the rows."""
    import torch
    h, d, t = 2, 64, 100
    q, k, v, _, _ = make_diff([t], h, h, d, "f16", 1)
    lam, _ = lambdas(h, d, False, 2)
    a = ops.DiffAttention(h, h, d, lam, INIT, None)
    for bad in ([0, 50, 101], [0, 60, 40, 100], [-5, 50, 100], [0, 2 ** 30, 100], [0, -(2 ** 31), 100]):
        run_diff(a, q, k, v, np.array(bad, np.int32), t, h, d, "f16", hint=100)
        with pytest.raises(LlmEmbedError) as e:
            a.sync()
        assert e.value.code == -3
        a.sync()
    good = np.array([0, 50, 100], np.int32)
    first = run_diff(a, q, k, v, good, t, h, d, "f16")
    assert torch.equal(first, run_diff(a, q, k, v, good, t, h, d, "f16"))
    a.sync()
    a.close()


@gpu
def test_diff_attention_refusals():
    import torch
    x = torch.zeros(8, 512, device="cuda", dtype=torch.float16)
    o = torch.zeros(8, device="cuda", dtype=torch.int32)
    a = ops.DiffAttention(2, 1, 64, np.zeros((4, 64), np.float32), INIT)
    p = x.data_ptr()

    def call(dtype="f16", q=p, k=p, v=p, offs=o.data_ptr(), nseq=1, t=2, hint=0, out=p + 4096, **kw):
        a.run_device(dtype, q, k, v, offs, nseq, t, hint, out, stream=stream(), **kw)

    for bad in (dict(dtype="f32"), dict(q=0), dict(k=0), dict(v=0), dict(offs=0), dict(out=0), dict(nseq=-1), dict(t=-1),
                dict(hint=-1), dict(q=p + 8), dict(out=p + 2), dict(q_stride=255), dict(q_stride=260),
                dict(k_stride=120), dict(v_stride=100), dict(out_stride=248), dict(offs=o.data_ptr() + 1)):
        expect_einval(lambda: call(**bad))
    call(nseq=0, q=0, k=0, v=0, out=0, offs=0)
    call(t=0, q=0, k=0, v=0, out=0, offs=0)
    a.close()


# ---------------------------------------------------------------- together --

@gpu
@pytest.mark.parametrize("lens", [[8], [16, 100, 31, 128], [300, 40]])
def test_attention_layer(lens):
    """A layer's attention as it is used: e4m3 QKV projection, norm and
    rotation of the heads in place, differential attention, e4m3 output
    projection; captured in a graph and replayed, on a stream of its own, from
    several threads with handles shared."""
    import torch
    H, h, d = 768, 6, 64
    offs = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    t = int(offs[-1])
    d_offs = torch.from_numpy(offs).cuda()
    pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]).cuda()
    w1, s1 = make_f8(3 * H, H, 1)
    w2, s2 = make_f8(H, H, 3)
    qkv_w = ops.F8Weight(w1.data_ptr(), s1.data_ptr(), 3 * H, H)
    out_w = ops.F8Weight(w2.data_ptr(), s2.data_ptr(), H, H)
    rope = ops.Rope(512, d)
    lam, val = lambdas(h, d, False, 7)
    nw = np.linspace(0.5, 1.5, 2 * d).astype(np.float32)
    attn = ops.DiffAttention(h, h, d, lam, INIT, nw)

    class Buffers:
        def __init__(self):
            self.x = torch.zeros(t, H, device="cuda", dtype=torch.float16)
            self.qkv = torch.zeros(t, 3 * H, device="cuda", dtype=torch.float16)
            self.att = torch.zeros(t, H, device="cuda", dtype=torch.float16)
            self.y = torch.zeros(t, H, device="cuda")
            self.work = torch.empty(qkv_w.workspace_bytes(t, "f16"), device="cuda", dtype=torch.uint8)

    def layer(b, s):
        wk = dict(d_work=b.work.data_ptr(), work_bytes=b.work.numel(), stream=s)
        qkv_w.matmul_device(b.x.data_ptr(), t, b.qkv.data_ptr(), **wk)
        q, k, v = (b.qkv.data_ptr() + 2 * H * i for i in range(3))
        rope.qk_norm_device("f16", t, 2 * h, 2 * h, d, q, k, pos.data_ptr(), q, k, q_stride=3 * H, k_stride=3 * H,
                            q_out_stride=3 * H, k_out_stride=3 * H, stream=s)
        attn.run_device("f16", q, k, v, d_offs.data_ptr(), len(lens), t, max(lens), b.att.data_ptr(), q_stride=3 * H,
                        k_stride=3 * H, v_stride=3 * H, stream=s)
        out_w.matmul_device(b.att.data_ptr(), t, b.y.data_ptr(), "f16", "f32", **wk)

    def check(b):
        """Each step against its formula on the step's own inputs (the QKV
        rows are overwritten in place, so their product is made again)."""
        qkv = run_product(qkv_w, b.x, 3 * H, "f16", "f16")
        check_product(qkv, *product64(b.x, w1, s1), H, "f16")
        for i in (0, 1):
            check_qk(b.qkv[:, i * H:(i + 1) * H], qk64(qkv[:, i * H:(i + 1) * H], 2 * h, d, d, "interleaved", None, pos,
                                                        10000.0, 1e-6), "f16")
        assert torch.equal(b.qkv[:, 2 * H:], qkv[:, 2 * H:])
        q, k, v = b.qkv.split(H, 1)
        check_diff(b.att, *diff64(q, k, v, offs.tolist(), h, h, d, val, INIT, torch.from_numpy(nw).cuda(), 1e-5), "f16")
        check_product(b.y, *product64(b.att, w2, s2), H, "f32")

    x = torch.randn(t, H, device="cuda", generator=gen(5)).half()
    b = Buffers()
    b.x.copy_(x)
    layer(b, stream())
    torch.cuda.synchronize()
    check(b)
    want = b.y.clone()

    g, c = torch.cuda.CUDAGraph(), Buffers()
    with torch.cuda.graph(g):
        layer(c, stream())
    c.x.copy_(x)
    for _ in range(2):
        c.y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.y, want)

    bufs = [Buffers() for _ in range(3)]
    errs = []

    def work(buf):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                buf.x.copy_(x)
                for _ in range(5):
                    layer(buf, s.cuda_stream)
                s.synchronize()
        except Exception as e:  # noqa: BLE001
            errs.append(repr(e))

    torch.cuda.synchronize()
    th = [threading.Thread(target=work, args=(bf,)) for bf in bufs]
    for i in th:
        i.start()
    for i in th:
        i.join()
    assert not errs, errs
    assert all(torch.equal(bf.y, want) for bf in bufs)
    for hnd in (qkv_w, out_w, rope, attn):
        hnd.sync()
    del g
    for hnd in (qkv_w, out_w, rope, attn):
        hnd.close()


@gpu
@pytest.mark.parametrize("heads", [1, 16])
@pytest.mark.parametrize("count", [900, 1500])
def test_diff_attention_mostly_empty_sequences(heads, count):
    """Tiles without rows among short ones: a CTA asks for its next tile again
    and again with nothing published between, several heads of one lookup."""
    import torch
    d = 64
    lens = [(s % 7 == 3) * (1 + s % 90) for s in range(count)]
    q, k, v, offs, t = make_diff(lens, heads, heads, d, "f16", count)
    lam, val = lambdas(heads, d, True, 3)
    a = ops.DiffAttention(heads, heads, d, lam, INIT, None)
    out = run_diff(a, q, k, v, offs, t, heads, d, "f16", 0)
    a.sync()
    for _ in range(5):
        assert torch.equal(out, run_diff(a, q, k, v, offs, t, heads, d, "f16", 0))
    a.sync()
    ref, mag = diff64(q, k, v, offs.tolist(), heads, heads, d, val, INIT, None, 0)
    check_diff(out, ref, mag, "f16")
    a.close()


@gpu
@pytest.mark.parametrize("hint", [0, 1, 100])
@pytest.mark.parametrize("bad", [[0, 300, 200, 400], [0, 300, 401], [-128, 0, 400], [0, 399, 0, 400], [400, 0, 400],
                                 [0, 2 ** 31 - 1, 128, 400], [0] * 50 + [300, 200] + [400] * 50])
def test_diff_attention_bad_offsets_of_any_kernel(bad, hint):
    """Every kernel reports them, also where no tile begins with the sequence
    that descends (the first list: numbers 0, 3 and 3), and writes only rows of
    the batch; the next call is as ever."""
    import torch
    h, d, t = 2, 64, 400
    q, k, v, _, _ = make_diff([t], h, h, d, "f16", 1)
    lam, val = lambdas(h, d, False, 2)
    a = ops.DiffAttention(h, h, d, lam, INIT, None)
    out = torch.full((t + 260, 2 * h * d), 7.0, device="cuda", dtype=torch.float16)
    o = torch.tensor(bad, dtype=torch.int32, device="cuda")
    a.run_device("f16", q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), len(bad) - 1, t, hint,
                 out[130].data_ptr(), q_stride=q.stride(0), k_stride=k.stride(0), v_stride=v.stride(0), stream=stream())
    with pytest.raises(LlmEmbedError) as e:
        a.sync()
    assert e.value.code == -3
    assert (out[:130] == 7).all() and (out[130 + t:] == 7).all()
    good = np.array([0, 250, 400], np.int32)
    ref, mag = diff64(q, k, v, good.tolist(), h, h, d, val, INIT, None, 0)
    check_diff(run_diff(a, q, k, v, good, t, h, d, "f16", hint), ref, mag, "f16")
    a.sync()
    a.close()


def sink_and_small_weights(n, d, name):
    """One head of n keys: key 0 takes nearly all of both maps and has no value,
    the others' weights lie near 2^-20 and 2^-19; and the exact result."""
    import torch
    q = torch.zeros(n, 2 * d, device="cuda")
    k, v = torch.zeros_like(q), torch.randn(n, 2 * d, device="cuda", generator=gen(n)).abs()
    q[:, 0], q[:, d] = 8, 8
    k[0, 0], k[0, d] = math.log(2) * 20 * math.sqrt(d) / 8, math.log(2) * 19 * math.sqrt(d) / 8
    k[1:, 1::2] = 0.1 * torch.randn(n - 1, d, device="cuda", generator=gen(n + 1))
    v[0] = 0
    return [x.to(T(name)) for x in (q, k, v)]


@gpu
@pytest.mark.parametrize("n,hint", [(16, 16), (60, 60), (100, 100), (128, 128), (100, 1), (1000, 1), (1000, 100)])
@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("d", [32, 64])
@pytest.mark.parametrize("norm", [True, False])
def test_diff_attention_small_weights(n, hint, name, d, norm):
    """Weights far below the row's largest keep their half step: the formula's
    tolerance holds where fp16's own range (2^-14) would not give it."""
    q, k, v = sink_and_small_weights(n, d, name)
    offs = np.array([0, n] + [n] * (n // 8), np.int32)  # short on average
    nw = np.linspace(0.5, 1.5, 2 * d).astype(np.float32) if norm else None
    lam, val = lambdas(1, d, True, 2)
    a = ops.DiffAttention(1, 1, d, lam, INIT, nw, 1e-20)
    import torch
    ref, mag = diff64(q, k, v, offs.tolist(), 1, 1, d, val, INIT, None if nw is None else torch.from_numpy(nw).cuda(), 1e-20)
    out = run_diff(a, q, k, v, offs, n, 1, d, name, hint)
    a.sync()
    # Scores reach 20 log 2 = 14: their sums have at most two terms, off by
    # 2^-24 of 14, which check_diff's 2^-13 covers.
    check_diff(out, ref, mag, name)
    a.close()


@gpu
@pytest.mark.parametrize("n,hint", [(9, 9), (60, 60), (100, 100), (300, 1)])
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_diff_attention_large_lambda(n, hint, name):
    """A lambda past fp16's largest value: the weights' difference stays in range."""
    import torch
    h, d = 2, 64
    q, k, v, offs, t = make_diff([n] + [0] * n, h, h, d, name, n)
    lam = np.zeros((4, d), np.float32)
    lam[0, 0], lam[1, 0] = 4, 3  # exp(12) = 162755
    val = [math.exp(12.0) - 1 + INIT] * h
    nw = np.ones(2 * d, np.float32)
    a = ops.DiffAttention(h, h, d, lam, INIT, nw, 1e-5)
    ref, mag = diff64(q, k, v, offs.tolist(), h, h, d, val, INIT, torch.from_numpy(nw).cuda(), 1e-5)
    out = run_diff(a, q, k, v, offs, t, h, d, name, hint)
    a.sync()
    assert torch.isfinite(ref).all()
    check_diff(out, ref, mag, name)
    a.close()


@gpu
@pytest.mark.parametrize("hint", [0, 1])
def test_diff_attention_flat_rows_of_many_keys(hint):
    """Equal scores over 65536 keys: (1 - lambda) times the mean value, with
    weights of 5e-6 (85.47 of fp16's smallest steps) where they are divided
    by their sums first."""
    import torch
    n, d = 65536, 32
    q = torch.zeros(n, 2 * d, device="cuda", dtype=torch.float16)
    k, v = torch.ones_like(q), (1 + 0.25 * torch.randn(n, 2 * d, device="cuda", generator=gen(1))).half()
    a = ops.DiffAttention(1, 1, d, np.zeros((4, d), np.float32), INIT, None)
    out = run_diff(a, q, k, v, np.array([0, n], np.int32), n, 1, d, "f16", hint)
    a.sync()
    mean, mag = v.double().mean(0), v.double().abs().mean(0)
    ref = ((1 - INIT) * mean).expand(n, -1)
    check_diff(out, ref, ((1 + INIT) * mag).expand(n, -1), "f16")
    a.close()


@gpu
@pytest.mark.parametrize("n", [16, 100, 1000, 5000])
@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("d", [32, 64])
def test_diff_attention_small_weights_in_tiles(n, name, d):
    """test_diff_attention_small_weights for the tiles of longer texts."""
    q, k, v = sink_and_small_weights(n, d, name)
    offs = np.array([0, n], np.int32)
    lam, val = lambdas(1, d, True, 2)
    a = ops.DiffAttention(1, 1, d, lam, INIT, None)
    ref, mag = diff64(q, k, v, [0, n], 1, 1, d, val, INIT, None, 0)
    out = run_diff(a, q, k, v, offs, n, 1, d, name, 0)
    a.sync()
    check_diff(out, ref, mag, name)
    a.close()


@gpu
def test_diff_attention_tiles_largest_weights():
    """fp16 weights past the maximum they refer to: scores that grow by less
    than what moves it, up to 2^8 times the first block's."""
    import torch
    n, d = 640, 64
    q = torch.zeros(n, 2 * d, device="cuda")
    k, v = torch.zeros_like(q), torch.randn(n, 2 * d, device="cuda", generator=gen(3))
    q[:, 0], q[:, d] = 8, 8
    k[:, 0] = torch.arange(n, device="cuda") // 64 * 0.61  # 9 * 0.61 = 5.49, 2^7.92
    k[:, d] = 5.5 * (torch.arange(n, device="cuda") >= 64)
    q, k, v = q.half(), k.half(), v.half()
    lam, val = lambdas(1, d, True, 2)
    a = ops.DiffAttention(1, 1, d, lam, INIT, None)
    ref, mag = diff64(q, k, v, [0, n], 1, 1, d, val, INIT, None, 0)
    out = run_diff(a, q, k, v, np.array([0, n], np.int32), n, 1, d, "f16", 0)
    a.sync()
    check_diff(out, ref, mag, "f16")
    a.close()


# ----------------------------------------------------------------- streams --

def test_operators_share_one_default_stream():
    """One call's result is the next one's input: without a stream of the
    caller's all of them go to the same."""
    import inspect
    calls = (ops.f8_quantize_device, ops.F8Weight.matmul_device, ops.Rope.qk_norm_device, ops.DiffAttention.run_device)
    assert [inspect.signature(c).parameters["stream"].default for c in calls] == [ops.LEGACY_STREAM] * 4


@gpu
def test_default_streams_are_ordered():
    """Quantiser, product, head norm and attention without a stream argument,
    behind work on the legacy stream that takes a while."""
    import torch
    t, h, d = 40, 2, 64
    W = 2 * h * d
    w8, ws = make_f8(3 * W, W, 1)
    w = ops.F8Weight(w8.data_ptr(), ws.data_ptr(), 3 * W, W)
    rope = ops.Rope(t, d)
    a = ops.DiffAttention(h, h, d, np.zeros((4, d), np.float32), INIT)
    pos = torch.arange(t, device="cuda", dtype=torch.int32)
    offs = torch.tensor([0, t], device="cuda", dtype=torch.int32)
    x = torch.randn(t, W, device="cuda", generator=gen(2)).half()

    def layer(**kw):
        q, s = torch.zeros(t, W, device="cuda", dtype=torch.uint8), torch.zeros(-(-W // 128), t, device="cuda")
        qkv, out = (torch.zeros(t, n, device="cuda", dtype=torch.float16) for n in (3 * W, W))
        torch.cuda.synchronize()
        torch.cuda._sleep(20_000_000)  # 10 ms on the legacy stream
        ops.f8_quantize_device(x.data_ptr(), "f16", t, W, q.data_ptr(), s.data_ptr(), **kw)
        w.matmul_device(q.data_ptr(), t, qkv.data_ptr(), "e4m3", "f16", d_x_scales=s.data_ptr(), **kw)
        pq, pk, pv = (qkv.data_ptr() + 2 * W * i for i in range(3))
        rope.qk_norm_device("f16", t, 2 * h, 2 * h, d, pq, pk, pos.data_ptr(), pq, pk, 3 * W, 3 * W, 3 * W, 3 * W, **kw)
        a.run_device("f16", pq, pk, pv, offs.data_ptr(), 1, t, t, out.data_ptr(), 3 * W, 3 * W, 3 * W, **kw)
        torch.cuda.synchronize()
        return out

    want = layer(stream=ops.LEGACY_STREAM)  # and loads the kernels, which waits for the device
    assert torch.equal(layer(), want)
    for hnd in (w, rope, a):
        hnd.close()


def test_refusals_of_array_types():
    """Scales in another type are refused, not reinterpreted; sizes of zero."""
    w = np.zeros((16, 16), np.uint8)
    for bad in (np.ones((1, 1), np.int32), np.ones((1, 1), np.uint32), np.ones((1, 1), np.float16)):
        expect_einval(lambda: ops.F8Weight(w, bad, 16, 16))
    for bad in (w.astype(np.float32), w.astype(np.uint16), w[:, :8]):
        expect_einval(lambda: ops.F8Weight(bad, np.ones((1, 1), np.float32), 16, 16))
    expect_einval(lambda: ops.DiffAttention(1, 1, 0, np.zeros(0, np.float32), 0.8))
    expect_einval(lambda: ops.DiffAttention(0, 1, 64, np.zeros((0, 4, 64), np.float32), 0.8))


@gpu
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,rot", [(64, 16), (128, 96), (50, 20), (64, 0)])
@pytest.mark.parametrize("pairing", ["interleaved", "half"])
def test_qk_norm_infinite_values(name, d, rot, pairing):
    """A head with an infinity has norm factor 0: the infinity's own column (with
    the rotation, its pair) is NaN, every other one 0, whichever kernel."""
    import torch
    t = 2 * d
    q = torch.randn(t, 2 * d, device="cuda", generator=gen(d)).to(T(name))
    for i in range(d):
        q[i, i] = float("inf")
        q[d + i, i] = float("-inf")
    pos = torch.arange(t, device="cuda", dtype=torch.int32)
    out = torch.empty_like(q)
    r = ops.Rope(t, rot, 10000.0, pairing)
    r.qk_norm_device(name, t, 2, 0, d, q.data_ptr(), 0, pos.data_ptr(), out.data_ptr(), 0, stream=stream())
    r.sync()
    ref = qk64(q, 2, d, rot, pairing, None, pos, 10000.0, 1e-6)
    got = out.double().reshape(ref.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    assert int(torch.isnan(ref[:, 0]).sum()) == 2 * d + 2 * rot and (got[:, 0].nan_to_num(0) == 0).all()
    check_qk(out.reshape(ref.shape)[:, 1:], ref[:, 1:], name)
    r.close()


# ------------------------------------------------- products of many tiles --

# (m, k, n, ldy, tile): more tiles than run at once, several K blocks and a short
# last one, rows that end inside a tile or (4097) fill one CTA of a pair only,
# y rows that TMA stores take and (ldy or n not on 16 bytes) plain ones.
MANY_TILES = [(4225, 784, 2312, 0, 256), (4097, 784, 2296, 0, 256), (4225, 784, 2310, 0, 256),
              (4300, 2064, 2312, 2315, 256), (4352, 16, 2560, 0, 256), (4225, 128, 2311, 0, 256),
              (8000, 128, 1032, 1033, 128),
              (33000, 400, 257, 0, 128), (20000, 784, 72, 0, 128), (19500, 784, 128, 131, 128), (20000, 16, 120, 0, 128),
              (20000, 784, 64, 0, 64), (40000, 400, 40, 0, 64), (40000, 784, 33, 37, 64), (40000, 16, 48, 0, 64)]


def test_products_of_many_tiles_take_the_tile_they_are_for():
    for m, _, n, _, tile in MANY_TILES:
        assert ops.lib().le_f8gemm_tile(m, n) == tile, (m, n)
    assert [ops.lib().le_f8gemm_tile(m, 768) for m in (0, 1, 32, 33)] == [0, 16, 16, 64]


@gpu
@pytest.mark.parametrize("m,k,n,ldy,tile", MANY_TILES)
@pytest.mark.parametrize("xt,yt", [("f16", "f16"), ("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")])
def test_product_many_tiles(m, k, n, ldy, tile, xt, yt):
    """A CTA takes several tiles: stages, accumulators and scales go on from one
    to the next; a NaN stays in its row, and twice gives the same bits."""
    import torch
    w8, ws = make_f8(n, k, m)
    x = (torch.randn(m, k, device="cuda", generator=gen(k)) * torch.exp(
        torch.randn(m, 1, device="cuda", generator=gen(n)))).to(T(xt))
    w = ops.F8Weight(w8.data_ptr(), ws.data_ptr(), n, k)
    ref, mag = product64(x, w8, ws)
    y = run_product(w, x, n, xt, yt, ldy=ldy)
    check_product(y, ref, mag, k, yt)
    assert torch.equal(run_product(w, x, n, xt, yt, ldy=ldy), y)
    x[m - 2, k - 1] = float("nan")
    z = run_product(w, x, n, xt, yt, ldy=ldy)
    bad = torch.isnan(z)
    assert bad[m - 2].all() and int(bad.sum()) == n
    z[m - 2] = y[m - 2]
    assert torch.equal(z, y)
    w.sync()
    w.close()


@gpu
@pytest.mark.parametrize("m,k,n,ldy,tile", [c for c in MANY_TILES if c[1] == 784])
def test_product_of_quantised_many_tiles(m, k, n, ldy, tile):
    """The same with rows that are quantised already, inside wider ones."""
    import torch
    w8, ws = make_f8(n, k, m)
    w = ops.F8Weight(w8.data_ptr(), ws.data_ptr(), n, k)
    x = torch.randn(m, k, device="cuda", generator=gen(m))
    q = torch.empty(m, k, device="cuda", dtype=torch.uint8)
    s = torch.empty(-(-k // 128), m, device="cuda")
    ops.f8_quantize_device(x.data_ptr(), "f32", m, k, q.data_ptr(), s.data_ptr(), stream=stream())
    wide = torch.full((m, k + 32), 0x7F, device="cuda", dtype=torch.uint8)  # NaN behind the rows
    wide[:, :k] = q
    s *= 1.3
    ref, mag = product64_q(q.view(torch.float8_e4m3fn).double(), s.double(), w8, ws)
    check_product(run_product(w, wide[:, :k], n, "e4m3", "f16", ldy=ldy, scales=s), ref, mag, k, "f16")
    w.close()


# ------------------------------------------------ head norms of many heads --

@gpu
@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("pairing", ["interleaved", "half"])
@pytest.mark.parametrize("t,hq,hk,d,rot", [(5003, 8, 8, 64, 64), (5003, 16, 8, 64, 48), (40011, 8, 8, 32, 32),
                                           (20011, 16, 8, 128, 96), (30011, 8, 8, 128, 128), (9001, 16, 8, 256, 256),
                                           (12001, 32, 8, 96, 64), (20011, 12, 9, 128, 96), (40011, 7, 13, 64, 64)])
@pytest.mark.parametrize("packed", [False, True])
def test_qk_norm_many_heads(name, pairing, t, hq, hk, d, rot, packed):
    """Eight and four heads a lane, below and above the size of the L2, into
    other rows and in place inside packed ones with values behind."""
    import torch
    g = gen(t + d)
    wide = (hq + 2 * hk) * d if packed else (hq + hk) * d
    rows = torch.randn(t + 1, wide, device="cuda", generator=g).to(T(name))
    before = rows.clone()
    q, k = rows[:t, :hq * d], rows[:t, hq * d:(hq + hk) * d]
    qw, kw = (1 + 0.3 * torch.randn(d, device="cuda", generator=g) for _ in range(2))
    pos = torch.randint(0, 4000, (t,), device="cuda", generator=g, dtype=torch.int32)
    qo, ko = (q, k) if packed else (torch.full((t, h * d), 9.0, device="cuda", dtype=T(name)) for h in (hq, hk))
    r = ops.Rope(4000, rot, 10000.0, pairing)
    r.qk_norm_device(name, t, hq, hk, d, q.data_ptr(), k.data_ptr(), pos.data_ptr(), qo.data_ptr(), ko.data_ptr(), wide,
                     wide, qo.stride(0), ko.stride(0), qw.data_ptr(), kw.data_ptr(), 1e-6, stream())
    r.sync()
    for got, first, heads, w in ((qo, 0, hq, qw), (ko, hq * d, hk, kw)):
        for a in range(0, t, 8192):  # the reference in 64 bits, a part at a time
            x = before[a:min(t, a + 8192), first:first + heads * d]
            check_qk(got[a:a + 8192].contiguous(), qk64(x, heads, d, rot, pairing, w, pos[a:a + 8192], 10000.0, 1e-6), name)
    assert torch.equal(rows[t], before[t])
    assert torch.equal(rows[:, (hq + hk) * d:], before[:, (hq + hk) * d:])
    if not packed:
        assert torch.equal(rows, before)
    r.close()


@gpu
@pytest.mark.parametrize("m", [300, 4225])
def test_product_behind_a_long_kernel(m):
    """The product's kernel starts while the one before it (seconds on one SM)
    still runs, and waits for it without its own limits running out."""
    import torch
    n, d, k, cols = 51200, 32, 272, 2312
    q = torch.zeros(n, 2 * d, device="cuda", dtype=torch.float16)
    out = torch.empty_like(q)
    offs = torch.tensor([0, n], device="cuda", dtype=torch.int32)
    a = ops.DiffAttention(1, 1, d, np.zeros((4, d), np.float32), INIT, None)
    w8, ws = make_f8(cols, k, m)
    w = ops.F8Weight(w8.data_ptr(), ws.data_ptr(), cols, k)
    x = torch.randn(m, k, device="cuda", generator=gen(m))
    x8, xs = torch.empty(m, k, device="cuda", dtype=torch.uint8), torch.empty(3, m, device="cuda")
    ops.f8_quantize_device(x.data_ptr(), "f32", m, k, x8.data_ptr(), xs.data_ptr(), stream=stream())
    want = run_product(w, x8, cols, "e4m3", "f16", scales=xs)
    y = torch.zeros(m, cols, device="cuda", dtype=torch.float16)
    e = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    torch.cuda.synchronize()
    e[0].record()
    a.run_device("f16", *(3 * [q.data_ptr()]), offs.data_ptr(), 1, n, 1, out.data_ptr(), stream=stream())
    w.matmul_device(x8.data_ptr(), m, y.data_ptr(), "e4m3", "f16", d_x_scales=xs.data_ptr(), stream=stream())
    e[1].record()
    w.sync()
    a.sync()
    assert torch.equal(y, want) and e[0].elapsed_time(e[1]) > 2500  # the limit is 2 s
    w.close()
    a.close()


@gpu
@pytest.mark.parametrize("m", [6, 24, 300, 5000])
@pytest.mark.parametrize("ld", [256, 257])
def test_chain_of_products(m, ld):
    """Each product's result is the next one's input, in the same two buffers
    (every kernel starts while the one before it ends): the bits of the same
    calls one at a time."""
    import torch
    n = 256
    w = ops.F8Weight.from_float(np.random.default_rng(m).standard_normal((n, n)).astype(np.float32) / 16)
    x = torch.randn(m, n, device="cuda", generator=gen(m)).half()
    work = torch.empty(w.workspace_bytes(m, "f16"), device="cuda", dtype=torch.uint8)

    def chain(wait):
        a, b = (torch.zeros(m, ld, device="cuda", dtype=torch.float16) for _ in range(2))
        a[:, :n] = x
        torch.cuda.synchronize()
        for _ in range(60):
            w.matmul_device(a.data_ptr(), m, b.data_ptr(), ldx=ld, ldy=ld, d_work=work.data_ptr(),
                            work_bytes=work.numel(), stream=stream())
            if wait:
                torch.cuda.synchronize()
            a, b = b, a
        torch.cuda.synchronize()
        return a[:, :n].clone()

    want = chain(True)
    assert torch.isfinite(want).all() and float(want.abs().max()) > 0
    for _ in range(5):
        assert torch.equal(chain(False), want)
    w.close()
