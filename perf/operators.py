"""The framework's stand-alone operators as they are measured: the 8-bit product
and its quantiser, the norm and rotation of query and key heads, and
differential attention.  `run` computes each in plain torch, or, where `own`
is true, through llm_embed_b200.ops.

Encoder shapes (768 columns, 12 heads of 64, texts of 16 to 128 tokens, one
text of 8 tokens, texts of 512) are this framework's own model and benchmark;
the 4096-column ones stand for a larger encoder.
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 128


# ------------------------------------------------------------------ cases --

def listed():
    return [
        # One token through a QKV projection: latency of the smallest call.
        f8("product 1x768x2304", 1, 768, 2304, "f16", "f16"),
        # A few short texts at once: the weight's bytes bound it.
        f8("product 24x4096x4096", 24, 4096, 4096, "bf16", "bf16"),
        # A ragged small batch, float32 in and out as le_qgemm_device has it.
        f8("product 333x768x2304", 333, 768, 2304, "f32", "f32"),
        # The largest device call's tokens through an attention projection.
        f8("product 32768x768x2304", 32768, 768, 2304, "f16", "f16"),
        # A larger encoder's projection, tensor-core bound.
        f8("product 8192x4096x4096", 8192, 4096, 4096, "bf16", "bf16"),
        # Activations of one text of 8 tokens, and of a batch of 256 texts.
        quant("quantise 8x768", 8, 768, "f16"),
        quant("quantise 18431x4096", 18431, 4096, "bf16"),
        # One text of 8 tokens, heads inside the packed QKV rows.
        qk("head norm 8 tokens", 8, 12, 12, 64, 64, "interleaved", "f16", True, 2048),
        # A large batch with grouped keys, half-split rotation of part of the head.
        qk("head norm 32767 tokens", 32767, 32, 8, 128, 96, "half", "bf16", False, 8192),
        # One text of 8 tokens; the benchmark's batch of short texts; long texts.
        diff("differential 8 tokens", 1, 8, 8, 6, 6, 64, "f16", True),
        diff("differential 256x16-128", 256, 16, 128, 6, 6, 64, "f16", True),
        diff("differential 16x2047", 16, 1024, 2047, 6, 6, 64, "bf16", True),
    ]


def f8(name, m, k, n, xt, yt):
    return {"name": name, "op": "f8", "m": m, "k": k, "n": n, "x": xt, "y": yt}


def quant(name, m, k, xt):
    return {"name": name, "op": "quant", "m": m, "k": k, "x": xt}


def qk(name, t, hq, hk, d, rot, pairing, dt, packed, max_pos):
    return {"name": name, "op": "qk", "t": t, "hq": hq, "hk": hk, "d": d, "rot": rot, "pairing": pairing, "x": dt,
            "packed": packed, "max_pos": max_pos}


def diff(name, nseq, lo, hi, h, hkv, d, dt, norm):
    return {"name": name, "op": "diff", "nseq": nseq, "lo": lo, "hi": hi, "h": h, "hkv": hkv, "d": d, "x": dt,
            "norm": norm}


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["f8", "f8", "quant", "qk", "diff", "diff"])
    t = rng.choice(list(TYPES))
    if op == "f8":
        while True:
            m, k, n = _log(rng, 1, 32768), 16 * _log(rng, 4, 512), _log(rng, 16, 8192)
            if m * k * n <= 8192 * 4096 * 4096:
                break
        c = f8("", m, k, n, t, rng.choice(list(TYPES)))
    elif op == "quant":
        while True:
            m, k = _log(rng, 1, 32768), 16 * _log(rng, 4, 512)
            if m * k * SIZE[t] <= 18431 * 4096 * 2:
                break
        c = quant("", m, k, t)
    elif op == "qk":
        while True:
            d = rng.choice([32, 64, 96, 128, 256])
            hk = rng.randint(1, 12)
            c = qk("", _log(rng, 1, 32767), hk * rng.randint(1, 4), hk, d, 16 * rng.randint(1, d // 16),
                   rng.choice(["interleaved", "half"]), t, rng.random() < 0.5, _log(rng, 512, 131072))
            if c["t"] * (c["hq"] + c["hk"]) * d * SIZE[t] <= 32767 * 40 * 128 * 2:
                break
    else:
        t = rng.choice(["f16", "bf16"])
        while True:
            hi = _log(rng, 1, 8192)
            hkv = rng.randint(1, 6)
            c = diff("", _log(rng, 1, 512), rng.randint(max(1, hi // 8), hi), hi, hkv * rng.choice([1, 1, 2]), hkv,
                     rng.choice([32, 64]), t, rng.random() < 0.7)
            if c["nseq"] * hi * hi * c["h"] <= 16 * 2047 * 2047 * 6:
                break
    c.pop("name")
    return c


# ----------------------------------------------------------------- inputs --

def lengths(c):
    r = random.Random("%d %d %d" % (c["nseq"], c["lo"], c["hi"]))
    return [r.randint(c["lo"], c["hi"]) for _ in range(c["nseq"])]


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _activations(m, k, t, seed):
    """Normal values with a few loud columns and rows of different scale, as a
    layer's activations have them."""
    g = _gen(seed)
    x = torch.randn(m, k, device="cuda", generator=g)
    x *= torch.exp(0.5 * torch.randn(m, 1, device="cuda", generator=g))
    loud = torch.rand(1, k, device="cuda", generator=g) < 0.01
    return torch.where(loud, 8 * x, x).to(TYPES[t])


def prepare(case, seed):
    c, g = case, _gen(seed + 1)
    s = {"c": c}
    if c["op"] == "f8":
        s["x"] = _activations(c["m"], c["k"], c["x"], seed)
        # An 8-bit checkpoint's weight: e4m3 values and a float32 scale for
        # each 128 x 128 block.
        nb, kb = -(-c["n"] // BLOCK), -(-c["k"] // BLOCK)
        s["w8"] = (100 * torch.randn(c["n"], c["k"], device="cuda", generator=g)).clamp(-448, 448).to(
            torch.float8_e4m3fn)
        s["ws"] = 0.0002 * (0.5 + torch.rand(nb, kb, device="cuda", generator=g))
        s["y"] = torch.empty(c["m"], c["n"], device="cuda", dtype=TYPES[c["y"]])
        if own:
            from llm_embed_b200 import ops
            s["w"] = ops.F8Weight(s["w8"].data_ptr(), s["ws"].data_ptr(), c["n"], c["k"])
            s["work"] = torch.empty(max(1, s["w"].workspace_bytes(c["m"], c["x"])), device="cuda", dtype=torch.uint8)
    elif c["op"] == "quant":
        s["x"] = _activations(c["m"], c["k"], c["x"], seed)
        s["q"] = torch.empty(c["m"], c["k"], device="cuda", dtype=torch.float8_e4m3fn)
        s["s"] = torch.empty(-(-c["k"] // BLOCK), c["m"], device="cuda")
    elif c["op"] == "qk":
        t, hq, hk, d = c["t"], c["hq"], c["hk"], c["d"]
        wide = (hq + 2 * hk) * d  # a packed row: queries, keys, values
        rows = _activations(t, wide, c["x"], seed)
        q, k = rows[:, :hq * d], rows[:, hq * d:(hq + hk) * d]
        s["q"], s["k"] = (q, k) if c["packed"] else (q.contiguous(), k.contiguous())
        s["qo"] = torch.empty(t, hq * d, device="cuda", dtype=TYPES[c["x"]])
        s["ko"] = torch.empty(t, hk * d, device="cuda", dtype=TYPES[c["x"]])
        s["qw"] = 1 + 0.2 * torch.randn(d, device="cuda", generator=g)
        s["kw"] = 1 + 0.2 * torch.randn(d, device="cuda", generator=g)
        # Texts of up to 512 tokens one after another; a long one starts late.
        at = torch.arange(t, device="cuda")
        first = torch.randint(0, max(1, c["max_pos"] - 511), (1 + t // 512,), device="cuda", generator=g)
        s["pos"] = (first[at // 512] + at % 512).clamp(max=c["max_pos"] - 1).to(torch.int32)
        p = torch.arange(c["max_pos"], device="cuda", dtype=torch.float64)
        a = p[:, None] * 10000.0 ** (-torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float64) / c["rot"])
        s["cos"], s["sin"] = a.cos().float(), a.sin().float()
        if own:
            from llm_embed_b200 import ops
            s["rope"] = ops.Rope(c["max_pos"], c["rot"], 10000.0, c["pairing"])
    else:
        lens = lengths(c)
        offs = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        t, h, hkv, d = int(offs[-1]), c["h"], c["hkv"], c["d"]
        rows = torch.randn(t, (2 * h + 4 * hkv) * d, device="cuda", generator=_gen(seed))
        # Heads of different sharpness: scores from nearly flat to a few
        # standard deviations of 3.
        rows[:, :2 * h * d] *= (0.5 + 2.5 * torch.rand(2 * h, device="cuda", generator=g)).repeat_interleave(d)
        rows = rows.to(TYPES[c["x"]])
        s["q"], s["k"], s["v"] = rows.split([2 * h * d, 2 * hkv * d, 2 * hkv * d], 1)
        s["offs"] = torch.from_numpy(offs).cuda()
        s["t"], s["max"] = t, max(lens)
        s["lam"] = 0.1 * torch.randn(4, d, device="cuda", generator=g)
        s["init"] = 0.8 - 0.6 * math.exp(-0.3 * 5)
        s["nw"] = 1 + 0.2 * torch.randn(2 * d, device="cuda", generator=g) if c["norm"] else None
        s["out"] = torch.empty(t, 2 * h * d, device="cuda", dtype=TYPES[c["x"]])
        if own:
            from llm_embed_b200 import ops
            s["attn"] = ops.DiffAttention(h, hkv, d, s["lam"].cpu().numpy(), s["init"],
                                          None if s["nw"] is None else s["nw"].cpu().numpy(), 1e-5)
    return s


# -------------------------------------------------------------- plain form --

def _blocks(x):
    """x [m, k] in 32 bits as [m, blocks, 128], zeros behind the last column."""
    m, k = x.shape
    return torch.nn.functional.pad(x.float(), (0, -k % BLOCK)).view(m, -1, BLOCK)


def _quantise(x):
    """Values e4m3 [m, blocks, 128] and scales [m, blocks] of x: each scale the
    smallest power of two that brings its block's largest value to 448 or less."""
    b = _blocks(x)
    top, e = torch.frexp(b.abs().amax(2))
    scale = (((e - 9 + (top > 0.875).int()).clamp(min=-126) + 127) << 23).view(torch.float32)  # exact, as pow() is not
    scale = torch.where(top == 0, torch.ones_like(scale), scale)
    return (b / scale[:, :, None]).to(torch.float8_e4m3fn), scale


def _plain_f8(s):
    c = s["c"]
    q, scale = _quantise(s["x"])
    x = (q.float() * scale[:, :, None]).view(c["m"], -1)[:, :c["k"]]
    n = torch.arange(c["n"], device="cuda") // BLOCK
    k = torch.arange(c["k"], device="cuda") // BLOCK
    return (x @ (s["w8"].float() * s["ws"][n][:, k]).t()).to(s["y"].dtype)


def _plain_quant(s):
    c = s["c"]
    q, scale = _quantise(s["x"])
    return q.view(c["m"], -1)[:, :c["k"]].contiguous(), scale.t().contiguous()


def _plain_norm_rope(x, heads, w, s):
    c = s["c"]
    d, rot = c["d"], c["rot"]
    u = x.float().reshape(-1, heads, d)
    u = u * torch.rsqrt((u * u).mean(2, keepdim=True) + 1e-6) * w
    cos, sin = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]
    r = u[:, :, :rot]
    a, b = (r[:, :, 0::2], r[:, :, 1::2]) if c["pairing"] == "interleaved" else (r[:, :, :rot // 2], r[:, :, rot // 2:])
    ra, rb = a * cos - b * sin, a * sin + b * cos
    r = torch.stack([ra, rb], 3).flatten(2) if c["pairing"] == "interleaved" else torch.cat([ra, rb], 2)
    return torch.cat([r, u[:, :, rot:]], 2).reshape(-1, heads * d).to(x.dtype)


def _plain_diff(s):
    """Every sequence padded to the longest; one softmax map for each of a
    head's two parts."""
    c = s["c"]
    h, hkv, d, n, t = c["h"], c["hkv"], c["d"], s["max"], s["t"]
    start, end = s["offs"][:-1, None].long(), s["offs"][1:, None].long()
    at = torch.arange(n, device="cuda")
    row = start + at  # [sequences, n]
    there = row < end
    row = torch.where(there, row, 0)

    def heads(x, kinds):  # [sequences, heads, kinds, n, columns]
        return x.float()[row].view(len(start), n, -1, kinds, 2 * d // kinds).permute(0, 2, 3, 1, 4)

    q, k = heads(s["q"], 2), heads(s["k"], 2).repeat_interleave(h // hkv, 1)
    v = heads(s["v"], 1).repeat_interleave(h // hkv, 1)
    score = (q @ k.transpose(3, 4) / math.sqrt(d)).masked_fill(~there[:, None, None, None], -math.inf)
    p = torch.exp(score - score.amax(4, keepdim=True))
    p = p / p.sum(4, keepdim=True)
    lam = s["lam"]
    lam = torch.exp((lam[0] * lam[1]).sum()) - torch.exp((lam[2] * lam[3]).sum()) + s["init"]
    o = (p[:, :, 0] - lam * p[:, :, 1]) @ v[:, :, 0]  # [sequences, heads, n, 2d]
    if s["nw"] is not None:
        o = (1 - s["init"]) * o * torch.rsqrt((o * o).mean(3, keepdim=True) + 1e-5) * s["nw"]
    return o.permute(0, 2, 1, 3).reshape(-1, n, 2 * h * d)[there].to(s["out"].dtype)


def run(state):
    s = state
    op = s["c"]["op"]
    if own:
        return _own(s)
    if op == "f8":
        return _plain_f8(s)
    if op == "quant":
        return _plain_quant(s)
    if op == "qk":
        return (_plain_norm_rope(s["q"], s["c"]["hq"], s["qw"], s), _plain_norm_rope(s["k"], s["c"]["hk"], s["kw"], s))
    return _plain_diff(s)


def _own(s):
    from llm_embed_b200 import ops
    c = s["c"]
    stream = torch.cuda.current_stream().cuda_stream or ops.LEGACY_STREAM
    if c["op"] == "f8":
        s["w"].matmul_device(s["x"].data_ptr(), c["m"], s["y"].data_ptr(), c["x"], c["y"],
                             d_work=s["work"].data_ptr(), work_bytes=s["work"].numel(), stream=stream)
        return s["y"]
    if c["op"] == "quant":
        ops.f8_quantize_device(s["x"].data_ptr(), c["x"], c["m"], c["k"], s["q"].data_ptr(), s["s"].data_ptr(),
                               stream=stream)
        return s["q"], s["s"]
    if c["op"] == "qk":
        s["rope"].qk_norm_device(c["x"], c["t"], c["hq"], c["hk"], c["d"], s["q"].data_ptr(), s["k"].data_ptr(),
                                 s["pos"].data_ptr(), s["qo"].data_ptr(), s["ko"].data_ptr(),
                                 q_stride=s["q"].stride(0), k_stride=s["k"].stride(0),
                                 d_q_weight=s["qw"].data_ptr(), d_k_weight=s["kw"].data_ptr(), eps=1e-6,
                                 stream=stream)
        return s["qo"], s["ko"]
    s["attn"].run_device(c["x"], s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["offs"].data_ptr(),
                         c["nseq"], s["t"], s["max"], s["out"].data_ptr(), q_stride=s["q"].stride(0),
                         k_stride=s["k"].stride(0), v_stride=s["v"].stride(0), stream=stream)
    return s["out"]


# ------------------------------------------------------------------- work --

def work(case):
    c = case
    if c["op"] == "f8":
        return {"bytes": c["m"] * c["k"] * SIZE[c["x"]] + c["n"] * c["k"] + c["m"] * c["n"] * SIZE[c["y"]],
                "flops": 2 * c["m"] * c["n"] * c["k"]}
    if c["op"] == "quant":
        return {"bytes": c["m"] * c["k"] * (SIZE[c["x"]] + 1) + 4 * c["m"] * -(-c["k"] // BLOCK),
                "flops": 3 * c["m"] * c["k"]}
    if c["op"] == "qk":
        v = c["t"] * (c["hq"] + c["hk"]) * c["d"]
        return {"bytes": 2 * v * SIZE[c["x"]] + 4 * c["t"], "flops": 8 * v}
    return {"bytes": sum(lengths(c)) * (4 * c["h"] + 4 * c["hkv"]) * c["d"] * SIZE[c["x"]],
            "flops": 12 * c["d"] * c["h"] * sum(n * n for n in lengths(c))}


# ------------------------------------------------------------------ exact --

def _two_to(e):
    """2^e exactly (pow() may be an ulp off)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_quantise(x):
    """Block by block from the definition, in 64 bits; the rounding to e4m3 by
    its step, 2^-3 of the value's power of two and 2^-9 at least."""
    m, k = x.shape
    values, scales = torch.empty(m, k, device="cuda", dtype=torch.float64), []
    for a in range(0, k, BLOCK):
        b = x[:, a:a + BLOCK].double()
        top = b.abs().max(1, keepdim=True).values
        e = torch.ceil(torch.log2(torch.where(top > 0, top, 448.0) / 448))
        e = torch.where(top > 448 * _two_to(e), e + 1, e)
        e = torch.where(top <= 448 * _two_to(e - 1), e - 1, e)
        e = torch.where(top > 0, e.clamp(min=-126), 0.0)
        b = b / _two_to(e)
        near = torch.floor(torch.log2(b.abs().clamp(min=2.0 ** -6)))
        near = torch.where(b.abs() >= _two_to(near + 1), near + 1, near)
        near = torch.where(b.abs() < _two_to(near), near - 1, near).clamp(min=-6)
        step = _two_to(near - 3)
        values[:, a:a + BLOCK] = torch.round(b / step) * step
        scales.append(_two_to(e))
    return values, torch.cat(scales, 1)


def _exact_head(x, w, s, c):
    u = x.double()
    u = u / (u.square().sum(1, keepdim=True) / c["d"] + 1e-6).sqrt() * w.double()
    out, half = u.clone(), c["rot"] // 2
    for i in range(half):
        angle = s["pos"].double() * 10000.0 ** (-2 * i / c["rot"])
        a, b = (2 * i, 2 * i + 1) if c["pairing"] == "interleaved" else (i, i + half)
        out[:, a] = u[:, a] * angle.cos() - u[:, b] * angle.sin()
        out[:, b] = u[:, a] * angle.sin() + u[:, b] * angle.cos()
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "quant":
        q, scale = _exact_quantise(s["x"])
        return q, scale.t().contiguous()
    if c["op"] == "f8":
        q, scale = _exact_quantise(s["x"])
        y = torch.zeros(c["m"], c["n"], device="cuda", dtype=torch.float64)
        for b, a in enumerate(range(0, c["k"], BLOCK)):
            w = s["w8"][:, a:a + BLOCK].float().double()
            for j in range(0, c["n"], BLOCK):
                w[j:j + BLOCK] *= s["ws"][j // BLOCK, b].double()
            y += scale[:, b:b + 1] * (q[:, a:a + BLOCK] @ w.t())
        return y
    if c["op"] == "qk":
        d, outs = c["d"], []
        for x, n, w in ((s["q"], c["hq"], s["qw"]), (s["k"], c["hk"], s["kw"])):
            outs.append(torch.cat([_exact_head(x[:, i * d:(i + 1) * d], w, s, c) for i in range(n)], 1))
        return tuple(outs)
    h, d, offs = c["h"], c["d"], s["offs"].tolist()
    out = torch.empty(s["t"], 2 * h * d, device="cuda", dtype=torch.float64)
    l64 = s["lam"].double()
    lam = torch.exp(l64[0] @ l64[1]) - torch.exp(l64[2] @ l64[3]) + s["init"]
    for a, b in zip(offs, offs[1:]):
        for j in range(h):
            g = j // (h // c["hkv"])
            maps = []
            for part in (0, 1):
                x = s["q"][a:b, (2 * j + part) * d:(2 * j + part + 1) * d].double()
                y = s["k"][a:b, (2 * g + part) * d:(2 * g + part + 1) * d].double()
                maps.append(torch.softmax(x @ y.t() * d ** -0.5, 1))
            o = (maps[0] - lam * maps[1]) @ s["v"][a:b, 2 * g * d:2 * (g + 1) * d].double()
            if s["nw"] is not None:
                o = (1 - s["init"]) * o / (o.square().sum(1, keepdim=True) / (2 * d) + 1e-5).sqrt() * s["nw"].double()
            out[a:b, 2 * j * d:2 * (j + 1) * d] = o
    return out
