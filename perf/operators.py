"""Measured cases of the float linear operator and of the fused query/key norm + rotation.

linear        y = act(x . w^T + b) [* (x . u^T + c)] + r: the projections of a transformer block, from one
              decoded token to a batched encoder's rows (slx_linear_prepare, slx_linear_device).
qk_norm_rope  RmsNorm of every query and key head followed by the rotary positions, in float and in
              the Q30 integers of the causal path (slx_rope_create, slx_qk_norm_prepare,
              slx_qk_norm_rope_device).

Plain forms are elementary torch operations; with `own` the framework's operators run.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "q30": torch.int64}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "q30": 8}
MOST_FLOPS = 2.0 * 4096 * 4096 * 11008   # the largest listed product
MOST_F32 = 2.0 * 8192 * 768 * 2304       # the largest listed product in fp32
MOST_WEIGHTS = 64 << 20
MOST_HEADS = 8192 * 40 * 128             # the largest listed rotation, in elements


def linear(name, dtype, m, k, n, act="none", gated=False, bias=False, residual=False, pad=0):
    return {"name": name, "op": "linear", "dtype": dtype, "m": m, "k": k, "n": n, "act": act, "gated": gated,
            "bias": bias, "residual": residual, "pad": pad}


def rotation(name, dtype, m, t, heads, kv_heads, hd, rot, rows, base, norm=True, fused=False, ragged=False):
    return {"name": name, "op": "qk_norm_rope", "dtype": dtype, "m": m, "t": t, "heads": heads, "kv_heads": kv_heads,
            "hd": hd, "rot": rot, "rows": rows, "base": base, "norm": norm, "fused": fused, "ragged": ragged}


def listed():
    return [
        # one decoded token through an encoder-width output projection: latency
        linear("linear f32 1x768x768", "f32", 1, 768, 768, bias=True, residual=True),
        # one decoded token through a wide FFN matrix: the weight stream
        linear("linear bf16 1x4096x11008", "bf16", 1, 4096, 11008, act="silu"),
        # a few sequences decoded together
        linear("linear f16 8x4096x4096", "f16", 8, 4096, 4096, residual=True),
        # a short prompt, every size odd, rows of x, r and y longer than their widths
        linear("linear f16 129x1001x1111", "f16", 129, 1001, 1111, act="gelu_erf", bias=True, residual=True, pad=5),
        # the causal LM's gated FFN on its 512-token prompt
        linear("linear bf16 512x2048x16384 gated", "bf16", 512, 2048, 16384, act="silu", gated=True),
        # the batched encoder's QKV projection in the float twin's type
        linear("linear f32 8192x768x2304", "f32", 8192, 768, 2304, bias=True),
        # a long prefill through a wide matrix
        linear("linear bf16 4096x4096x11008", "bf16", 4096, 4096, 11008, act="gelu_tanh", bias=True, residual=True),
        # one decoded token of the causal LM's head layout, far into its context
        rotation("rotation bf16 1x(8+1)x256", "bf16", 1, 1, 8, 1, 256, 256, 2048, 10000.0, ragged=True),
        # the batched encoder's rows: no norm, q and k read from the fused [q | k | v] rows
        rotation("rotation f32 513x(12+12)x64 no norm", "f32", 513, 171, 12, 12, 64, 64, 512, 1000.0, norm=False, fused=True),
        # the causal LM's prompt plus one token in its Q30 integers
        rotation("rotation q30 513x(8+1)x256", "q30", 513, 513, 8, 1, 256, 256, 2048, 10000.0),
        # packed sequences of unequal lengths, part of each head rotated
        rotation("rotation f16 3001x(20+4)x96/64", "f16", 3001, 3001, 20, 4, 96, 64, 8192, 500000.0, fused=True, ragged=True),
        # a long prefill with grouped heads
        rotation("rotation bf16 8192x(32+8)x128", "bf16", 8192, 2048, 32, 8, 128, 128, 32768, 1000000.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.6:
        dtype = rng.choice(["f32", "f16", "bf16"])
        m = rng.randint(1, 16) if rng.random() < 0.35 else _log(rng, 1, 8192)
        k, n = _log(rng, 48, 8192), _log(rng, 48, 16384)
        if rng.random() < 0.6:  # widths of real layers are multiples of 32
            k, n = max(32, k // 32 * 32), max(32, n // 32 * 32)
        gated = rng.random() < 0.3
        while k * n * (2 if gated else 1) > MOST_WEIGHTS:
            n = n // 2 + 1
        while 2.0 * m * k * n * (2 if gated else 1) > (MOST_F32 if dtype == "f32" else MOST_FLOPS):
            m = m // 2 + 1
        act = rng.choice(["silu", "gelu_tanh", "gelu_erf"]) if gated else rng.choice(["none", "none", "relu", "silu", "gelu_tanh", "gelu_erf"])
        c = linear("", dtype, m, k, n, act, gated, rng.random() < 0.5, rng.random() < 0.5, rng.choice([0, 0, 0, 3, 8]))
    else:
        dtype = rng.choice(["f32", "f16", "bf16", "q30"])
        hd = 2 * rng.randint(8, 128) if rng.random() < 0.3 else rng.choice([32, 64, 96, 128, 256])
        rot = hd if dtype == "q30" or rng.random() < 0.7 else 2 * rng.randint(1, hd // 2)
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.randint(1, 8)
        m = rng.randint(1, 16) if rng.random() < 0.35 else _log(rng, 1, 8192)
        while m * (heads + kv) * hd * BYTES[dtype] > MOST_HEADS * 2:
            m = m // 2 + 1
        rows = _log(rng, 512, 4096 if dtype == "q30" else 32768)
        c = rotation("", dtype, m, min(rows, rng.randint(1, m)), heads, kv, hd, rot, rows,
                     rng.choice([1000.0, 10000.0, 1000000.0]), dtype == "q30" or rng.random() < 0.8, rng.random() < 0.5,
                     rng.random() < 0.5)
    del c["name"]
    return c


# ---- inputs ------------------------------------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rows(g, m, width, pad, dtype, scale=1.0):
    """m rows of `width` values, `pad` further elements between a row's end and the next one."""
    return (scale * torch.randn(m, width + pad, generator=g, device="cuda")).to(dtype)[:, :width]


def _prepare_linear(c, seed):
    g, dt = _gen(seed), TYPES[c["dtype"]]
    m, k, n, pad = c["m"], c["k"], c["n"], c["pad"]
    s = {"case": c, "x": _rows(g, m, k, pad, dt), "w": _rows(g, n, k, 0, dt, 1.0 / math.sqrt(k)),
         "gate": _rows(g, n, k, 0, dt, 1.0 / math.sqrt(k)) if c["gated"] else None,
         "b": 0.5 * torch.randn(n, generator=g, device="cuda") if c["bias"] else None,
         "gb": 0.5 * torch.randn(n, generator=g, device="cuda") if c["bias"] and c["gated"] else None,
         "r": _rows(g, m, n, pad, dt) if c["residual"] else None}
    if own:
        import spatialdb_b200 as slx
        at = lambda v: v.data_ptr() if v is not None else 0  # noqa: E731
        code, size = _code(slx, c["dtype"]), n * k * BYTES[c["dtype"]]
        torch.cuda.synchronize()
        s["op"] = slx.Linear(code, at(s["w"]), size, code, n, k, d_bias=at(s["b"]), act=getattr(slx, "ACT_" + c["act"].upper()),
                             d_gate=at(s["gate"]), gate_bytes=size if c["gated"] else 0, d_gate_bias=at(s["gb"]))
        s["y"] = torch.empty(m, n + pad, dtype=dt, device="cuda")[:, :n]
    return s


def _q30_tables(rows, rot, base):
    """The integer rotation cache: the C library's pow, cos and sin in double, truncated to 30 bits."""
    half = rot // 2
    theta = [math.pow(base, -2.0 * i / rot) for i in range(half)]
    one = float(1 << 30)
    cos = torch.tensor([int(math.cos(t * a) * one) for t in range(rows) for a in theta], dtype=torch.int64)
    sin = torch.tensor([int(math.sin(t * a) * one) for t in range(rows) for a in theta], dtype=torch.int64)
    return cos.view(rows, half).cuda(), sin.view(rows, half).cuda()


def _angles(c, pos):
    half = c["rot"] // 2
    theta = torch.pow(torch.tensor(c["base"], dtype=torch.float64, device="cuda"),
                      -2.0 * torch.arange(half, dtype=torch.float64, device="cuda") / c["rot"])
    return pos.to(torch.float64)[:, None] * theta


def _prepare_rotation(c, seed):
    g, dt = _gen(seed), TYPES[c["dtype"]]
    m, nq, nk, hd = c["m"], c["heads"] * c["hd"], c["kv_heads"] * c["hd"], c["hd"]
    q30 = c["dtype"] == "q30"
    width = nq + 2 * nk
    x = torch.randn(m, width, generator=g, device="cuda")
    x = (x.double() * float(1 << 30)).to(dt) if q30 else x.to(dt)
    q, k = x[:, :nq], x[:, nq:nq + nk]
    if not c["fused"]:
        q, k = q.contiguous(), k.contiguous()
    wq = wk = None
    if c["norm"]:
        wq, wk = (1.0 + 0.2 * torch.randn(hd, generator=g, device="cuda") for _ in range(2))
        if q30:
            wq, wk = ((w.double() * float(1 << 30)).to(dt) for w in (wq, wk))
    if c["ragged"]:  # sequences of unequal lengths packed one after another, each from a place of its own
        length = torch.randint(1, min(m, c["rows"]) + 1, (m,), generator=g, device="cuda")
        ends = torch.cumsum(length, 0)
        at = torch.arange(m, device="cuda")
        which = torch.searchsorted(ends, at, right=True)
        begin = torch.randint(0, 1 << 30, (m,), generator=g, device="cuda") % (c["rows"] - length + 1)
        pos = (at - (ends - length)[which] + begin[which]).to(torch.int32)
    else:
        pos = None
    s = {"case": c, "q": q, "k": k, "wq": wq, "wk": wk, "pos": pos}
    if q30:
        s["cos"], s["sin"] = _q30_tables(c["rows"], c["rot"], c["base"])
    else:
        a = _angles(c, torch.arange(c["rows"], device="cuda"))
        s["cos"], s["sin"] = torch.cos(a).float(), torch.sin(a).float()
    if own:
        import spatialdb_b200 as slx
        code = _code(slx, c["dtype"])
        torch.cuda.synchronize()
        s["table"] = slx.RopeTable(c["rows"], c["rot"], c["base"], q30=q30)
        s["op"] = slx.QkNormRope(s["table"], code, c["heads"], c["kv_heads"], hd, d_wq=wq.data_ptr() if c["norm"] else 0,
                                 d_wk=wk.data_ptr() if c["norm"] else 0, eps=0.0 if q30 else 1e-6)
        s["qo"], s["ko"] = (torch.empty(m, n, dtype=dt, device="cuda") for n in (nq, nk))
    return s


def _code(slx, dtype):
    return {"f32": slx.DTYPE_F32, "f16": slx.DTYPE_F16, "bf16": slx.DTYPE_BF16, "q30": slx.DTYPE_Q30}[dtype]


def prepare(case, seed):
    return _prepare_linear(case, seed) if case["op"] == "linear" else _prepare_rotation(case, seed)


# ---- plain forms -------------------------------------------------------------------------------------


def _act(v, name):
    if name == "relu":
        return v.clamp_min(0)
    if name == "silu":
        return v / (1 + torch.exp(-v))
    if name == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    if name == "gelu_erf":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    return v


def _linear_in(s, num):
    """The linear operator with every number of type `num`, before the last rounding."""
    c, x = s["case"], s["x"].to(num)
    y = x @ s["w"].to(num).T
    if s["b"] is not None:
        y = y + s["b"].to(num)
    if c["gated"]:
        g = x @ s["gate"].to(num).T
        if s["gb"] is not None:
            g = g + s["gb"].to(num)
        y = _act(g, c["act"]) * y
    else:
        y = _act(y, c["act"])
    return y + s["r"].to(num) if s["r"] is not None else y


def _positions(s):
    c = s["case"]
    return s["pos"].long() if s["pos"] is not None else torch.arange(c["m"], device="cuda") % c["t"]


def _heads_in(x, w, cos, sin, c, num):
    """Norm and rotation of one tensor's heads, with every number of type `num`."""
    u = x.reshape(x.shape[0], -1, c["hd"]).to(num)
    if w is not None:
        u = u / torch.sqrt((u * u).mean(-1, keepdim=True) + 1e-6) * w.to(num)
    h = c["rot"] // 2
    a, b, rest = u[..., :h], u[..., h:2 * h], u[..., 2 * h:]
    cos, sin = cos[:, None, :], sin[:, None, :]
    return torch.cat([a * cos - b * sin, a * sin + b * cos, rest], -1).reshape(x.shape)


def _mean_square(x):
    """floor(sum x^2 / n) of the last axis, each square formed from 17-bit halves so that no sum overflows."""
    n, lo, hi = x.shape[-1], x & ((1 << 17) - 1), x >> 17
    a, b, c = (hi * hi).sum(-1), (hi * lo).sum(-1), (lo * lo).sum(-1)
    low = ((a % n) << 34) + (b << 18) + c
    return ((a // n) << 34) + torch.div(low, n, rounding_mode="floor")


def _shift30(x, c, y, s):
    """(x c + y s) >> 30 from 15-bit parts of x and y."""
    low = (x & 32767) * c + (y & 32767) * s
    return ((x >> 15) * c + (y >> 15) * s + (low >> 15)) >> 15


def _heads_q30(x, w, cos, sin, c):
    """The integer norm (truncating division by the floored root of the mean square), then the floored rotation."""
    v = x.reshape(x.shape[0], -1, c["hd"])
    ms = _mean_square(v)
    root = torch.sqrt(ms.double()).long()
    root = root - (root * root > ms).long()
    root = (root + ((root + 1) * (root + 1) <= ms).long()).unsqueeze(-1)
    av, aw = v.abs(), w.abs()
    quo = torch.floor(av.double() * aw.double() / root.double()).long()
    rem = av * aw - quo * root  # exact where the products wrap: the true value is small
    quo = quo - (rem < 0).long() + (rem >= root).long()
    u = quo * torch.sign(v) * torch.sign(w)
    h = c["rot"] // 2
    a, b = u[..., :h], u[..., h:]
    cos, sin = cos[:, None, :], sin[:, None, :]
    return torch.cat([_shift30(a, cos, b, -sin), _shift30(a, sin, b, cos)], -1).reshape(x.shape)


def run(s):
    c = s["case"]
    if own:
        if c["op"] == "linear":
            x, y, r = s["x"], s["y"], s["r"]
            s["op"].apply_device(x.data_ptr(), c["m"], y.data_ptr(), ldx=x.stride(0), ldo=y.stride(0),
                                 d_residual=0 if r is None else r.data_ptr(), ldr=0 if r is None else r.stride(0), stream=1)
            return y
        q, k, pos = s["q"], s["k"], s["pos"]
        s["op"].apply_device(q.data_ptr(), k.data_ptr(), c["m"], s["qo"].data_ptr(), s["ko"].data_ptr(), T=c["t"],
                             d_pos=0 if pos is None else pos.data_ptr(), ldq=q.stride(0), ldk=k.stride(0), stream=1)
        return s["qo"], s["ko"]
    if c["op"] == "linear":
        return _linear_in(s, torch.float32).to(s["x"].dtype)
    at = _positions(s)
    cos, sin = s["cos"][at], s["sin"][at]
    if c["dtype"] == "q30":
        return _heads_q30(s["q"], s["wq"], cos, sin, c), _heads_q30(s["k"], s["wk"], cos, sin, c)
    dt = s["q"].dtype
    return (_heads_in(s["q"], s["wq"], cos, sin, c, torch.float32).to(dt),
            _heads_in(s["k"], s["wk"], cos, sin, c, torch.float32).to(dt))


# ---- in 64 bits --------------------------------------------------------------------------------------


def _exact_linear(s):
    c = s["case"]
    d = {k: None if v is None else v.double() for k, v in s.items() if k in ("x", "w", "gate", "b", "gb", "r")}

    def product(w, b):
        p = torch.einsum("mk,nk->mn", d["x"], w)
        return p if b is None else p + b[None, :]

    acts = {"none": lambda v: v, "relu": lambda v: torch.where(v > 0, v, torch.zeros_like(v)),
            "silu": lambda v: v * torch.special.expit(v),
            "gelu_tanh": lambda v: v * torch.special.expit(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)),
            "gelu_erf": lambda v: v * torch.special.ndtr(v)}
    y = product(d["w"], d["b"])
    y = acts[c["act"]](product(d["gate"], d["gb"])) * y if c["gated"] else acts[c["act"]](y)
    return y if d["r"] is None else y + d["r"]


def _exact_rotation(s):
    c = s["case"]
    z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda").expand(c["m"], c["rot"] // 2),
                    _angles(c, _positions(s)))[:, None, :]

    def heads(x, w):
        v = x.double().reshape(c["m"], -1, c["hd"])
        if w is not None:
            v = v * w.double() / (v.square().sum(-1, keepdim=True) / c["hd"] + 1e-6).sqrt()
        pair = torch.complex(v[..., :c["rot"] // 2], v[..., c["rot"] // 2:c["rot"]]) * z
        return torch.cat([pair.real, pair.imag, v[..., c["rot"]:]], -1).reshape(x.shape)

    return heads(s["q"], s["wq"]), heads(s["k"], s["wk"])


def exact(case, seed):
    if case["dtype"] == "q30":  # whole numbers, compared for equality
        return None
    s = prepare(case, seed)
    return _exact_linear(s) if case["op"] == "linear" else _exact_rotation(s)


def work(c):
    e = BYTES[c["dtype"]]
    if c["op"] == "linear":
        m, k, n, sides = c["m"], c["k"], c["n"], 2 if c["gated"] else 1
        vectors = 4 * n * sides if c["bias"] else 0
        return {"bytes": e * (m * k + sides * n * k + m * n * (2 if c["residual"] else 1)) + vectors,
                "flops": 2.0 * m * k * n * sides}
    width = (c["heads"] + c["kv_heads"]) * c["hd"]
    table = c["m"] if c["ragged"] else min(c["m"], c["t"])
    entry = 8 if c["dtype"] == "q30" else 4
    return {"bytes": 2 * e * c["m"] * width + entry * c["rot"] * table + (2 * entry * c["hd"] if c["norm"] else 0)
            + (4 * c["m"] if c["ragged"] else 0),
            "flops": 7.0 * c["m"] * width}
