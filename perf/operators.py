"""Measured cases of the transformer-block operators next to VC-Attention:
``qk_norm_rope``, ``quantize_blocks``, ``matmul_blocks`` and
``packed_attention``.

Each case has a plain form (elementary torch operations in float32, rounded
once at the end) and the framework's own call (``own = True``).  The sizes are
those of the H3 profile (56 heads x 128, hidden 5376, QKV width 7168, FFN
14336, 96 of 128 channels rotated) and generic ones.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ES = {"bf16": 2, "f16": 2, "f32": 4}
BLK = 128


def listed():
    return [
        # one new row of a prompt encoder with grouped heads: launch latency
        {"name": "rope_one_token", "op": "rope", "dtype": "bf16", "b": 1, "n": 1, "hq": 32, "hk": 8, "d": 128,
         "rot": 128, "layout": "half", "fused": True},
        # two text prompts (an odd length), head dim 64, pairs side by side
        {"name": "rope_text", "op": "rope", "dtype": "f16", "b": 2, "n": 333, "hq": 24, "hk": 24, "d": 64,
         "rot": 64, "layout": "interleaved", "fused": False},
        # one 16K-row clip, 56 heads, views into the fused QKV projection's output
        {"name": "rope_clip", "op": "rope", "dtype": "bf16", "b": 1, "n": 16384, "hq": 56, "hk": 56, "d": 128,
         "rot": 96, "layout": "half", "fused": True},
        # one activation row before a projection: launch latency
        {"name": "quant_one_token", "op": "quant", "dtype": "bf16", "m": 1, "k": 5376, "rows": 1},
        # the clip's FFN activations before the down projection
        {"name": "quant_clip", "op": "quant", "dtype": "bf16", "m": 16384, "k": 14336, "rows": 1},
        # attention output projection of one new row: bound by the weight's bytes
        {"name": "matmul_one_token", "op": "matmul", "dtype": "bf16", "m": 1, "n": 5376, "k": 7168, "bias": False},
        # FFN up projection of a text prompt (odd row count), bias, f16
        {"name": "matmul_text", "op": "matmul", "dtype": "f16", "m": 333, "n": 14336, "k": 5376, "bias": True},
        # Q projection of a 16K-row clip: bound by the tensor cores
        {"name": "matmul_clip", "op": "matmul", "dtype": "bf16", "m": 16384, "n": 7168, "k": 5376, "bias": False},
        # a batch of single new tokens against their ragged histories: bound by the K/V bytes
        {"name": "attn_one_token", "op": "attn", "dtype": "bf16", "hq": 32, "hk": 8, "d": 128, "causal": True,
         "q_lens": "1,1,1,1,1,1,1,1,1,1,1,1", "k_lens": "8192,301,4096,1,7777,2050,640,5000,1023,8190,129,3300"},
        # six packed prompts through a bidirectional text encoder: small tiles, ragged ends
        {"name": "attn_text", "op": "attn", "dtype": "f16", "hq": 16, "hk": 16, "d": 64, "causal": False,
         "q_lens": "1,77,128,200,333,512", "k_lens": "1,77,128,200,333,512"},
        # causal prompts with grouped heads, some continuing an earlier part
        {"name": "attn_prompt", "op": "attn", "dtype": "bf16", "hq": 32, "hk": 8, "d": 128, "causal": True,
         "q_lens": "2048,1500,1,511,37", "k_lens": "4096,1500,700,511,2085"},
        # exact attention over a whole 16K-row clip, a quarter of the 56 heads (one of four GPUs)
        {"name": "attn_clip", "op": "attn", "dtype": "bf16", "hq": 14, "hk": 14, "d": 128, "causal": False,
         "q_lens": "16384", "k_lens": "16384"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "quant", "matmul", "attn"])
    if op == "rope":
        d = rng.choice([64, 128])
        hq = rng.choice([8, 14, 24, 32, 40, 56])
        hk = rng.choice([h for h in (1, 2, 8, 14, 24, 32, 40, 56) if hq % h == 0])
        b = rng.choice([1, 1, 2, 3])
        n = max(1, min(_log(rng, 1, 16384), 16384 * 112 * 128 // (b * (hq + hk) * d)))
        return {"op": op, "dtype": rng.choice(["bf16", "f16"]), "b": b, "n": n, "hq": hq, "hk": hk, "d": d,
                "rot": rng.choice([32, 48, 64] if d == 64 else [64, 96, 128]),
                "layout": rng.choice(["half", "interleaved"]), "fused": rng.random() < 0.5}
    if op == "quant":
        k = rng.choice([_log(rng, 64, 14336), 5376, 7168, 14336])
        return {"op": op, "dtype": rng.choice(["bf16", "f16"]), "m": _log(rng, 1, 16384), "k": k,
                "rows": rng.choice([1, 1, 1, 128])}
    if op == "matmul":
        while True:
            c = {"op": op, "dtype": rng.choice(["bf16", "f16"]), "m": _log(rng, 1, 16384),
                 "n": rng.choice([5376, 7168, 14336, 8 * _log(rng, 16, 2048)]),
                 "k": rng.choice([5376, 7168, 14336, 16 * _log(rng, 8, 1024)]), "bias": rng.random() < 0.5}
            if c["m"] * c["n"] * c["k"] <= 16384 * 7168 * 5376:
                return c
    while True:
        hq, hk = rng.choice([(32, 8), (40, 8), (16, 16), (14, 14), (56, 56), (24, 24), (16, 1)])
        causal = rng.random() < 0.6
        kind = rng.choice(["whole", "chunk", "one"])
        ns = rng.randint(1, 12)
        kl = [_log(rng, 1, 16384 if ns == 1 else 8192) for _ in range(ns)]
        ql = {"whole": kl, "chunk": [max(1, min(x, _log(rng, 1, 2048))) for x in kl], "one": [1] * ns}[kind]
        c = {"op": "attn", "dtype": rng.choice(["bf16", "f16"]), "hq": hq, "hk": hk, "d": rng.choice([64, 128]),
             "causal": causal, "q_lens": ",".join(map(str, ql)), "k_lens": ",".join(map(str, kl))}
        if sum(ql) * sum(kl) * hq * c["d"] <= 16384 * 16384 * 14 * 128:
            return c


# ---------------------------------------------------------------- inputs ----
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _lens(text):
    return [int(x) for x in text.split(",")]


def _rope_inputs(c, g):
    dt, b, n, hq, hk, d = DTYPES[c["dtype"]], c["b"], c["n"], c["hq"], c["hk"], c["d"]
    if c["fused"]:   # (B, N, (Hq + 2 Hk) D) projection output: q and k are strided views of it
        qkv = _normal(g, b, n, hq + 2 * hk, d).to(dt)
        q, k = qkv[:, :, :hq].transpose(1, 2), qkv[:, :, hq:hq + hk].transpose(1, 2)
    else:
        q, k = _normal(g, b, hq, n, d).to(dt), _normal(g, b, hk, n, d).to(dt)
    half = c["rot"] // 2
    freq = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    start = torch.randint(0, 4096, (1,), generator=g, device="cuda")
    ang = (torch.arange(n, device="cuda") + start).to(torch.float64)[:, None] * freq
    return {"q": q, "k": k, "cos": ang.cos().float(), "sin": ang.sin().float(),
            "qw": 1 + 0.1 * _normal(g, d), "kw": 1 + 0.1 * _normal(g, d), "eps": 1e-5}


def _spread(g, rows, cols):
    """Rows of different size, as activations and weights have."""
    return _normal(g, rows, cols) * torch.exp(0.5 * _normal(g, rows, 1))


def _matmul_inputs(c, g):
    m, n, k = c["m"], c["n"], c["k"]
    kb = -(-k // BLK)
    a8 = (100.0 * _normal(g, m, k)).clamp_(-448, 448).to(torch.float8_e4m3fn)
    b8 = (100.0 * _normal(g, n, k)).clamp_(-448, 448).to(torch.float8_e4m3fn)
    # per (row, block) and per (128 rows, block) scales, stored block-major
    sa = torch.exp(0.5 * _normal(g, kb, m)).mul_(0.01).t()
    sb = torch.exp(0.3 * _normal(g, kb, -(-n // BLK))).mul_(0.01 / math.sqrt(k)).t()
    bias = _normal(g, n) if c["bias"] else None
    return {"a8": a8, "sa": sa, "b8": b8, "sb": sb, "bias": bias}


def _attn_inputs(c, g):
    dt, d = DTYPES[c["dtype"]], c["d"]
    ql, kl = _lens(c["q_lens"]), _lens(c["k_lens"])
    q = _normal(g, sum(ql), c["hq"], d).to(dt)
    # keys with a common per-channel offset, as trained keys have
    k = (_normal(g, sum(kl), c["hk"], d) + 0.5 * _normal(g, 1, c["hk"], d)).to(dt)
    v = _normal(g, sum(kl), c["hk"], d).to(dt)
    t = lambda x: x.transpose(0, 1).unsqueeze(0)  # noqa: E731  (1, H, T, D) views of (T, H, D) rows
    s = {"q": t(q), "k": t(k), "v": t(v), "ql": torch.tensor(ql, device="cuda"), "kl": torch.tensor(kl, device="cuda")}
    if own:   # the layout of the batch, kept for all layers of a model
        from comfyui_vc_attention_b200.vc_attention import packed_plan
        s["plan"] = packed_plan(ql, kl, heads=c["hq"], kv_heads=c["hk"], head_dim=d, causal=c["causal"])
    return s


def prepare(case, seed):
    g = _gen(seed)
    c = dict(case)
    if c["op"] == "rope":
        return {"c": c, **_rope_inputs(c, g)}
    if c["op"] == "quant":
        return {"c": c, "x": _spread(g, c["m"], c["k"]).to(DTYPES[c["dtype"]])}
    if c["op"] == "matmul":
        return {"c": c, **_matmul_inputs(c, g)}
    return {"c": c, **_attn_inputs(c, g)}


# ------------------------------------------------------------ plain forms ----
def _rope_plain(x, w, cos, sin, rot, layout, eps):
    y = x.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + eps) * w
    r, rest = y[..., :rot], y[..., rot:]
    if layout == "half":
        x1, x2 = r[..., :rot // 2], r[..., rot // 2:]
        r = torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1)
    else:
        x1, x2 = r[..., 0::2], r[..., 1::2]
        r = torch.stack([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1).flatten(-2)
    return torch.cat([r, rest], -1).to(x.dtype)


def _quant_plain(x, rows):
    m, k = x.shape
    mb, kb = -(-m // rows), -(-k // BLK)
    f = torch.nn.functional.pad(x.float(), (0, kb * BLK - k, 0, mb * rows - m)).view(mb, rows, kb, BLK)
    s = f.abs().amax((1, 3)).clamp(min=1e-30) / 448.0
    codes = (f / s[:, None, :, None]).to(torch.float8_e4m3fn)
    return codes.view(mb * rows, kb * BLK)[:m, :k], s


def _matmul_plain(a8, sa, b8, sb, bias, dtype):
    k, n = a8.shape[1], b8.shape[0]
    a = a8.float() * sa.repeat_interleave(BLK, 1)[:, :k]
    b = b8.float() * sb.repeat_interleave(BLK, 0)[:n].repeat_interleave(BLK, 1)[:, :k]
    c = a @ b.t()
    return (c if bias is None else c + bias).to(dtype)


def _attn_plain(q, k, v, ql, kl, causal):
    hq, tq, d = q.shape[1:]
    hk, tk = k.shape[1:3]
    qf = q[0].float() * d ** -0.5
    kf, vf = (x[0].float().repeat_interleave(hq // hk, 0) for x in (k, v))
    ids = torch.arange(ql.numel(), device=q.device)
    sq, sk = ids.repeat_interleave(ql, output_size=tq), ids.repeat_interleave(kl, output_size=tk)
    # position of the last key that a causal row sees, among all keys
    last = torch.arange(tq, device=q.device) - (ql.cumsum(0) - kl.cumsum(0))[sq]
    hide = sq[:, None] != sk
    if causal:
        hide |= torch.arange(tk, device=q.device) > last[:, None]
    s = (qf @ kf.transpose(1, 2)).masked_fill_(hide, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(m.masked_fill_(m == -math.inf, 0.0)).exp_()
    l = p.sum(-1, keepdim=True)
    o = (p @ vf) / l.masked_fill(l == 0, 1.0)
    return o.to(q.dtype).unsqueeze(0)


def run(state):
    c = state["c"]
    if own:
        return _run_own(state, c)
    if c["op"] == "rope":
        a = (state["cos"], state["sin"], c["rot"], c["layout"], state["eps"])
        return [_rope_plain(state["q"], state["qw"], *a), _rope_plain(state["k"], state["kw"], *a)]
    if c["op"] == "quant":
        return list(_quant_plain(state["x"], c["rows"]))
    if c["op"] == "matmul":
        return _matmul_plain(state["a8"], state["sa"], state["b8"], state["sb"], state["bias"], DTYPES[c["dtype"]])
    return _attn_plain(state["q"], state["k"], state["v"], state["ql"], state["kl"], c["causal"])


def _run_own(state, c):
    from comfyui_vc_attention_b200 import vc_attention as vc
    if c["op"] == "rope":
        return list(vc.qk_norm_rope(state["q"], state["k"], state["cos"], state["sin"], state["qw"], state["kw"],
                                    layout=c["layout"], eps=state["eps"]))
    if c["op"] == "quant":
        b = vc.quantize_blocks(state["x"], rows=c["rows"])
        return [b.codes, b.scale]
    if c["op"] == "matmul":
        return vc.matmul_blocks(vc.Fp8Blocks(state["a8"], state["sa"], 1), vc.Fp8Blocks(state["b8"], state["sb"], BLK),
                                bias=state["bias"], dtype=DTYPES[c["dtype"]])
    return vc.packed_attention(state["q"], state["k"], state["v"], state["plan"])


# ------------------------------------------------------- work and 64 bits ----
def _pairs(c):
    """Number of (query, key) pairs of one head that take part."""
    t = 0
    for a, b in zip(_lens(c["q_lens"]), _lens(c["k_lens"])):
        if not c["causal"]:
            t += a * b
        else:   # row i sees max(0, i + 1 + b - a) keys
            first = max(0, a - b)
            r = a - first
            t += r * (first + 1 + b - a) + r * (r - 1) // 2
    return t


def work(case):
    c = case
    es = ES[c["dtype"]]
    if c["op"] == "rope":
        x = c["b"] * c["n"] * (c["hq"] + c["hk"]) * c["d"]
        return {"bytes": 2 * es * x + 4 * c["n"] * c["rot"] + 8 * c["d"], "flops": 7 * x}
    if c["op"] == "quant":
        x = c["m"] * c["k"]
        return {"bytes": (es + 1) * x + 4 * -(-c["m"] // c["rows"]) * -(-c["k"] // BLK), "flops": 3 * x}
    if c["op"] == "matmul":
        m, n, k = c["m"], c["n"], c["k"]
        kb = -(-k // BLK)
        return {"bytes": (m + n) * k + es * m * n + 4 * kb * (m + -(-n // BLK)) + (4 * n if c["bias"] else 0),
                "flops": 2 * m * n * k}
    tq, tk = sum(_lens(c["q_lens"])), sum(_lens(c["k_lens"]))
    return {"bytes": 2 * es * c["d"] * (c["hq"] * tq + c["hk"] * tk), "flops": 4 * c["d"] * c["hq"] * _pairs(c)}


def _rope_exact(x, w, s, rot, layout):
    """The rotation as a product of complex numbers, in 64 bits."""
    x = x.double()
    y = w.double() * x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + s["eps"])
    turn = torch.complex(s["cos"].double(), s["sin"].double())
    h = rot // 2
    i, j = ((slice(0, h), slice(h, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2)))
    z = torch.complex(y[..., i], y[..., j]) * turn
    out = y.clone()
    out[..., i], out[..., j] = z.real, z.imag
    return out


def _e4m3_exact(v):
    """Nearest E4M3 value (4 significant bits, least step 2^-9, ties to even), in 64 bits."""
    step = torch.exp2(torch.frexp(v)[1].double() - 4).clamp(min=2.0 ** -9)
    return (torch.round(v / step) * step).clamp(-448, 448)


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["op"] == "rope":
        return [_rope_exact(s["q"], s["qw"], s, c["rot"], c["layout"]),
                _rope_exact(s["k"], s["kw"], s, c["rot"], c["layout"])]
    if c["op"] == "quant":
        x, rows = s["x"].double(), c["rows"]
        scale = torch.empty(-(-c["m"] // rows), -(-c["k"] // BLK), dtype=torch.float64, device="cuda")
        codes = torch.empty_like(x)
        for j in range(scale.shape[1]):
            part = x[:, j * BLK:(j + 1) * BLK]
            top = torch.nn.functional.pad(part.abs().amax(1), (0, scale.shape[0] * rows - c["m"])).view(-1, rows).amax(1)
            scale[:, j] = top.clamp(min=1e-30) / 448
            codes[:, j * BLK:(j + 1) * BLK] = _e4m3_exact(part / scale[:, j].repeat_interleave(rows)[:c["m"], None])
        return [codes, scale]
    if c["op"] == "matmul":
        out = torch.zeros(c["m"], c["n"], dtype=torch.float64, device="cuda")
        if s["bias"] is not None:
            out += s["bias"].double()
        row = torch.arange(c["n"], device="cuda") // BLK
        for j in range(-(-c["k"] // BLK)):
            a, b = (s[n][:, j * BLK:(j + 1) * BLK].to(torch.float64) for n in ("a8", "b8"))
            out += (a @ b.t()) * s["sa"][:, j, None].double() * s["sb"][row, j].double()
        return out
    ql, kl, rep = _lens(c["q_lens"]), _lens(c["k_lens"]), c["hq"] // c["hk"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    q0 = k0 = 0
    for a, b in zip(ql, kl):
        for h in range(c["hq"]):
            kk, vv = (s[n][0, h // rep, k0:k0 + b].double() for n in ("k", "v"))
            x = s["q"][0, h, q0:q0 + a].double() @ kk.t() / math.sqrt(c["d"])
            if c["causal"]:
                x += torch.triu(torch.full((a, b), -math.inf, dtype=torch.float64, device="cuda"), b - a + 1)
            live = (x > -math.inf).any(1)
            out[0, h, q0:q0 + a][live] = torch.softmax(x[live], 1) @ vv
        q0, k0 = q0 + a, k0 + b
    return out
