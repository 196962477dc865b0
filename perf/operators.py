"""What is measured of the device-buffer operators (`laya_rust_b200.ops`).

Two operators that run side by side in an encoder layer:

  lora  a projection shared by many requests, each with its own low-rank
        adapter: y = x W^T + bias + s_a (x A_a^T) B_a^T, the adapter `a` given
        per segment of rows (or none)
  rope  rotary positions of the queries and keys that projection leaves

With `own` false `run` computes them from elementary torch operations in 32
bits (angles in 64); with `own` true it calls the framework's operators.
`exact` is the definition in 64 bits, written apart from both.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}


def _lora(name, type, rows, segs, adapters, bare, rank, mixed, inn, out, bias, mix):
    """rows in `segs` segments over `adapters` adapters, `bare` of the segments without one; rank: of every adapter, or
    the largest where `mixed`; mix: which split into segments."""
    c = dict(op="lora", type=type, rows=rows, segs=segs, adapters=adapters, bare=bare, rank=rank, mixed=mixed, inn=inn,
             out=out, bias=bias, mix=mix)
    return dict(c, name=name) if name else c


def _rope(name, type, tokens, segs, q_heads, k_heads, dim, rot, layout, where, scaling, factor, inverse, packed):
    """tokens in `segs` sequences; where: "start" (positions count from 0 in each sequence) or "far" (each sequence starts
    at its own far position, as a token appended to a long context does); packed: q and k are columns of one q|k|v buffer."""
    c = dict(op="rope", type=type, tokens=tokens, segs=segs, q_heads=q_heads, k_heads=k_heads, dim=dim, rot=rot,
             layout=layout, where=where, scaling=scaling, factor=factor, inverse=inverse, packed=packed)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token of one request through the attention input projection: latency alone
        _lora("lora-one-row", "f16", 1, 1, 1, 0, 16, False, 1024, 3072, False, 0),
        # 48 single rows, every one of another request with an adapter of its own
        _lora("lora-48-adapters", "bf16", 48, 48, 48, 0, 16, False, 1024, 3072, False, 1),
        # one request of two questions: few rows, the second FFN projection (long inner sum, few output columns)
        _lora("lora-request", "f16", 179, 2, 1, 0, 32, False, 2624, 1024, False, 2),
        # odd everything: widths that are no multiple of any tile, a rank of 11, some segments without an adapter
        _lora("lora-odd", "bf16", 1357, 23, 5, 4, 11, True, 1000, 1531, True, 3),
        # the packed 128-question batch, 16 tenants, attention input projection
        _lora("lora-batch-qkv", "f16", 9872, 128, 16, 0, 16, False, 1024, 3072, False, 4),
        # long states, high mixed ranks, the wide FFN projection: the largest product
        _lora("lora-long-ffn", "f16", 16384, 32, 8, 2, 128, True, 1024, 5248, False, 5),
        # one token: latency alone
        _rope("rope-one-token", "f16", 1, 1, 16, 16, 64, 64, "half", "far", "none", 1.0, False, True),
        # 64 requests each at its own far position, grouped keys, part of the head rotated
        _rope("rope-64-far", "bf16", 64, 64, 32, 8, 128, 64, "interleaved", "far", "parts", 8.0, False, False),
        # the packed 128-question batch in the q|k|v buffer
        _rope("rope-batch-qkv", "f16", 9872, 128, 16, 16, 64, 64, "half", "start", "none", 1.0, False, True),
        # odd head and rotated part, 32 bits, backwards
        _rope("rope-odd-back", "f32", 3001, 7, 12, 3, 80, 20, "half", "start", "linear", 4.0, True, False),
        # one context of 65536 tokens at four times the trained length
        _rope("rope-long", "bf16", 65536, 1, 32, 8, 128, 128, "half", "start", "base", 4.0, False, False),
    ]


LARGEST_PRODUCT = 16384 * 1024 * 5248
LARGEST_ROPE = 65536 * 40 * 128


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.55:
        inn, out = _spread(rng, 64, 4096), _spread(rng, 64, 5248)
        if rng.random() < 0.5:
            inn, out = (inn + 63) // 64 * 64, (out + 63) // 64 * 64
        rows = _spread(rng, 1, min(16384, LARGEST_PRODUCT // (inn * out)))
        segs = _spread(rng, 1, min(rows, 256))
        adapters = _spread(rng, 1, min(segs, 64))
        bare = rng.randrange(0, segs // 3 + 1)
        return _lora(None, rng.choice(["f16", "bf16"]), rows, segs, adapters, bare, _spread(rng, 1, 128),
                     rng.random() < 0.5, inn, out, rng.random() < 0.3, rng.randrange(1 << 20))
    q_heads, dim = _spread(rng, 1, 64), 2 * _spread(rng, 8, 128)
    if rng.random() < 0.6:
        dim = (dim + 15) // 16 * 16
    k_heads = max(1, q_heads // rng.choice([1, 2, 4, 8]))
    rot = dim if rng.random() < 0.5 else 2 * rng.randrange(1, dim // 2 + 1)
    tokens = _spread(rng, 1, min(65536, LARGEST_ROPE // ((q_heads + k_heads) * dim)))
    scaling = rng.choice(["none", "linear", "base", "parts"])
    if rot == 2 and scaling == "base":
        scaling = "linear"
    return _rope(None, rng.choice(["f16", "bf16", "f32"]), tokens, _spread(rng, 1, min(tokens, 256)), q_heads, k_heads, dim,
                 rot, rng.choice(["half", "interleaved"]), rng.choice(["start", "far"]), scaling,
                 1.0 if scaling == "none" else float(rng.choice([2, 4, 8, 16])), rng.random() < 0.3, rng.random() < 0.4)


# ---- shapes that follow from a case alone ------------------------------------
def _split(total, parts, rng):
    """`total` into `parts` whole numbers of at least 1."""
    cuts = sorted(rng.sample(range(1, total), parts - 1)) if parts > 1 else []
    ends = cuts + [total]
    return [b - a for a, b in zip([0] + cuts, ends)]


def _segments(case):
    """(rows of each segment, its adapter or -1, rank of each adapter)."""
    rng = random.Random(case["mix"])
    lens = _split(case["rows"], case["segs"], rng)
    slots = [i % case["adapters"] for i in range(case["segs"])]
    rng.shuffle(slots)
    for i in rng.sample(range(case["segs"]), case["bare"]):
        slots[i] = -1
    ranks = [rng.randrange(1, case["rank"] + 1) if case["mixed"] else case["rank"] for _ in range(case["adapters"])]
    ranks[0] = case["rank"]
    return lens, slots, ranks


def _up8(n):
    return (n + 7) // 8 * 8


def work(case):
    if case["op"] == "lora":
        lens, slots, ranks = _segments(case)
        m, k, n = case["rows"], case["inn"], case["out"]
        used = sum(ranks[s] for s in set(slots) if s >= 0)
        low = sum(ln * ranks[s] for ln, s in zip(lens, slots) if s >= 0)
        return {"bytes": 2 * (m * k + n * k + m * n + used * (k + n)) + (4 * n if case["bias"] else 0),
                "flops": 2 * m * k * n + 2 * low * (k + n)}
    el = case["tokens"] * (case["q_heads"] + case["k_heads"])
    return {"bytes": 2 * el * case["dim"] * BYTES[case["type"]] + 4 * case["tokens"], "flops": 3 * el * case["rot"]}


# ---- inputs ------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, shape, std):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32) * std


def _lora_inputs(case, seed):
    """x, W with rows padded to 16 bytes, the adapters and the bias: activations after a norm, weights as a linear layer
    holds them, adapters as training leaves them (A about 1/sqrt(in), B small), scale alpha / r = 2."""
    t = TYPES[case["type"]]
    g = _gen(seed)
    lens, slots, ranks = _segments(case)
    m, k, n = case["rows"], case["inn"], case["out"]
    x = torch.zeros(m, _up8(k), device=DEV, dtype=t)
    x[:, :k] = _normal(g, (m, k), 1.0).to(t)
    w = torch.zeros(n, _up8(k), device=DEV, dtype=t)
    w[:, :k] = _normal(g, (n, k), 0.02).to(t)
    a = [_normal(g, (r, k), k ** -0.5).to(t) for r in ranks]
    b = [_normal(g, (n, r), 0.02).to(t) for r in ranks]
    scale = [2.0 - 0.125 * (i % 5) for i in range(len(ranks))]
    bias = _normal(g, (n,), 0.5) if case["bias"] else None
    return x, w, a, b, scale, bias, lens, slots


def _positions(case):
    rng = random.Random(case["tokens"] * 7919 + case["segs"])
    pos = []
    for ln in _split(case["tokens"], case["segs"], rng):
        p0 = rng.randrange(1000, 1 << 20) if case["where"] == "far" else 0
        pos.extend(range(p0, p0 + ln))
    return pos


ROPE_BASE, TRAINED, LOW, HIGH = 10000.0, 8192.0, 1.0, 32.0


def _rope_inputs(case, seed):
    """q and k as an input projection leaves them, as [tokens, heads, dim] views."""
    t = TYPES[case["type"]]
    g = _gen(seed)
    n, hq, hk, d = case["tokens"], case["q_heads"], case["k_heads"], case["dim"]
    if case["packed"]:
        buf = _normal(g, (n, (hq + 2 * hk) * d), 1.0).to(t)
        q = buf[:, :hq * d].unflatten(1, (hq, d))
        k = buf[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d))
    else:
        q, k = _normal(g, (n, hq, d), 1.0).to(t), _normal(g, (n, hk, d), 1.0).to(t)
    return q, k, torch.tensor(_positions(case), dtype=torch.int32, device=DEV)


def prepare(case, seed):
    if case["op"] == "lora":
        x, w, a, b, scale, bias, lens, slots = _lora_inputs(case, seed)
        s = dict(case=case, x=x, w=w, bias=bias)
        if own:
            from laya_rust_b200 import ops
            s["lora"] = ops.Lora(ops.TYPE[case["type"]], case["inn"], case["out"], w.data_ptr(), w.stride(0),
                                 bias.data_ptr() if bias is not None else 0, slots=len(a))
            for i in range(len(a)):
                s["lora"].set(i, a[i].float().cpu().numpy(), b[i].float().cpu().numpy(), scale[i])
            s["plan"] = s["lora"].plan(lens, slots)
            s["y"] = torch.empty(case["rows"], _up8(case["out"]), device=DEV, dtype=x.dtype)
        else:
            owner = torch.repeat_interleave(torch.tensor(slots), torch.tensor(lens))
            s.update(a=a, b=b, scale=scale, rows=[(owner == i).nonzero()[:, 0].to(DEV) for i in range(len(a))])
        return s
    q, k, pos = _rope_inputs(case, seed)
    s = dict(case=case, q=q, k=k, pos=pos)
    if own:
        from laya_rust_b200 import ops
        scaling = {"none": None, "linear": ops.RopeScaling(ops.ROPE_LINEAR, case["factor"]),
                   "base": ops.RopeScaling(ops.ROPE_BASE, case["factor"]),
                   "parts": ops.RopeScaling(ops.ROPE_PARTS, case["factor"], TRAINED, LOW, HIGH)}[case["scaling"]]
        freqs, mscale = ops.rope_freqs(ROPE_BASE, case["rot"], scaling)
        s["spec"] = ops.RopeSpec(ops.TYPE[case["type"]], case["dim"], case["rot"], freqs,
                                 ops.ROPE_HALF if case["layout"] == "half" else ops.ROPE_INTERLEAVED, case["inverse"], mscale)
        s["out_q"], s["out_k"] = (torch.empty(v.shape, device=DEV, dtype=v.dtype) for v in (q, k))
    else:
        s["freqs"], s["mscale"] = _plain_freqs(case)
    return s


# ---- the plain forms -----------------------------------------------------------
def _plain_lora(s):
    case = s["case"]
    n, k = case["out"], case["inn"]
    x = s["x"][:, :k].float()
    y = x @ s["w"][:, :k].float().T
    if s["bias"] is not None:
        y += s["bias"]
    for rows, a, b, scale in zip(s["rows"], s["a"], s["b"], s["scale"]):
        if len(rows):
            y[rows] += scale * ((x[rows] @ a.float().T) @ b.float().T)
    return y.to(s["x"].dtype)


def _plain_freqs(case):
    """Frequencies in 64 bits and the factor on cos and sin."""
    rot, s = case["rot"], case["factor"]
    j = torch.arange(rot // 2, device=DEV, dtype=torch.float64)
    base, m = ROPE_BASE, 1.0
    if case["scaling"] == "base":
        base = ROPE_BASE * s ** (rot / (rot - 2))
    f = base ** (-2.0 * j / rot)
    if case["scaling"] == "linear":
        f = f / s
    elif case["scaling"] == "parts":
        turns = TRAINED * f / (2 * math.pi)
        keep = ((turns - LOW) / (HIGH - LOW)).clamp(0, 1)
        f = f / s * (1 - keep) + f * keep
        m = 0.1 * math.log(s) + 1.0
    return f, m


def _plain_rope_one(x, cos, sin, case):
    rot = case["rot"]
    v = x.float()
    out = v.clone()
    if case["layout"] == "half":
        a, b = v[..., :rot // 2], v[..., rot // 2:rot]
        out[..., :rot // 2] = a * cos - b * sin
        out[..., rot // 2:rot] = b * cos + a * sin
    else:
        a, b = v[..., 0:rot:2], v[..., 1:rot:2]
        out[..., 0:rot:2] = a * cos - b * sin
        out[..., 1:rot:2] = b * cos + a * sin
    return out.to(x.dtype)


def _plain_rope(s):
    case = s["case"]
    ang = s["pos"].double()[:, None] * s["freqs"][None, :]
    cos = (ang.cos() * s["mscale"]).float()[:, None, :]
    sin = (ang.sin() * (-s["mscale"] if case["inverse"] else s["mscale"])).float()[:, None, :]
    return [_plain_rope_one(s["q"], cos, sin, case), _plain_rope_one(s["k"], cos, sin, case)]


def run(state):
    case = state["case"]
    if not own:
        return _plain_lora(state) if case["op"] == "lora" else _plain_rope(state)
    from laya_rust_b200 import ops
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "lora":
        x, y = state["x"], state["y"]
        state["lora"].run(state["plan"], x.data_ptr(), x.stride(0), y.data_ptr(), y.stride(0), stream=stream)
        return y[:, :case["out"]]
    q, k, oq, ok = state["q"], state["k"], state["out_q"], state["out_k"]
    ops.rope(state["spec"], [ops.RopeTensor(v.data_ptr(), o.data_ptr(), v.shape[1], v.stride(0), v.stride(1), o.stride(0),
                                            o.stride(1)) for v, o in ((q, oq), (k, ok))],
             case["tokens"], pos=state["pos"].data_ptr(), stream=stream)
    return [oq, ok]


# ---- the definition in 64 bits -------------------------------------------------
def exact(case, seed):
    if case["op"] == "lora":
        x, w, a, b, scale, bias, lens, slots = _lora_inputs(case, seed)
        k = case["inn"]
        row_slot = torch.repeat_interleave(torch.tensor(slots, device=DEV), torch.tensor(lens, device=DEV))
        xd = x[:, :k].double()
        y = torch.einsum("mk,nk->mn", xd, w[:, :k].double())
        for i in range(len(a)):
            rows = (row_slot == i).nonzero()[:, 0]
            low = torch.einsum("mk,rk->mr", xd[rows], a[i].double()) * scale[i]
            y[rows] = y[rows] + torch.einsum("mr,nr->mn", low, b[i].double())
        return y if bias is None else y + bias.double()
    q, k, pos = _rope_inputs(case, seed)
    rot, s = case["rot"], case["factor"]
    f = []
    for j in range(rot // 2):
        v = math.exp(-2.0 * j / rot * math.log(ROPE_BASE))
        if case["scaling"] == "linear":
            v /= s
        elif case["scaling"] == "base":
            v *= s ** (-2.0 * j / (rot - 2))
        elif case["scaling"] == "parts":
            g = min(1.0, max(0.0, (TRAINED * v / (2.0 * math.pi) - LOW) / (HIGH - LOW)))
            v *= g + (1.0 - g) / s
        f.append(v)
    m = 0.1 * math.log(s) + 1.0 if case["scaling"] == "parts" else 1.0
    theta = torch.outer(pos.double(), torch.tensor(f, device=DEV, dtype=torch.float64))
    turn = torch.polar(torch.full_like(theta, m), -theta if case["inverse"] else theta)[:, None, :]
    outs = []
    for v in (q, k):
        o = v.double()
        if case["layout"] == "half":
            z = torch.complex(o[..., :rot // 2], o[..., rot // 2:rot]) * turn
            outs.append(torch.cat([z.real, z.imag, o[..., rot:]], dim=-1))
        else:
            z = torch.view_as_complex(o[..., :rot].unflatten(-1, (rot // 2, 2)).contiguous()) * turn
            outs.append(torch.cat([torch.view_as_real(z).flatten(-2), o[..., rot:]], dim=-1))
    return outs
