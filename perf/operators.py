"""Performance cases of the decoder-layer operators around attention: the
projections with their epilogue, the mixture-of-experts layer for a few tokens
and rotary positions of several axes.

listed() holds the cases, draw() more of the same ranges.  prepare() makes
what a program has in hand before the call, run() is one pass through the
operator, exact() the same pass from its definition in 64 bits, work() the
bytes and operations that the pass cannot do without.  With `own` false run()
computes the operator in elementary torch operations in 32 bits (angles in
64), rounded once at the end; with `own` true it calls this library.

Kinds of case:
  linear  out = act(x W^T + bias) + residual, or with a gated weight
          out = act(x Wg^T + bg) * (x Wu^T + bu) + residual
  moe     softmax over the router's logits, the top k experts of each token,
          act(x Wg^T) * (x Wu^T) and the product with the down weight in each,
          summed with the routing weights
  rope    query and key rotated by positions of several axes (in place), with
          the rotated key and the value stored into the paged cache or not
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
BASE = 1000000.0
TABLE = 4096  # positions of a cos / sin table


def listed():
    return [
        # The attention output product of one decoding sequence with the
        # residual added: the smallest call, one stream of the weight.
        dict(name="linear_decode_o", kind="linear", m=1, n=4096, k=4096, act=None, gated=False,
             bias=False, residual=True, xpad=0, dtype="f16"),
        # Gate and up of a decode batch, their product formed in the epilogue.
        dict(name="linear_decode_gated", kind="linear", m=24, n=14336, k=4096, act="silu",
             gated=True, bias=False, residual=False, xpad=0, dtype="bf16"),
        # The down product of a chunk of a prompt between decode steps: few
        # rows, a long K, the residual added.
        dict(name="linear_chunk_down", kind="linear", m=333, n=4096, k=14336, act=None,
             gated=False, bias=False, residual=True, xpad=0, dtype="bf16"),
        # Patch embedding of an image tower: 14 x 14 x 3 pixels to a row, rows
        # not in whole 16-byte words, bias and activation, positions added.
        dict(name="linear_patches", kind="linear", m=2917, n=1152, k=588, act="gelu_tanh",
             gated=False, bias=True, residual=True, xpad=0, dtype="f16"),
        # Gate and up of a full prefill batch: the largest product.
        dict(name="linear_prefill_gated", kind="linear", m=8192, n=14336, k=4096, act="silu",
             gated=True, bias=False, residual=False, xpad=0, dtype="bf16"),
        # One sequence decodes with few large experts: two of eight are read.
        dict(name="moe_b1_large", kind="moe", tokens=1, pad=0, hidden=4096, inter=14336, experts=8,
             top_k=2, renorm=True, logits="f32", dtype="bf16"),
        # A few sequences decode with many small experts.
        dict(name="moe_b4_small", kind="moe", tokens=4, pad=0, hidden=2048, inter=768, experts=128,
             top_k=8, renorm=True, logits="f32", dtype="f16"),
        # A decode batch in a graph of fixed size: three padded rows route
        # nowhere; weights of the whole softmax.
        dict(name="moe_b64_padded", kind="moe", tokens=64, pad=3, hidden=2048, inter=1408,
             experts=64, top_k=6, renorm=False, logits="same", dtype="bf16"),
        # A large decode batch: every expert is read for some rows.
        dict(name="moe_b256", kind="moe", tokens=256, pad=0, hidden=4096, inter=1024, experts=128,
             top_k=8, renorm=True, logits="f32", dtype="bf16"),
        # One decode step of four sequences, (time, height, width) interleaved
        # over the frequencies, angles from the model's table.
        dict(name="rope_decode", kind="rope", tokens=4, heads=32, kv_heads=8, head=128, rot=128,
             axes=3, layout="interleaved", neox=True, table=True, cache=True, block=16, far=0,
             dtype="f16", seed=1),
        # A prefill batch of text and images at far positions, the axes in
        # ranges of the frequencies, angles computed.
        dict(name="rope_prefill", kind="rope", tokens=8191, heads=32, kv_heads=8, head=128, rot=128,
             axes=3, layout="contiguous", neox=True, table=False, cache=True, block=16,
             far=200000, dtype="bf16", seed=2),
        # An image tower: (height, width) with frequencies of their own, heads
        # of 80, query and key as slices of one product's rows.
        dict(name="rope_image", kind="rope", tokens=16380, heads=16, kv_heads=16, head=80, rot=80,
             axes=2, layout="per_axis", neox=True, table=False, cache=False, block=0, far=0,
             dtype="f16", seed=3),
    ]


# ----------------------------------------------------------------- drawing

HEADS = [(32, 8), (32, 8), (16, 2), (16, 4), (16, 16), (40, 8), (64, 8), (32, 32)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    kind = rng.choice(["linear", "linear", "moe", "moe", "rope"])
    dtype = rng.choice(["f16", "bf16"])
    if kind == "linear":
        # widths in whole 16-byte words mostly, any width at times
        unit = rng.choice([64, 64, 8, 1])
        n = max(16, unit * max(1, _log(rng, 64, 28672) // unit))
        k = max(16, unit * max(1, _log(rng, 64, 16384) // unit))
        gated = rng.random() < 0.35
        if gated:
            n = max(16, n // 2)
        act = rng.choice(["silu", "gelu", "gelu_tanh"] if gated
                         else [None, None, "relu", "silu", "gelu", "gelu_tanh"])
        return dict(kind=kind, m=_log(rng, 1, 8192), n=n, k=k, act=act, gated=gated,
                    bias=rng.random() < 0.5, residual=rng.random() < 0.4,
                    xpad=rng.choice([0, 0, 0, 64]), dtype=dtype)
    if kind == "moe":
        experts = rng.choice([4, 8, 8, 16, 32, 60, 64, 128, 128, 160])
        tokens = _log(rng, 1, 512)
        return dict(kind=kind, tokens=tokens, pad=rng.choice([0, 0, min(tokens - 1, 5)]),
                    hidden=64 * _log(rng, 8, 112), inter=32 * _log(rng, 8, 448), experts=experts,
                    top_k=rng.randint(1, min(8, experts)), renorm=rng.random() < 0.7,
                    logits=rng.choice(["f32", "same"]), dtype=dtype)
    heads, kv_heads = rng.choice(HEADS)
    head = rng.choice([64, 80, 96, 128, 128, 128])
    layout = rng.choice(["contiguous", "interleaved", "per_axis"])
    table = layout != "per_axis" and rng.random() < 0.5
    cache = layout != "per_axis" and rng.random() < 0.7
    return dict(kind=kind, tokens=_log(rng, 1, 16384 if not cache else 8192), heads=heads,
                kv_heads=kv_heads, head=head, rot=rng.choice([head, head, 32]),
                axes=2 if layout == "per_axis" else rng.choice([2, 3, 3, 4]), layout=layout,
                neox=rng.random() < 0.75, table=table, cache=cache,
                block=rng.choice([16, 16, 32, 64]) if cache else 0,
                far=0 if table else rng.choice([0, 30000, 200000]), dtype=dtype,
                seed=rng.randrange(1 << 20))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        m = most.setdefault(c["kind"], {"bytes": 0, "flops": 0})
        for key in m:
            m[key] = max(m[key], w[key])
    while True:
        c = _draw_once(rng)
        w, m = work(c), most[c["kind"]]
        if c["kind"] == "moe" and _expert_bytes(c) > 3.3e9:
            continue
        if all(w[key] <= m[key] for key in m):
            return c


# ------------------------------------------------------------ sizes of a case

def _expert_bytes(c):
    return 2.0 * c["experts"] * 3 * c["hidden"] * c["inter"]


def work(c):
    """Bytes and operations of one pass that it cannot do without."""
    if c["kind"] == "linear":
        rows = c["n"] * (2 if c["gated"] else 1)
        by = c["m"] * c["k"] + rows * c["k"] + c["m"] * c["n"] * (2 if c["residual"] else 1)
        by += rows if c["bias"] else 0
        return {"bytes": 2 * by, "flops": 2 * c["m"] * rows * c["k"]}
    if c["kind"] == "moe":
        t, e, k = c["tokens"] - c["pad"], c["experts"], c["top_k"]
        read = e * (1.0 - (1.0 - k / e) ** t)  # experts that some token chose, expected
        expert = 3 * c["hidden"] * c["inter"]
        size = 4 if c["logits"] == "f32" else 2
        by = 2 * read * expert + 4 * c["tokens"] * c["hidden"] + c["tokens"] * (e * size + 8 * k)
        return {"bytes": by, "flops": 2 * t * k * expert}
    t, q, kv = c["tokens"], c["heads"] * c["head"], c["kv_heads"] * c["head"]
    by = 4 * t * q + (8 * t * kv if c["cache"] else 4 * t * kv) + 8 * t * c["axes"]
    by += 8 * t if c["cache"] else 0
    return {"bytes": by, "flops": 3 * t * (q + kv)}


# ------------------------------------------------------------------- inputs

class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(self, *shape, scale=1.0, dtype=torch.float16):
        out = torch.empty(shape, dtype=dtype, device="cuda")
        flat = out.view(-1)
        for i in range(0, flat.numel(), 1 << 27):  # bounds the 32-bit intermediate
            part = flat[i:i + (1 << 27)]
            part.copy_(torch.randn(part.numel(), generator=self.g, device="cuda").mul_(scale))
        return out

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")


def sections(c):
    """Frequencies of each axis: those of an image evenly, else a quarter (in
    ranges) or about an equal part (interleaved) to the first axis and the rest
    to the others evenly."""
    half, axes = c["rot"] // 2, c["axes"]
    if c["layout"] == "per_axis":
        other = half // axes
    elif c["layout"] == "interleaved":
        other = half // axes - half // 64
    else:
        other = half * 3 // (4 * (axes - 1))
    return [half - (axes - 1) * other] + [other] * (axes - 1)


def axis_of(c):
    """Axis of each frequency.  Interleaved: frequency i takes axis i % axes
    while that axis has frequencies left, then the first axis."""
    sec, half = sections(c), c["rot"] // 2
    if c["layout"] != "interleaved":
        return [a for a, n in enumerate(sec) for _ in range(n)]
    out = []
    for i in range(half):
        a = i % c["axes"]
        out.append(a if a > 0 and i < c["axes"] * sec[a] else 0)
    return out


def _positions(c):
    """int64 [axes, tokens]: spans of text, whose axes agree, and grids of
    image tokens; for two axes (rows, columns) of grids alone."""
    r, t, axes = random.Random(c["seed"]), c["tokens"], c["axes"]
    cols, at, n = [[] for _ in range(axes)], c["far"] + r.randrange(64), 0
    limit = TABLE if c["table"] else 1 << 40
    while n < t:
        if axes > 2 and r.random() < 0.5:
            m = min(t - n, r.randint(1, 200))
            for col in cols:
                col.extend(range(at, at + m))
            at += m
        else:
            h, w = r.randint(2, 60), r.randint(2, 60)
            m = min(t - n, h * w)
            first = 0 if axes == 2 else at
            for a, col in enumerate(cols):
                if a == axes - 1:
                    col.extend(first + i % w for i in range(m))
                elif a == axes - 2:
                    col.extend(first + i // w for i in range(m))
                else:
                    col.extend([at] * m)
            at += max(h, w)
        n += m
        if at + 256 > limit:
            at = r.randrange(64)
    return torch.tensor(cols, dtype=torch.int64).cuda()


def _table(c):
    """float32 [positions, rot] cos then sin, as a model keeps it."""
    inv = BASE ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device="cuda") / c["rot"])
    a = torch.arange(TABLE, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).float()


def prepare(c, seed):
    r, dt = _Rand(seed), DTYPES[c["dtype"]]
    if own:
        _library()
    s = {"case": c}
    if c["kind"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        rows = 2 * n if c["gated"] else n
        s.update(x=r.normal(m, k + c["xpad"], dtype=dt)[:, :k],
                 w=r.normal(rows, k, scale=k ** -0.5, dtype=dt),
                 bias=r.normal(rows, scale=0.5, dtype=dt) if c["bias"] else None,
                 residual=r.normal(m, n, dtype=dt) if c["residual"] else None,
                 out=torch.empty(m, n, dtype=dt, device="cuda"))
        return s
    if c["kind"] == "moe":
        t, h, i, e = c["tokens"], c["hidden"], c["inter"], c["experts"]
        logits = r.normal(t, e, scale=1.5, dtype=torch.float32)
        logits[t - c["pad"]:] = -math.inf
        s.update(x=r.normal(t, h, dtype=dt),
                 w_in=r.normal(e, 2 * i, h, scale=h ** -0.5, dtype=dt),
                 w_out=r.normal(e, h, i, scale=i ** -0.5, dtype=dt),
                 logits=logits if c["logits"] == "f32" else logits.to(dt),
                 out=torch.empty(t, h, dtype=dt, device="cuda"),
                 ids=torch.empty(t, c["top_k"], dtype=torch.int32, device="cuda"),
                 weights=torch.empty(t, c["top_k"], dtype=torch.float32, device="cuda"))
        return s
    t, h, kv, d = c["tokens"], c["heads"], c["kv_heads"], c["head"]
    qkv = r.normal(t, (h + 2 * kv) * d, dtype=dt)
    s.update(q=qkv[:, :h * d], k=qkv[:, h * d:(h + kv) * d], v=qkv[:, (h + kv) * d:],
             positions=_positions(c), angles=_table(c) if c["table"] else None)
    if c["cache"]:
        pages = max(4, (t + t // 4 + c["block"] - 1) // c["block"])
        shape = (pages, kv, c["block"], d)
        s.update(slots=r.perm(pages * c["block"])[:t].contiguous(),
                 kc=torch.zeros(shape, dtype=dt, device="cuda"),
                 vc=torch.zeros(shape, dtype=dt, device="cuda"))
    return s


# -------------------------------------------------------------------- one pass

def _library():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "teco-ops_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import tecoops
    return tecoops


def _run_own(s):
    c, tecoops = s["case"], _library()
    if c["kind"] == "linear":
        tecoops.linear(s["x"], s["w"], s["out"], bias=s["bias"], residual=s["residual"],
                       activation=c["act"], gated=c["gated"])
        return s["out"]
    if c["kind"] == "moe":
        tecoops.moe_layer(s["x"], s["w_in"], s["w_out"], s["logits"], c["top_k"], s["out"],
                          renormalize=c["renorm"], topk_ids=s["ids"], topk_weights=s["weights"])
        return {"out": s["out"], "ids": s["ids"], "weights": s["weights"]}
    if c["cache"]:
        tecoops.rotary_axes_reshape_and_cache(
            s["positions"], s["q"], s["k"], s["v"], s["slots"], s["kc"], s["vc"], c["head"],
            sections(c), cos_sin_cache=s["angles"], is_neox=c["neox"], base=BASE,
            rot_dim=c["rot"], layout=c["layout"])
        return {"q": s["q"], "kc": s["kc"], "vc": s["vc"]}
    tecoops.rotary_embedding_axes(s["positions"], s["q"], s["k"], c["head"], sections(c),
                                  cos_sin_cache=s["angles"], is_neox=c["neox"], base=BASE,
                                  rot_dim=c["rot"], layout=c["layout"])
    return {"q": s["q"], "k": s["k"]}


def _act(y, name):
    if name == "relu":
        return y.clamp(min=0)
    if name == "silu":
        return y / (1 + torch.exp(-y))
    if name == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    return y


def _plain_linear(s):
    c = s["case"]
    y = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        y += s["bias"].float()
    if c["gated"]:
        y = _act(y[:, :c["n"]], c["act"]) * y[:, c["n"]:]
    else:
        y = _act(y, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _plain_moe(s):
    c = s["case"]
    logits, x = s["logits"].float(), s["x"].float()
    best, ids = torch.sort(logits, dim=-1, descending=True, stable=True)
    best, ids = best[:, :c["top_k"]], ids[:, :c["top_k"]]
    chosen = best > -math.inf
    over = best if c["renorm"] else logits
    top = best[:, :1].clamp(min=-3e38)
    weights = torch.exp(best - top) / torch.exp(over - top).sum(-1, keepdim=True)
    weights = torch.where(chosen, weights, 0.0)
    ids = torch.where(chosen, ids, -1)
    rows = {}
    for t, of_token in enumerate(ids.tolist()):
        for j, e in enumerate(of_token):
            if e >= 0:
                rows.setdefault(e, []).append((t, j))
    out = torch.zeros_like(x)
    for e, pairs in sorted(rows.items()):
        at = torch.tensor(pairs, device="cuda")
        t, j = at[:, 0], at[:, 1]
        y = x[t] @ s["w_in"][e].float().t()
        y = _act(y[:, :c["inter"]], "silu") * y[:, c["inter"]:]
        out.index_add_(0, t, weights[t, j][:, None] * (y @ s["w_out"][e].float().t()))
    return {"out": out.to(s["x"].dtype), "ids": ids.int(), "weights": weights}


def _rotated(c, x, cos, sin, heads):
    """x [tokens, heads * head] turned by cos / sin [tokens, rot / 2]."""
    x = x.reshape(x.shape[0], heads, c["head"])
    half, cos, sin = c["rot"] // 2, cos[:, None], sin[:, None]
    turn, rest = x[..., :c["rot"]], x[..., c["rot"]:]
    if c["neox"]:
        a, b = turn[..., :half], turn[..., half:]
        turn = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = turn[..., 0::2], turn[..., 1::2]
        turn = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turn, rest], -1)


def _plain_rope(s):
    c, half = s["case"], s["case"]["rot"] // 2
    axis = torch.tensor(axis_of(c), device="cuda")
    pos = s["positions"][axis].t()  # [tokens, rot / 2]
    if s["angles"] is not None:
        i = torch.arange(half, device="cuda")
        cos, sin = s["angles"][pos, i], s["angles"][pos, half + i]
    else:
        i, n = torch.arange(half, dtype=torch.float64, device="cuda"), float(half)
        if c["layout"] == "per_axis":
            sec = torch.tensor(sections(c), device="cuda")
            i = i - (torch.cumsum(sec, 0) - sec)[axis]
            n = sec[axis].double()
        angle = pos.double() * BASE ** (-i / n)
        cos, sin = angle.cos().float(), angle.sin().float()
    q = _rotated(c, s["q"].float(), cos, sin, c["heads"]).to(s["q"].dtype)
    k = _rotated(c, s["k"].float(), cos, sin, c["kv_heads"]).to(s["k"].dtype)
    s["q"].copy_(q.flatten(1))
    if not c["cache"]:
        s["k"].copy_(k.flatten(1))
        return {"q": s["q"], "k": s["k"]}
    page, row = s["slots"] // c["block"], s["slots"] % c["block"]
    s["kc"][page, :, row] = k
    s["vc"][page, :, row] = s["v"].reshape(k.shape)
    return {"q": s["q"], "kc": s["kc"], "vc": s["vc"]}


def run(s):
    if own:
        return _run_own(s)
    return {"linear": _plain_linear, "moe": _plain_moe, "rope": _plain_rope}[s["case"]["kind"]](s)


# ------------------------------------------------------------- 64-bit results

def _act64(y, name):
    if name == "relu":
        return torch.where(y > 0, y, torch.zeros_like(y))
    if name == "silu":
        return y * torch.sigmoid(y)
    if name == "gelu":
        return y * 0.5 * torch.erfc(-y / math.sqrt(2))
    if name == "gelu_tanh":
        return y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
    return y


def _exact_linear(c, s):
    n, x = c["n"], s["x"].double()
    out = torch.empty(c["m"], n, dtype=torch.float64, device="cuda")
    for lo in range(0, n, 4096):
        hi = min(n, lo + 4096)
        y = x @ s["w"][lo:hi].double().t().contiguous()
        if c["bias"]:
            y += s["bias"][lo:hi].double()
        y = _act64(y, c["act"])
        if c["gated"]:
            up = x @ s["w"][n + lo:n + hi].double().t().contiguous()
            if c["bias"]:
                up += s["bias"][n + lo:n + hi].double()
            y *= up
        out[:, lo:hi] = y
    return out + s["residual"].double() if c["residual"] else out


def _exact_moe(c, s):
    logits, x, i = s["logits"].double().cpu(), s["x"].double(), c["inter"]
    ids = torch.full((c["tokens"], c["top_k"]), -1, dtype=torch.int32)
    weights = torch.zeros(c["tokens"], c["top_k"], dtype=torch.float64)
    pairs = {}
    for t in range(c["tokens"]):
        row = logits[t].tolist()
        order = sorted((e for e in range(c["experts"]) if row[e] > -math.inf),
                       key=lambda e: (-row[e], e))[:c["top_k"]]
        among = order if c["renorm"] else [e for e in range(c["experts"]) if row[e] > -math.inf]
        total = sum(math.exp(row[e] - row[order[0]]) for e in among) if order else 1.0
        for j, e in enumerate(order):
            ids[t, j] = e
            weights[t, j] = math.exp(row[e] - row[order[0]]) / total
            pairs.setdefault(e, []).append((t, float(weights[t, j])))
    out = torch.zeros(c["tokens"], c["hidden"], dtype=torch.float64, device="cuda")
    for e, of_expert in pairs.items():
        t = torch.tensor([p[0] for p in of_expert], device="cuda")
        w = torch.tensor([p[1] for p in of_expert], dtype=torch.float64, device="cuda")
        w_in = s["w_in"][e].double()
        gate = x[t] @ w_in[:i].t().contiguous()
        up = x[t] @ w_in[i:].t().contiguous()
        y = (_act64(gate, "silu") * up) @ s["w_out"][e].double().t().contiguous()
        out[t] += w[:, None] * y  # a token is at most once in an expert's rows
    return {"out": out, "ids": ids.cuda(), "weights": weights.cuda()}


def _exact_rope(c, s):
    half, t = c["rot"] // 2, c["tokens"]
    cos = torch.empty(t, half, dtype=torch.float64, device="cuda")
    sin = torch.empty_like(cos)
    sec, axis = sections(c), axis_of(c)
    for i, a in enumerate(axis):
        p = s["positions"][a]
        if c["table"]:
            cos[:, i], sin[:, i] = s["angles"][p, i].double(), s["angles"][p, half + i].double()
            continue
        j, n = (i - sum(sec[:a]), sec[a]) if c["layout"] == "per_axis" else (i, half)
        angle = p.double() * BASE ** (-j / n)
        cos[:, i], sin[:, i] = torch.cos(angle), torch.sin(angle)

    def turned(x, heads):
        x = x.double().reshape(t, heads, c["head"])
        y = x.clone()
        one = slice(0, half) if c["neox"] else slice(0, c["rot"], 2)
        two = slice(half, c["rot"]) if c["neox"] else slice(1, c["rot"], 2)
        y[..., one] = x[..., one] * cos[:, None] - x[..., two] * sin[:, None]
        y[..., two] = x[..., two] * cos[:, None] + x[..., one] * sin[:, None]
        return y

    q, k = turned(s["q"], c["heads"]).flatten(1), turned(s["k"], c["kv_heads"])
    if not c["cache"]:
        return {"q": q, "k": k.flatten(1)}
    kc, vc = s["kc"].double(), s["vc"].double()
    kc[s["slots"] // c["block"], :, s["slots"] % c["block"]] = k
    vc[s["slots"] // c["block"], :, s["slots"] % c["block"]] = s["v"].double().reshape(k.shape)
    return {"q": q, "kc": kc, "vc": vc}


def exact(c, seed):
    s = prepare(c, seed)
    return {"linear": _exact_linear, "moe": _exact_moe, "rope": _exact_rope}[c["kind"]](c, s)
