"""Performance cases of a decode path held in 4 bits: the norms of queries and
keys with the position rotation, the paged cache of 4-bit keys and values with
the attention that reads it, and products with 4-bit weights.

listed() holds the cases, draw() more of the same ranges.  prepare() makes
what a program has in hand before the call, run() is one pass through the
operator, exact() the same pass from its definition in 64 bits, work() the
bytes and operations that the pass cannot do without.  With `own` false run()
computes the operator in elementary torch operations in 32 bits (angles in
64), rounded once at the end; with `own` true it calls this library.

Kinds of case:
  qknorm  every head of query and key scaled to a mean square of one, times a
          weight per element, then rotated by the token's position (in place),
          with the key and the value stored into the paged cache or not
  append  keys and values stored into the paged 4-bit cache: a row x of a head
          as codes n of 0..15 and a (scale, low) pair, x ~ scale * n + low, with
          low = min x, scale = (max x - min x) / 15 in 32 bits, then in x's
          type, and n = (x - low) / scale to the nearest, ties to even
  attend  attention over such a cache through a block table: causal from the
          bottom right, grouped heads, ragged lengths
  gemv    out = x W^T with W in 4-bit codes, W = (n - zero) * scale by groups
          along a row, the zeros given or 8
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
BASE = 1000000.0
TABLE = 8192  # positions of a cos / sin table
EPS = 1e-6


def listed():
    return [
        # Four sequences decode: their queries, keys and values on the way from
        # the qkv product to the cache. The smallest call, all latency.
        dict(name="qk_decode_cache", kind="qknorm", tokens=4, heads=32, kv_heads=8, head=128,
             rot=128, neox=True, table=True, far=0, cache=True, block=16, dtype="f16"),
        # A prefill batch at far positions, angles computed.
        dict(name="qk_prefill_cache", kind="qknorm", tokens=8191, heads=32, kv_heads=8, head=128,
             rot=128, neox=True, table=False, far=200000, cache=True, block=16, dtype="bf16"),
        # Heads of 96 of which 32 elements turn, in adjacent pairs, in place: a
        # small model's prefill.
        dict(name="qk_partial", kind="qknorm", tokens=2049, heads=16, kv_heads=4, head=96, rot=32,
             neox=False, table=True, far=0, cache=False, block=0, dtype="bf16"),
        # A decode batch appends one row a sequence, four of them padding.
        dict(name="append_decode", kind="append", tokens=64, pad=4, kv_heads=8, head=128, block=16,
             dtype="bf16"),
        # A prefill batch appends whole prompts.
        dict(name="append_prefill", kind="append", tokens=8192, pad=0, kv_heads=8, head=128,
             block=32, dtype="f16"),
        # One sequence decodes over a short context.
        dict(name="attend_b1_short", kind="attend", batch=1, rows=1, low=777, high=777, heads=32,
             kv_heads=8, head=128, block=16, dtype="f16"),
        # A serving batch decodes over ragged contexts: the cache is the work.
        dict(name="attend_b64_ragged", kind="attend", batch=64, rows=1, low=512, high=8192, heads=32,
             kv_heads=8, head=128, block=16, dtype="bf16"),
        # Chunks of prompts over long contexts: few rows, many keys.
        dict(name="attend_chunk", kind="attend", batch=2, rows=203, low=9000, high=16300, heads=40,
             kv_heads=8, head=128, block=16, dtype="bf16"),
        # Second halves of prompts: the product of queries and keys is the work.
        dict(name="attend_prefill", kind="attend", batch=4, rows=2048, low=3500, high=4096, heads=32,
             kv_heads=8, head=128, block=16, dtype="bf16"),
        # The attention output product of one decoding sequence.
        dict(name="gemv_b1", kind="gemv", batch=1, n=4096, k=4096, group=128, zeros=False,
             dtype="f16"),
        # Gate and up of a decode batch, zeros of their own, small groups.
        dict(name="gemv_b16_gate_up", kind="gemv", batch=16, n=28672, k=4096, group=64, zeros=True,
             dtype="bf16"),
        # The down product of a larger batch: a long K.
        dict(name="gemv_b33_down", kind="gemv", batch=33, n=4096, k=14336, group=128, zeros=True,
             dtype="bf16"),
    ]


# ----------------------------------------------------------------- drawing

HEADS = [(32, 8), (32, 8), (16, 2), (16, 4), (16, 16), (40, 8), (64, 8), (8, 1)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    kind = rng.choice(["qknorm", "qknorm", "append", "attend", "attend", "attend", "gemv", "gemv"])
    dtype = rng.choice(["f16", "bf16"])
    heads, kv_heads = rng.choice(HEADS)
    block = rng.choice([16, 16, 32, 64, 24])
    if kind == "qknorm":
        head = rng.choice([64, 80, 96, 128, 128, 128, 192, 256])
        table, cache = rng.random() < 0.5, rng.random() < 0.6
        return dict(kind=kind, tokens=_log(rng, 1, 8191), heads=heads, kv_heads=kv_heads, head=head,
                    rot=rng.choice([head, head, head, 32]), neox=rng.random() < 0.75, table=table,
                    far=0 if table else rng.choice([0, 30000, 200000]), cache=cache,
                    block=block if cache else 0, dtype=dtype)
    if kind == "append":
        tokens = _log(rng, 1, 8192)
        return dict(kind=kind, tokens=tokens, pad=rng.choice([0, min(tokens - 1, 3)]),
                    kv_heads=kv_heads, head=rng.choice([64, 96, 128, 128, 192]), block=block,
                    dtype=dtype)
    if kind == "attend":
        rows = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 300), _log(rng, 300, 2048)])
        high = _log(rng, max(16, rows), 16384)
        return dict(kind=kind, batch=_log(rng, 1, 64), rows=rows,
                    low=rng.choice([high, max(1, high // 8)]), high=high, heads=heads,
                    kv_heads=kv_heads, head=rng.choice([64, 96, 128, 128, 128, 192]), block=block,
                    dtype=dtype)
    group = rng.choice([32, 64, 128, 128, 256])
    return dict(kind=kind, batch=rng.choice([1, 1, _log(rng, 1, 64)]), n=_log(rng, 64, 28672),
                k=group * max(1, _log(rng, 256, 16384) // group), group=group,
                zeros=rng.random() < 0.6, dtype=dtype)


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
        # keys padded to the longest context, and their scores, in 32 bits
        if c["kind"] == "attend" and (c["batch"] * c["high"] * c["kv_heads"] * c["head"] > 64 << 23 or
                                      c["batch"] * c["high"] * c["heads"] * c["rows"] > 1 << 30):
            continue
        if all(w[key] <= m[key] for key in m):
            return c


# ------------------------------------------------------------ sizes of a case

def _lengths(c):
    """(query rows, keys) of each sequence: the first with most of both, the
    others anywhere between the least and the most keys; now and then a
    sequence of a larger batch is padding without rows or keys."""
    r = random.Random(1000003 * c["batch"] + 1009 * c["high"] + c["rows"])
    got = []
    for b in range(c["batch"]):
        rows = c["rows"] if b == 0 or c["rows"] < 9 else r.randint(c["rows"] // 2, c["rows"])
        keys = c["high"] if b == 0 else r.randint(min(c["low"], c["high"]), c["high"])
        got.append((0, 0) if c["batch"] >= 16 and b % 16 == 15 else (min(rows, keys), keys))
    return got


def _visible(c):
    """Pairs of a query row and a key that it sees."""
    return sum(rows * (keys - rows) + rows * (rows + 1) // 2 for rows, keys in _lengths(c))


def work(c):
    """Bytes and operations of one pass that it cannot do without."""
    if c["kind"] == "qknorm":
        t, q, kv = c["tokens"], c["heads"] * c["head"], c["kv_heads"] * c["head"]
        by = 4 * t * q + (8 * t * kv + 8 * t if c["cache"] else 4 * t * kv) + 8 * t
        return {"bytes": by, "flops": t * (q + kv) * 7}
    if c["kind"] == "append":
        rows = 2 * (c["tokens"] - c["pad"]) * c["kv_heads"]
        return {"bytes": rows * (2 * c["head"] + c["head"] // 2 + 4) + 8 * c["tokens"],
                "flops": rows * c["head"] * 5}
    if c["kind"] == "attend":
        rows, keys = (sum(x) for x in zip(*_lengths(c)))
        by = 4 * rows * c["heads"] * c["head"] + 2 * keys * c["kv_heads"] * (c["head"] // 2 + 4)
        return {"bytes": by, "flops": 4 * c["heads"] * c["head"] * _visible(c)}
    n, k, b = c["n"], c["k"], c["batch"]
    by = n * k // 2 + 2 * n * (k // c["group"]) * (2 if c["zeros"] else 1) + 2 * b * (n + k)
    return {"bytes": by, "flops": 2 * b * n * k}


# ------------------------------------------------------------------- inputs

class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(self, *shape, scale=1.0, dtype=torch.float16):
        return torch.randn(shape, generator=self.g, device="cuda").mul_(scale).to(dtype)

    def uniform(self, *shape, lo=0.0, hi=1.0):
        return torch.rand(shape, generator=self.g, device="cuda").mul_(hi - lo).add_(lo)

    def codes(self, *shape):
        return torch.randint(0, 256, shape, generator=self.g, device="cuda", dtype=torch.uint8)

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")


def _packed(x):
    """Rows of x (its last dimension) as packed codes and (scale, low) pairs."""
    low, top = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((top.float() - low.float()) / 15).to(x.dtype)
    n = (x.float() - low.float()) / scale.float()
    n = torch.where(scale > 0, n, torch.zeros_like(n)).round().clamp(0, 15).to(torch.uint8)
    return n[..., 0::2] | (n[..., 1::2] << 4), torch.cat([scale, low], -1)


def _cache(c, r, pages, channels, dt):
    """A cache of rows drawn around `channels` (as models' keys have a few far
    ones), page by page to bound the 32-bit intermediates."""
    kv, block, d = c["kv_heads"], c["block"], c["head"]
    codes = torch.empty(pages, kv, block, d // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(pages, kv, block, 2, dtype=dt, device="cuda")
    step = max(1, (1 << 26) // (kv * block * d))
    for i in range(0, pages, step):
        n = min(step, pages - i)
        x = r.normal(n, kv, block, d, dtype=dt) + channels
        codes[i:i + n], scales[i:i + n] = _packed(x)
    return codes, scales


def prepare(c, seed):
    r, dt = _Rand(seed), DTYPES[c["dtype"]]
    s = {"case": c}
    if c["kind"] == "gemv":
        n, groups = c["n"], c["k"] // c["group"]
        s.update(w=r.codes(n, c["k"] // 2),
                 scales=(r.uniform(n, groups, lo=0.5, hi=1.5) * (0.2 * c["k"] ** -0.5)).to(dt),
                 zeros=r.uniform(n, groups, lo=5.5, hi=9.5).to(dt) if c["zeros"] else None,
                 x=r.normal(c["batch"], c["k"], dtype=dt),
                 out=torch.empty(c["batch"], n, dtype=dt, device="cuda"))
        return s
    kv, d, block = c["kv_heads"], c["head"], c["block"]
    if c["kind"] == "attend":
        lens = _lengths(c)
        used = [(keys + block - 1) // block for _, keys in lens]
        wide = max(used)
        table = torch.zeros(len(lens), wide, dtype=torch.int32)
        pages = sum(used) + 3
        free, at = r.perm(pages).int().cpu(), 0
        for b, n in enumerate(used):
            table[b, :n] = free[at:at + n]
            at += n
        channels = r.normal(kv, 1, d, scale=1.0, dtype=dt)
        kc, ks = _cache(c, r, pages, channels, dt)
        vc, vs = _cache(c, r, pages, torch.zeros_like(channels), dt)
        for b, (_, keys) in enumerate(lens):  # what lies behind the last key is anything
            if keys % block:
                ks[table[b, keys // block], :, keys % block:] = math.nan
                vs[table[b, keys // block], :, keys % block:] = math.nan
        rows = [x for x, _ in lens]
        s.update(q=r.normal(sum(rows), c["heads"], d, scale=1.2, dtype=dt), kc=kc, ks=ks, vc=vc,
                 vs=vs, table=table.cuda(), rows=rows, keys=[x for _, x in lens],
                 cu=torch.tensor([sum(rows[:b]) for b in range(len(rows) + 1)],
                                 dtype=torch.int32).cuda(),
                 used=torch.tensor([x for _, x in lens], dtype=torch.int32).cuda(),
                 out=torch.empty(sum(rows), c["heads"], d, dtype=dt, device="cuda"))
        return s
    t, h = c["tokens"], c.get("heads", 0)
    qkv = r.normal(t, (h + 2 * kv) * d, scale=2.0, dtype=dt)
    s.update(q=qkv[:, :h * d], k=qkv[:, h * d:(h + kv) * d], v=qkv[:, (h + kv) * d:])
    if block:
        pages = max(4, (t + t // 4 + block - 1) // block)
        s["slots"] = r.perm(pages * block)[:t].contiguous()
    if c["kind"] == "append":
        s["slots"][t - c["pad"]:] = -1
        for name in ("k", "v"):
            s[name] = s[name].view(t, kv, d)
            s[name + "c"] = torch.zeros(pages, kv, block, d // 2, dtype=torch.uint8, device="cuda")
            s[name + "s"] = torch.zeros(pages, kv, block, 2, dtype=dt, device="cuda")
        return s
    place = random.Random(seed)
    first = c["far"] + place.randrange(64)
    positions = torch.arange(first, first + t, dtype=torch.int64)
    s.update(positions=(positions % TABLE if c["table"] else positions).cuda(),
             qw=(1 + r.normal(d, scale=0.3, dtype=torch.float32)).to(dt),
             kw=(1 + r.normal(d, scale=0.3, dtype=torch.float32)).to(dt), angles=None)
    if c["table"]:  # float32 [positions, rot] cos then sin, as a model keeps it
        a = _turns(torch.arange(TABLE, device="cuda"), c["rot"])
        s["angles"] = torch.cat([a.cos(), a.sin()], 1).float()
    if c["cache"]:
        for name in ("kc", "vc"):
            s[name] = torch.zeros(pages, kv, block, d, dtype=dt, device="cuda")
    return s


def _turns(positions, rot):
    """Angles [tokens, rot / 2] in 64 bits."""
    i = torch.arange(0, rot, 2, dtype=torch.float64, device="cuda")
    return positions.double()[:, None] * BASE ** (-i / rot)


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
    if c["kind"] == "gemv":
        tecoops.gemv_int4(s["w"], s["scales"], s["x"], s["out"], zeros=s["zeros"])
        return s["out"]
    if c["kind"] == "attend":
        tecoops.flash_attn_varlen_int4(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], max(s["rows"]),
                                       s["cu"], max(s["keys"]), s["used"], None, True, s["table"],
                                       s["out"])
        return s["out"]
    if c["kind"] == "append":
        tecoops.reshape_and_cache_int4(s["k"], s["v"], s["slots"], s["kc"], s["vc"], s["ks"],
                                       s["vs"])
        return {name: s[name] for name in ("kc", "vc", "ks", "vs")}
    more = dict(eps=EPS, cos_sin_cache=s["angles"], is_neox=c["neox"], base=BASE, rot_dim=c["rot"])
    if c["cache"]:
        tecoops.qk_norm_rotary_reshape_and_cache(s["positions"], s["q"], s["k"], s["v"], s["qw"],
                                                 s["kw"], s["slots"], s["kc"], s["vc"], c["head"],
                                                 **more)
        return {"q": s["q"], "kc": s["kc"], "vc": s["vc"]}
    tecoops.qk_norm_rotary(s["positions"], s["q"], s["k"], s["qw"], s["kw"], c["head"], **more)
    return {"q": s["q"], "k": s["k"]}


def _unpacked(w):
    """Codes of packed bytes, the low half of a byte first."""
    return torch.stack([w & 15, w >> 4], -1).flatten(-2)


def _plain_gemv(s):
    c = s["case"]
    w = _unpacked(s["w"]).float().view(c["n"], -1, c["group"])
    w = (w - (8.0 if s["zeros"] is None else s["zeros"].float()[..., None])) * s["scales"].float()[..., None]
    return (s["x"].float() @ w.view(c["n"], -1).t()).to(s["x"].dtype)


def _held(codes, scales, pages, lengths):
    """The rows [sequences, kv heads, keys, head] that a cache holds for them, 0
    behind the last key."""
    b, wide = pages.shape
    kv, block = codes.shape[1:3]
    n = _unpacked(codes[pages].transpose(1, 2).reshape(b, kv, wide * block, -1))
    pair = scales[pages].transpose(1, 2).reshape(b, kv, wide * block, 2).float()
    there = torch.arange(wide * block, device="cuda") < lengths[:, None]
    pair = torch.where(there[:, None, :, None], pair, torch.zeros_like(pair))
    return n.float() * pair[..., :1] + pair[..., 1:]


def _plain_attend(s):
    c, d, kv = s["case"], s["case"]["head"], s["case"]["kv_heads"]
    most, group = max(s["rows"]), c["heads"] // kv
    rows, keys = s["cu"].diff().long(), s["used"].long()
    row = torch.arange(most, device="cuda")
    real = row < rows[:, None]
    at = torch.where(real, s["cu"][:-1, None].long() + row, torch.zeros_like(real, dtype=torch.int64))
    q = s["q"][at].float().view(c["batch"], most, kv, group, d).permute(0, 2, 3, 1, 4)
    q = q.reshape(c["batch"], kv, group * most, d)
    pages = s["table"].long()
    k = _held(s["kc"], s["ks"], pages, keys).transpose(2, 3).contiguous()
    p = (q @ k).mul_(d ** -0.5).view(c["batch"], kv, group, most, -1)
    del k
    seen = torch.arange(p.shape[-1], device="cuda") <= (keys - rows)[:, None, None] + row[:, None]
    seen &= real[..., None]
    p.masked_fill_(~seen[:, None, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    p.div_(p.sum(-1, keepdim=True).clamp(min=1e-30))
    out = p.view(c["batch"], kv, group * most, -1) @ _held(s["vc"], s["vs"], pages, keys)
    out = out.view(c["batch"], kv, group, most, d).permute(0, 3, 1, 2, 4)[real]
    return out.reshape(-1, c["heads"], d).to(s["q"].dtype)


def _plain_append(s):
    c = s["case"]
    stored = s["slots"] >= 0
    page, row = s["slots"][stored] // c["block"], s["slots"][stored] % c["block"]
    s["kc"][page, :, row], s["ks"][page, :, row] = _packed(s["k"][stored])
    s["vc"][page, :, row], s["vs"][page, :, row] = _packed(s["v"][stored])
    return {name: s[name] for name in ("kc", "vc", "ks", "vs")}


def _plain_turned(c, x, weight, cos, sin, heads):
    x = x.float().reshape(x.shape[0], heads, c["head"])
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    half, cos, sin = c["rot"] // 2, cos[:, None], sin[:, None]
    turn, rest = x[..., :c["rot"]], x[..., c["rot"]:]
    if c["neox"]:
        a, b = turn[..., :half], turn[..., half:]
        turn = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = turn[..., 0::2], turn[..., 1::2]
        turn = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turn, rest], -1)


def _plain_qknorm(s):
    c, half, dt = s["case"], s["case"]["rot"] // 2, s["q"].dtype
    if s["angles"] is not None:
        cos, sin = s["angles"][s["positions"], :half], s["angles"][s["positions"], half:]
    else:
        a = _turns(s["positions"], c["rot"])
        cos, sin = a.cos().float(), a.sin().float()
    q = _plain_turned(c, s["q"], s["qw"], cos, sin, c["heads"]).to(dt)
    k = _plain_turned(c, s["k"], s["kw"], cos, sin, c["kv_heads"]).to(dt)
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
    return {"gemv": _plain_gemv, "attend": _plain_attend, "append": _plain_append,
            "qknorm": _plain_qknorm}[s["case"]["kind"]](s)


# ------------------------------------------------------------- 64-bit results

def _halves(w):
    """Codes of packed bytes in 64 bits, by their definition: byte j holds
    elements 2j (low half) and 2j + 1."""
    n = torch.empty(*w.shape[:-1], 2 * w.shape[-1], dtype=torch.float64, device="cuda")
    high = torch.div(w, 16, rounding_mode="floor").double()
    n[..., 1::2] = high
    n[..., 0::2] = w.double() - 16 * high
    return n


def _exact_gemv(c, s):
    out = torch.empty(c["batch"], c["n"], dtype=torch.float64, device="cuda")
    x, g = s["x"].double(), c["group"]
    for lo in range(0, c["n"], 2048):
        n = _halves(s["w"][lo:lo + 2048])
        scale = s["scales"][lo:lo + 2048].double().repeat_interleave(g, 1)
        zero = s["zeros"][lo:lo + 2048].double().repeat_interleave(g, 1) if c["zeros"] else 8.0
        out[:, lo:lo + 2048] = x @ ((n - zero) * scale).t().contiguous()
    return out


def _exact_attend(c, s):
    d, block, group = c["head"], c["block"], c["heads"] // c["kv_heads"]
    out, first = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for b, (rows, keys) in enumerate(zip(s["rows"], s["keys"])):
        pages = s["table"][b, :(keys + block - 1) // block].long()
        for h in range(c["kv_heads"] if rows else 0):
            held = []
            for codes, pair in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
                n = _halves(codes[pages, h].reshape(-1, d // 2)[:keys])
                pr = pair[pages, h].reshape(-1, 2)[:keys].double()
                held.append(pr[:, :1] * n + pr[:, 1:])
            place = torch.arange(rows, device="cuda")[:, None] + (keys - rows)
            hidden = torch.arange(keys, device="cuda")[None] > place
            for g in range(h * group, (h + 1) * group):
                score = s["q"][first:first + rows, g].double() @ held[0].t() / math.sqrt(d)
                score[hidden] = -math.inf
                out[first:first + rows, g] = torch.softmax(score, -1) @ held[1]
        first += rows
    return out


def _exact_append(c, s):
    got = {}
    for name in ("k", "v"):
        codes, pairs = s[name + "c"].clone(), s[name + "s"].clone()
        keep = (s["slots"] >= 0).nonzero()[:, 0]
        x = s[name][keep].double()
        low = x.min(-1).values
        scale = ((x.max(-1).values - low) / 15).float().to(pairs.dtype)
        n = (x - low[..., None]) / scale.double()[..., None]
        n = torch.nan_to_num(n, nan=0.0, posinf=15.0).round().clamp(0, 15).long()
        page = torch.div(s["slots"][keep], c["block"], rounding_mode="floor")
        row = s["slots"][keep] - page * c["block"]
        codes[page, :, row] = (n[..., 0::2] + 16 * n[..., 1::2]).to(torch.uint8)
        pairs[page, :, row] = torch.stack([scale, low.to(pairs.dtype)], -1)
        got[name + "c"], got[name + "s"] = codes, pairs.double()
    return got


def _exact_qknorm(c, s):
    half, t = c["rot"] // 2, c["tokens"]
    if c["table"]:
        cos = s["angles"][s["positions"]][:, :half].double()
        sin = s["angles"][s["positions"]][:, half:].double()
    else:
        i = torch.arange(half, dtype=torch.float64, device="cuda")
        a = s["positions"].double()[:, None] / BASE ** (i / half)
        cos, sin = torch.cos(a), torch.sin(a)

    def turned(x, weight, heads):
        x = x.double().reshape(t, heads, c["head"])
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["head"] + EPS) * weight.double()
        y = x.clone()
        one = slice(0, half) if c["neox"] else slice(0, c["rot"], 2)
        two = slice(half, c["rot"]) if c["neox"] else slice(1, c["rot"], 2)
        y[..., one] = x[..., one] * cos[:, None] - x[..., two] * sin[:, None]
        y[..., two] = x[..., two] * cos[:, None] + x[..., one] * sin[:, None]
        return y

    q = turned(s["q"], s["qw"], c["heads"]).flatten(1)
    k = turned(s["k"], s["kw"], c["kv_heads"])
    if not c["cache"]:
        return {"q": q, "k": k.flatten(1)}
    kc, vc = s["kc"].double(), s["vc"].double()
    kc[s["slots"] // c["block"], :, s["slots"] % c["block"]] = k
    vc[s["slots"] // c["block"], :, s["slots"] % c["block"]] = s["v"].double().reshape(k.shape)
    return {"q": q, "kc": kc, "vc": vc}


def exact(c, seed):
    s = prepare(c, seed)
    return {"gemv": _exact_gemv, "attend": _exact_attend, "append": _exact_append,
            "qknorm": _exact_qknorm}[c["kind"]](c, s)
