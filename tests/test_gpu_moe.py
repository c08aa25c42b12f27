"""Mixture-of-experts layer (tecoops.moe_layer) against 64-bit references.

Whole numbers small enough for every intermediate to be exact, and routing
weights of exactly 1 / k, make the result the rounding of the exact value bit for
bit: a pair, a row or a part of K left out or taken twice shows.  Real inputs are
held to half a step of the result, the rounding of h (half a step of each h, of
independent signs, so within 4 times the root sum of squares of what they move:
7 standard deviations of a uniform error) and the fp32 sums."""
import ctypes
import math

import pytest
import torch

import tecoops
from tecoops import TecoopsError, _lib

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}
INF = math.inf


def route64(logits, top_k, renorm):
    """(ids, weights in 64 bits), in plain Python over the rows."""
    rows = logits.double().cpu().tolist()
    ids, weights = [], []
    for row in rows:
        live = [e for e, v in enumerate(row) if v > -INF]
        best = sorted(live, key=lambda e: (-row[e], e))[:top_k]
        top = row[best[0]] if best else 0.0
        ex = {e: 1.0 if row[e] == top else math.exp(row[e] - top) for e in live}
        total = sum(ex[e] for e in (best if renorm else live)) or 1.0
        ids.append(best + [-1] * (top_k - len(best)))
        weights.append([ex[e] / total for e in best] + [0.0] * (top_k - len(best)))
    return torch.tensor(ids, dtype=torch.int32), torch.tensor(weights, dtype=torch.float64)


def act64(y, name):
    if name == "relu":
        return y.clamp(min=0)
    if name == "silu":
        return y * torch.sigmoid(y)
    if name == "gelu":
        return y * 0.5 * torch.erfc(-y / math.sqrt(2))
    if name == "gelu_tanh":
        return y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
    return y


def layer64(x, w_in, w_out, ids, weights, act):
    """(out, root sum of squares of the terms w W h) in 64 bits, h not rounded."""
    out = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    spread = torch.zeros_like(out)
    inter = w_out.shape[2]
    for e in sorted(set(ids.flatten().tolist()) - {-1}):
        t, j = (ids == e).nonzero(as_tuple=True)
        w = weights[t, j].cuda()[:, None]
        y = x[t.cuda()].double() @ w_in[e].double().t().contiguous()
        h = act64(y[:, :inter], act) * y[:, inter:]
        w2 = w_out[e].double().t().contiguous()
        out.index_add_(0, t.cuda(), w * (h @ w2))
        spread.index_add_(0, t.cuda(), (w * w) * ((h * h) @ (w2 * w2)))
    return out, spread.sqrt()


def whole(g, *shape, dtype, most=1):
    return torch.randint(-most, most + 1, shape, generator=g, device="cuda").to(dtype)


def sparse_rows(g, *shape, dtype):
    """Entries of -1, 0, 1, at most 3 of a row not 0."""
    t = torch.zeros(shape, device="cuda")
    at = torch.randint(0, shape[-1], (*shape[:-1], 3), generator=g, device="cuda")
    t.scatter_(-1, at, whole(g, *shape[:-1], 3, dtype=torch.float32))
    return t.to(dtype)


def even_logits(g, tokens, experts, top_k, pad=0):
    """Exactly top_k logits of 0 in a row (weights of 1 / top_k), -inf the rest."""
    order = torch.rand(tokens, experts, generator=g, device="cuda").argsort(-1)[:, :top_k]
    logits = torch.full((tokens, experts), -INF, device="cuda")
    logits.scatter_(1, order, 0.0)
    if pad:
        logits[tokens - pad:] = -INF
    return logits


def run(x, w_in, w_out, logits, top_k, renorm=True, act="silu"):
    T = x.shape[0]
    out = torch.full(x.shape, float("nan"), dtype=x.dtype, device="cuda")
    ids = torch.full((T, top_k), 99, dtype=torch.int32, device="cuda")
    weights = torch.full((T, top_k), 9.0, device="cuda")
    tecoops.moe_layer(x, w_in, w_out, logits, top_k, out, renormalize=renorm, activation=act,
                      topk_ids=ids, topk_weights=weights)
    return out, ids, weights


# tokens, hidden, inter, experts, top_k, pad: one token, every size of item, more
# tokens than a slice, odd widths, one expert, a last block of rows cut short
SHAPES = [(1, 64, 32, 4, 2, 0), (1, 8, 8, 1, 1, 0), (1, 512, 1000, 8, 8, 0), (3, 136, 72, 128, 8, 1),
          (4, 1024, 264, 8, 2, 0), (5, 72, 40, 6, 4, 2), (8, 264, 136, 16, 4, 0),
          (9, 128, 128, 3, 1, 0), (16, 2048, 80, 60, 4, 3), (17, 200, 520, 4, 2, 0),
          (40, 128, 64, 64, 8, 5), (64, 520, 264, 8, 2, 0), (100, 256, 128, 4, 4, 0),
          (300, 64, 96, 16, 8, 7), (512, 32, 16, 2, 1, 0), (513, 48, 24, 8, 2, 0),
          (1100, 16, 40, 5, 1, 30), (2, 70, 33, 5, 2, 0), (30, 9, 7, 3, 2, 1), (600, 24, 17, 4, 1, 0),
          (64, 8, 8, 1, 1, 0), (1, 4096, 16, 4, 1, 0), (20, 16, 4096, 160, 8, 0),
          (4, 64, 32, 200, 8, 1), (8, 256, 2048, 1000, 8, 0), (2, 2048, 264, 160, 4, 0),
          (6, 32, 3000, 64, 8, 1), (8, 40, 64, 40, 32, 0), (7, 4104, 136, 9, 4, 0)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("T,H,I,E,k,pad", SHAPES)
def test_exact(T, H, I, E, k, pad, dtype):
    dt = DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(T * 3 + H + I)
    x = whole(g, T, H, dtype=dt, most=2)
    w_in, w_out = sparse_rows(g, E, 2 * I, H, dtype=dt), whole(g, E, H, I, dtype=dt)
    logits = even_logits(g, T, E, k, pad)
    ref_ids, ref_weights = route64(logits, k, True)
    for lg in (logits, logits.to(dt)):
        out, ids, weights = run(x, w_in, w_out, lg, k, act="relu")
        assert torch.equal(ids.cpu(), ref_ids)
        assert torch.equal(weights.cpu().double(), ref_weights)
        ref, _ = layer64(x, w_in, w_out, ref_ids, ref_weights, "relu")
        assert torch.equal(out, ref.to(dt))
        assert not pad or (out[T - pad:] == 0).all()


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh", None])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("T,H,I,E,k", [(1, 512, 384, 8, 2), (7, 256, 200, 16, 4), (50, 192, 264, 32, 3),
                                       (130, 96, 72, 4, 2), (3, 45, 35, 4, 2)])
def test_real(T, H, I, E, k, dtype, act):
    dt = DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(T + H)

    def real(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dt)

    x, w_in, w_out = real(T, H), real(E, 2 * I, H, scale=H ** -0.5), real(E, H, I, scale=I ** -0.5)
    for renorm in (True, False):
        for logits in (torch.randn(T, E, generator=g, device="cuda") * 2, real(T, E)):
            out, ids, weights = run(x, w_in, w_out, logits, k, renorm, act)
            ref_ids, ref_weights = route64(logits, k, renorm)
            assert torch.equal(ids.cpu(), ref_ids)
            # exp and the quotient: 4 units; the sum of E terms: E / 64 + 6 additions
            assert ((weights.cpu().double() - ref_weights).abs() <=
                    (10 + E / 64) * 2.0 ** -24 * ref_weights + 1e-30).all()
            ref, spread = layer64(x, w_in, w_out, ref_ids, ref_weights, act)
            half = torch.finfo(dt).eps / 2
            sums = ((H + I) / 8 + 60) * 2.0 ** -24
            bound = half * ref.abs() * 1.01 + (4.1 * half + 6 * sums) * spread + 20 * 2.0 ** -24 * ref.abs()
            bound += torch.finfo(dt).smallest_normal * half * 2
            err = (out.double() - ref).abs()
            assert (err <= bound).all(), (err / bound).max().item()


@pytest.mark.parametrize("E,k", [(1, 1), (7, 7), (63, 5), (64, 8), (65, 8), (128, 8), (160, 6), (1000, 32),
                                 (1024, 32), (33, 32)])
def test_routing(E, k):
    """Ties to the lowest index (and -0 ties with 0), -inf and NaN never chosen,
    +inf alone in its softmax, rows with fewer than k and with none."""
    T, H, I, dt = 40, 8, 8, torch.float16
    g = torch.Generator(device="cuda").manual_seed(E)
    x, w_in = torch.zeros(T, H, dtype=dt, device="cuda"), torch.zeros(E, 2 * I, H, dtype=dt, device="cuda")
    w_out = torch.zeros(E, H, I, dtype=dt, device="cuda")
    logits = torch.randn(T, E, generator=g, device="cuda") * 3
    logits[1] = 0
    logits[2] = torch.where(torch.arange(E, device="cuda") % 2 == 0, -0.0, 0.0)
    logits[3] = -INF
    logits[4, 1:] = -INF
    logits[5, :E - 1] = -INF
    logits[6] = float("nan")
    logits[7, ::2] = float("nan")
    logits[8, E // 2] = INF
    logits[9] = torch.randint(0, 3, (E,), generator=g, device="cuda").float()
    logits[10] = -3e38
    logits[11, E // 3] = 3e38
    logits[12] = -INF
    logits[12, E // 2:] = 5
    logits[13] *= 1e-30
    logits[14] += 1e4
    logits[15] = torch.randint(0, 2, (E,), generator=g, device="cuda").float() * -1e30
    for lg in (logits, logits.to(dt), ):
        for renorm in (True, False):
            clean = torch.where(torch.isnan(lg), torch.full_like(lg, -INF), lg)
            # 3e38 is +inf in fp16; more than one +inf has no softmax
            _, ids, weights = run(x, w_in, w_out, lg, k, renorm)
            ref_ids, ref = route64(clean, k, renorm)
            assert torch.equal(ids.cpu(), ref_ids)
            err = (weights.cpu().double() - ref).abs()
            # an argument d of exp is rounded by 2^-24 |d|, |d| at most 103 where exp is not 0
            assert (err <= (120 + E / 64) * 2.0 ** -24 * ref + 1e-37).all()
            assert ((weights.cpu() == 0) | (ids.cpu() >= 0)).all()


def test_one_expert_takes_all():
    """Every token to one expert: more items of it than any even spread makes."""
    dt = torch.bfloat16
    for T, E in ((200, 128), (512, 64), (64, 1000), (700, 16)):
        g = torch.Generator(device="cuda").manual_seed(T)
        H, I = 64, 48
        x = whole(g, T, H, dtype=dt, most=2)
        w_in, w_out = sparse_rows(g, E, 2 * I, H, dtype=dt), whole(g, E, H, I, dtype=dt)
        logits = torch.full((T, E), -INF, device="cuda")
        logits[:, E - 2] = 1.0
        ids, w = route64(logits, 1, True)
        out, got, _ = run(x, w_in, w_out, logits, 1, act="relu")
        assert torch.equal(got.cpu(), ids)
        assert torch.equal(out, layer64(x, w_in, w_out, ids, w, "relu")[0].to(dt))


@pytest.mark.parametrize("H", [64, 60])
def test_strides_and_poison(H):
    """Rows of x a distance apart with NaN between; NaN in the weights of experts
    that no token chose, in a padded token's row, and in one token's row."""
    T, I, E, k, dt = 12, 40, 16, 2, torch.float16
    g = torch.Generator(device="cuda").manual_seed(1)
    wide = torch.full((T, H + 8), float("nan"), dtype=dt, device="cuda")
    wide[:, :H] = whole(g, T, H, dtype=dt, most=2)
    x = wide[:, :H]
    w_in, w_out = sparse_rows(g, E, 2 * I, H, dtype=dt), whole(g, E, H, I, dtype=dt)
    logits = even_logits(g, T, E - 3, k, pad=2)
    logits = torch.cat([logits, torch.full((T, 3), -INF, device="cuda")], 1)
    ids, w = route64(logits, k, True)
    ref = layer64(x, w_in, w_out, ids, w, "relu")[0].to(dt)
    w_in[E - 3:], w_out[E - 3:] = float("nan"), float("inf")
    wide[T - 1] = float("nan")
    out = run(x, w_in, w_out, logits, k, act="relu")[0]
    assert torch.equal(out, ref)
    wide[4, 3] = float("nan")
    out = run(x, w_in, w_out, logits, k, act="relu")[0]
    rows = torch.arange(T, device="cuda") != 4
    assert torch.equal(out[rows], ref[rows]) and torch.isnan(out[4]).any()


@pytest.mark.parametrize("T,H,I", [(6, 128, 64), (70, 64, 96), (520, 32, 32), (5, 33, 31)])
def test_workspace(T, H, I):
    """A workspace of just the size, full of ones, nothing written past it; one
    too small or misaligned refused; none: the handle's scratch, refused while
    its stream is captured."""
    E, k, dt = 8, 2, torch.float16
    g = torch.Generator(device="cuda").manual_seed(T)
    x = whole(g, T, H, dtype=dt, most=2)
    w_in, w_out = sparse_rows(g, E, 2 * I, H, dtype=dt), whole(g, E, H, I, dtype=dt)
    logits = even_logits(g, T, E, k)
    ids, w = route64(logits, k, True)
    ref = layer64(x, w_in, w_out, ids, w, "relu")[0].to(dt)
    need = ctypes.c_size_t()
    _lib.call("tecoopsGetMoeLayerWorkspaceSize", T, H, I, E, k, ctypes.byref(need))
    L, h = _lib.lib(), tecoops._handle(x.device)
    ws = torch.full((need.value + 256,), 0xFF, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(x)

    def call(ptr, size):
        return L.tecoopsMoeLayer(h, x.data_ptr(), H, w_in.data_ptr(), w_out.data_ptr(),
                                 logits.data_ptr(), _lib.DATA_FLOAT, out.data_ptr(), None, None, T, H, I,
                                 E, k, 1, 1, ptr, size, _lib.DATA_HALF)

    assert call(ws.data_ptr(), need.value) == 0
    assert torch.equal(out, ref) and (ws[need.value:] == 0xFF).all()
    assert call(ws.data_ptr(), need.value - 1) == _lib.BAD_PARAM
    assert call(ws.data_ptr() + 8, need.value) == _lib.BAD_PARAM
    out.zero_()
    assert call(None, 0) == 0
    assert torch.equal(out, ref)
    torch.cuda.synchronize()
    status = []
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h = tecoops._handle(x.device)
        status.append(call(None, 0))
        out.zero_()
    assert status == [_lib.NOT_SUPPORTED]
    h = tecoops._handle(x.device)


def test_streams_and_graphs():
    """On a side stream; two captured graphs replayed in turn with eager calls
    between and new routings, each replay equal to the eager call."""
    dt = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(3)
    cases = []
    for T, H, I, E, k in ((4, 256, 128, 32, 4), (90, 128, 64, 8, 2)):
        cases.append(dict(x=torch.randn(T, H, generator=g, device="cuda").to(dt),
                          w_in=(torch.randn(E, 2 * I, H, generator=g, device="cuda") * H ** -0.5).to(dt),
                          w_out=(torch.randn(E, H, I, generator=g, device="cuda") * I ** -0.5).to(dt),
                          logits=torch.randn(T, E, generator=g, device="cuda"), k=k))

    def step(outs):
        for c, o in zip(cases, outs):
            tecoops.moe_layer(c["x"], c["w_in"], c["w_out"], c["logits"], c["k"], o)

    def eager():
        outs = [torch.empty_like(c["x"]) for c in cases]
        step(outs)
        torch.cuda.synchronize()
        return outs

    first = eager()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [torch.empty_like(c["x"]) for c in cases]
        step(outs)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, outs))
    graphs = []
    for _ in range(2):
        outs, graph = [torch.empty_like(c["x"]) for c in cases], torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(outs)
        graphs.append((graph, outs))
    for turn in range(5):
        for c in cases:
            c["x"].copy_(torch.randn(c["x"].shape, generator=g, device="cuda"))
            c["logits"].copy_(torch.randn(c["logits"].shape, generator=g, device="cuda") * (1 + turn))
            if turn == 2:
                c["logits"][:, 1:] = -INF  # one expert
            if turn == 3:
                c["logits"].fill_(-INF)    # none
        ref = eager()
        for graph, outs in graphs:
            for o in outs:
                o.fill_(7)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(ref, outs)), turn
        assert all(torch.equal(a, b) for a, b in zip(ref, eager()))
    assert all((o != 0).any() for o in ref)


def test_torch_op():
    dt = torch.float16
    g = torch.Generator(device="cuda").manual_seed(2)
    T, H, I, E, k = 10, 64, 32, 8, 2
    x = whole(g, T, H, dtype=dt, most=2)
    w_in, w_out = sparse_rows(g, E, 2 * I, H, dtype=dt), whole(g, E, H, I, dtype=dt)
    logits = even_logits(g, T, E, k)
    out, ids, weights = run(x, w_in, w_out, logits, k, act="relu")
    o2, i2, w2 = torch.empty_like(out), torch.empty_like(ids), torch.empty_like(weights)
    torch.ops.tecoops.moe_layer(x, w_in, w_out, logits, k, o2, True, "relu", i2, w2)
    assert torch.equal(out, o2) and torch.equal(ids, i2) and torch.equal(weights, w2)
    torch.ops.tecoops.moe_layer(x, w_in, w_out, logits, k, o2.zero_(), True, "relu", None, None)
    assert torch.equal(out, o2)


@pytest.mark.parametrize("T,H,I", [(3, 64, 32), (40, 64, 32), (3, 33, 31)])
def test_without_the_torch_library(T, H, I, monkeypatch):
    dt, E, k = torch.bfloat16, 8, 2
    g = torch.Generator(device="cuda").manual_seed(T)
    x = whole(g, T, H, dtype=dt, most=2)
    w_in, w_out = sparse_rows(g, E, 2 * I, H, dtype=dt), whole(g, E, H, I, dtype=dt)
    logits = torch.randn(T, E, generator=g, device="cuda")
    first = run(x, w_in, w_out, logits, k)
    second = run(x, torch.nn.Parameter(w_in), w_out, logits, k)
    monkeypatch.setattr(tecoops, "_moe_layer", None)
    for a, b, c in zip(first, second, run(x, w_in, w_out, logits, k)):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("T", [2, 20])
def test_past_32_bits(T):
    """Experts whose weights lie past 2^32 bytes."""
    dt, E, H, I = torch.bfloat16, 48, 4096, 12288
    w_in = torch.zeros(E, 2 * I, H, dtype=dt, device="cuda")
    w_out = torch.zeros(E, H, I, dtype=dt, device="cuda")
    w_in[E - 1, I - 1, 0], w_in[E - 1, 2 * I - 1, 1] = 1, 1  # the last gate and up rows
    w_out[E - 1, H - 1, I - 1], w_out[E - 1, 0, I - 1] = 1, 2
    x = torch.zeros(T, H, dtype=dt, device="cuda")
    x[:, 0], x[:, 1] = 2, 3
    logits = torch.zeros(T, E, device="cuda")
    logits[:, E - 1] = 1
    out, ids, _ = run(x, w_in, w_out, logits, 1, act="relu")
    assert (ids == E - 1).all()
    assert (out[:, H - 1] == 6).all() and (out[:, 0] == 12).all() and out.count_nonzero() == 2 * T


def test_no_tokens_and_refusals():
    dt, T, H, I, E = torch.float16, 4, 16, 8, 4
    x, out = (torch.zeros(T, H, dtype=dt, device="cuda") for _ in range(2))
    w_in = torch.zeros(E, 2 * I, H, dtype=dt, device="cuda")
    w_out, logits = torch.zeros(E, H, I, dtype=dt, device="cuda"), torch.zeros(T, E, device="cuda")
    tecoops.moe_layer(x[:0], w_in, w_out, logits[:0], 2, out[:0])
    for a in [(x[:3], w_in, w_out, logits, 2, out), (x, w_in[:3], w_out, logits, 2, out),
              (x, w_in[:, :8], w_out, logits, 2, out), (x, w_in, w_out, logits[:, :3], 2, out),
              (x, w_in, w_out, logits, 2, out[:, :8]), (x, w_in, w_out, logits.cpu(), 2, out),
              (x, w_in, w_out.transpose(1, 2).contiguous().transpose(1, 2), logits, 2, out),
              (x, w_in[0], w_out, logits, 2, out)]:
        with pytest.raises(ValueError):
            tecoops.moe_layer(*a)
    ids, weights = torch.zeros(T, 2, dtype=torch.int32, device="cuda"), torch.zeros(T, 2, device="cuda")
    for kw in (dict(topk_ids=ids[:3]), dict(topk_weights=weights[:, :1].contiguous()),
               dict(activation="swish")):
        with pytest.raises(ValueError):
            tecoops.moe_layer(x, w_in, w_out, logits, 2, out, **kw)
    for kw in (dict(topk_ids=ids.long()), dict(topk_weights=weights.double())):
        with pytest.raises(TypeError):
            tecoops.moe_layer(x, w_in, w_out, logits, 2, out, **kw)
    for a in [(x.float(), w_in, w_out, logits, 2, out), (x, w_in.bfloat16(), w_out, logits, 2, out),
              (x, w_in, w_out, logits.bfloat16(), 2, out), (x, w_in, w_out, logits, 2, out.float())]:
        with pytest.raises(TypeError):
            tecoops.moe_layer(*a)
    for k in (0, -1, E + 1):
        with pytest.raises(TecoopsError):
            tecoops.moe_layer(x, w_in, w_out, logits, k, out)
