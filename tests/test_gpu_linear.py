"""Matrix products with their epilogue (tecoops.linear) against 64-bit products.

Inputs of small whole numbers keep every sum exact in fp32, so that the result
is the rounding of the exact value: any product left out, doubled or taken from
another row shows.  Activations and real inputs are held to a bound of the
rounding of the result (half a step, eps / 2 of the type) and of the fp32 sums:
K / 8 + 16 additions, each within 2^-24 of a partial sum, whose terms have
independent signs and stay below 6 times their root sum of squares."""
import ctypes
import math

import pytest
import torch

import tecoops
from tecoops import _lib

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def whole(g, *shape, dtype, most=2):
    return torch.randint(-most, most + 1, shape, generator=g, device="cuda").to(dtype)


def real(g, *shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def act64(y, name):
    if name == "relu":
        return torch.where(y < 0, torch.zeros_like(y), y)
    if name == "silu":
        return y * torch.sigmoid(y)
    if name == "gelu":
        return y * 0.5 * torch.erfc(-y / math.sqrt(2))
    if name == "gelu_tanh":
        return y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
    return y


def product64(x, w):
    return x.double() @ w.double().t().contiguous()


def linear64(x, w, bias, residual, act, gated):
    y = product64(x, w)
    if bias is not None:
        y = y + bias.double()
    n = w.shape[0] // 2
    y = act64(y[:, :n], act) * y[:, n:] if gated else act64(y, act)
    return y if residual is None else y + residual.double()


def check_real(got, x, w, bias, residual, act, gated):
    """The bound of the module's docstring.  A step d of a sum moves an
    activation by 1.13 d at most; a gated output by 1.13 d |up| + |act| d."""
    ref = linear64(x, w, bias, residual, act, gated)
    n, k = got.shape[1], x.shape[1]
    spread = product64(x.double() ** 2, w.double() ** 2).sqrt()
    d = (k / 8 + 16) * 2.0 ** -24 * 6 * spread + 2.0 ** -23 * product64(x, w).abs()
    if bias is not None:
        d += 2.0 ** -23 * bias.double().abs()
    if gated:
        y = product64(x, w) + (0 if bias is None else bias.double())
        a, u = act64(y[:, :n], act), y[:, n:]
        d = 1.13 * d[:, :n] * u.abs() + (a.abs() + d[:, :n]) * d[:, n:] + 2.0 ** -21 * (a * u).abs()
    else:
        d = 1.13 * d + 2.0 ** -21 * act64(product64(x, w) + (0 if bias is None else bias.double()),
                                          act).abs()
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * half
    bound = half * (ref.abs() + d) + d + tiny + 2.0 ** -23 * ref.abs()
    err = (got.double() - ref).abs()
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), (err / bound).max().item()


# rows: below and above the streaming kernel's 64, tiles of 128 and 256 cut
# short; K: less than a stage, stages cut short, whole; N: odd, a tile and one
SHAPES = [(1, 1, 1), (1, 4096, 8), (3, 17, 40), (5, 130, 264), (16, 48, 1024), (33, 31, 72),
          (64, 256, 512), (65, 129, 8), (65, 128, 64), (66, 7, 72), (100, 300, 200),
          (129, 257, 136), (130, 64, 2048), (257, 100, 4096), (300, 1000, 1000),
          (2, 9, 7), (70, 33, 9), (131, 130, 63), (200, 50, 588), (90, 260, 65), (513, 385, 1027),
          (4000, 5000, 72), (2100, 8200, 200)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_exact(m, n, k, dtype):
    """Bit for bit the rounding of the exact value, plain and gated, with and
    without bias, residual and relu."""
    dt = DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(m * 7 + n * 3 + k)
    x = whole(g, m, k, dtype=dt)
    for gated in (False, True):
        rows = 2 * n if gated else n
        # gated products of two sums stay below 2^24 with entries of -1 .. 1
        w = whole(g, rows, k, dtype=dt, most=1)
        bias, res = whole(g, rows, dtype=dt), whole(g, m, n, dtype=dt)
        if gated:
            x = x.clamp(-1, 1)
            assert k * k < 2 ** 24 or k == 4096  # |sum| <= 4 sqrt(k) of its random signs
        for b, r, act in ((None, None, None), (bias, res, "relu"), (bias, None, None)):
            out = torch.full((m, n), float("nan"), dtype=dt, device="cuda")
            tecoops.linear(x, w, out, bias=b, residual=r, activation=act, gated=gated)
            assert torch.equal(out, linear64(x, w, b, r, act, gated).to(dt)), (gated, act)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh", None])
def test_activations(act, gated, dtype):
    dt = DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(11)
    for m, n, k in ((7, 65, 96), (150, 190, 333), (260, 129, 640)):
        rows = 2 * n if gated else n
        x, w = real(g, m, k, dtype=dt), real(g, rows, k, dtype=dt, scale=2 * k ** -0.5)
        bias, res = real(g, rows, dtype=dt), real(g, m, n, dtype=dt)
        for b, r in ((bias, res), (None, None)):
            out = torch.empty(m, n, dtype=dt, device="cuda")
            tecoops.linear(x, w, out, bias=b, residual=r, activation=act, gated=gated)
            check_real(out, x, w, b, r, act, gated)


@pytest.mark.parametrize("m,k", [(2, 64), (80, 72), (80, 70), (300, 4096)])
def test_activation_tails(m, k):
    """Sums far out on both sides: an activation goes to 0 or the sum, never to
    NaN, and gelu keeps its relative accuracy on the negative side."""
    n = 64
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = 1
    w = torch.zeros(n, k, dtype=torch.bfloat16, device="cuda")
    w[:, 0] = torch.linspace(-200, 200, n)
    for act in ("relu", "silu", "gelu", "gelu_tanh"):
        out = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
        tecoops.linear(x, w, out, activation=act)
        ref = act64(w[:, 0].double(), act).expand(m, n)
        assert (out.double() - ref).abs().le(2.0 ** -8 * ref.abs() * 1.01 + 1e-30).all(), act
    w[:, 0] = torch.linspace(-9, 0, n)
    out = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    tecoops.linear(x, w, out, activation="gelu")
    ref = act64(w[:, 0].double(), "gelu").expand(m, n)
    # erfc of the device is within 16 units in fp32's last place; its argument's
    # rounding, 2^-24 v^2 relative, 2^-17.6 at v = -9
    assert (out.double() - ref).abs().le((2.0 ** -8 + 2.0 ** -17) * ref.abs() + 1e-30).all()


@pytest.mark.parametrize("m", [1, 64, 65, 200])
@pytest.mark.parametrize("k", [64, 136, 75])
def test_strides_and_poison(m, k):
    """Rows of x, residual and out a distance apart: what lies between is not
    read into a result (NaN there) and not written; a row of NaN or infinity in
    x or W stays in its row or column."""
    n, pad, dt = 100, 24, torch.float16
    g = torch.Generator(device="cuda").manual_seed(m + k)
    wide = torch.full((m, k + pad), float("nan"), dtype=dt, device="cuda")
    wide[:, :k] = whole(g, m, k, dtype=dt)
    x = wide[:, :k]
    res_wide = torch.full((m, n + 3), float("nan"), dtype=dt, device="cuda")
    res_wide[:, :n] = whole(g, m, n, dtype=dt)
    out_wide = torch.full((m, n + 5), 7.0, dtype=dt, device="cuda")
    w = whole(g, n, k, dtype=dt)
    out, res = out_wide[:, :n], res_wide[:, :n]
    tecoops.linear(x, w, out, residual=res)
    ref = linear64(x, w, None, res, None, False).to(dt)
    assert torch.equal(out, ref)
    assert (out_wide[:, n:] == 7.0).all()
    # the last row of W is followed by nothing of W; the others by their next
    w[5] = float("inf")
    w[n - 1] = float("nan")
    tecoops.linear(x, w, out, residual=res)
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[5] = keep[n - 1] = False
    assert torch.equal(out[:, keep], ref[:, keep])
    assert torch.isnan(out[:, n - 1]).all()
    if m > 1:
        w = whole(g, n, k, dtype=dt)
        ref = linear64(x, w, None, res, None, False).to(dt)
        wide[m // 2, :k] = float("nan")
        tecoops.linear(x, w, out, residual=res)
        rows = torch.arange(m, device="cuda") != m // 2
        assert torch.equal(out[rows], ref[rows]) and torch.isnan(out[m // 2]).all()


@pytest.mark.parametrize("m,n,k", [(4, 128, 256), (70, 130, 1024), (130, 200, 4096), (90, 64, 333),
                                   (4200, 4100, 64)])
def test_residual_in_place(m, n, k):
    dt = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(5)
    x, w, out = whole(g, m, k, dtype=dt), whole(g, n, k, dtype=dt), whole(g, m, n, dtype=dt)
    ref = linear64(x, w, None, out, None, False).to(dt)
    tecoops.linear(x, w, out, residual=out)
    assert torch.equal(out, ref)


@pytest.mark.parametrize("gated", [0, 1])
@pytest.mark.parametrize("k", [4096, 4099])
def test_workspace_sizes(k, gated):
    """Split along K with a workspace, with one too small for every split, one
    of odd alignment and none: whole numbers give the same bits each way, and
    nothing is written past what was given."""
    m, n, dt = 100, 70, torch.float16
    g = torch.Generator(device="cuda").manual_seed(k)
    x, w = whole(g, m, k, dtype=dt, most=1), whole(g, n * (1 + gated), k, dtype=dt, most=1)
    w[:, 200:] = 0  # gated products stay exact
    ref = linear64(x, w, None, None, None, bool(gated)).to(dt)
    need = ctypes.c_size_t()
    _lib.call("tecoopsGetLinearWorkspaceSize", m, n, k, gated, ctypes.byref(need))
    assert need.value > 0
    L = _lib.lib()
    h = tecoops._handle(x.device)
    for size, at in ((need.value, 0), (need.value // 2, 0), (need.value // 3 + 1, 0), (100, 0),
                     (need.value, 2), (0, 0)):
        ws = torch.full((need.value + 64,), 0x5A, dtype=torch.uint8, device="cuda")
        out = torch.empty(m, n, dtype=dt, device="cuda")
        st = L.tecoopsLinear(h, x.data_ptr(), k, w.data_ptr(), None, None, 0, out.data_ptr(), n, m,
                             n, k, 0, gated, ws.data_ptr() + at if size else None, size,
                             _lib.DATA_HALF)
        assert st == 0
        assert torch.equal(out, ref), (size, at)
        assert (ws[at + size:] == 0x5A).all()


def test_streams_and_graph():
    """On a side stream, and captured twice (streamed, tiled and split products)
    and replayed in turn with eager calls between: always the eager bits."""
    dt = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(3)
    shapes = [(4, 256, 512, False), (100, 96, 4096, True), (300, 500, 333, False)]
    data = [(real(g, m, k, dtype=dt), real(g, n * (2 if t else 1), k, dtype=dt, scale=k ** -0.5),
             real(g, m, n, dtype=dt), t) for m, n, k, t in shapes]

    def step(outs):
        for (x, w, r, t), out in zip(data, outs):
            tecoops.linear(x, w, out, residual=r, activation="silu", gated=t)

    def outs():
        return [torch.empty_like(r) for _, _, r, _ in data]

    def eager():
        o = outs()
        step(o)
        torch.cuda.synchronize()
        return o

    first = eager()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = outs()
        step(o)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, o))
    graphs = []
    for _ in range(2):
        o, graph = outs(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(o)
        graphs.append((graph, o))
    for turn in range(4):
        for x, _, _, _ in data:
            x.copy_(real(g, *x.shape, dtype=dt))
        ref = eager()
        for graph, o in graphs:
            for t in o:
                t.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(ref, o)), turn
        assert all(torch.equal(a, b) for a, b in zip(ref, eager()))


def test_torch_op():
    dt = torch.float16
    g = torch.Generator(device="cuda").manual_seed(9)
    x, w = whole(g, 20, 64, dtype=dt), whole(g, 30, 64, dtype=dt)
    b, r = whole(g, 30, dtype=dt), whole(g, 20, 30, dtype=dt)
    out = torch.empty(20, 30, dtype=dt, device="cuda")
    torch.ops.tecoops.linear(x, w, out, b, r, "relu", False)
    assert torch.equal(out, linear64(x, w, b, r, "relu", False).to(dt))
    out15 = torch.empty(20, 15, dtype=dt, device="cuda")
    torch.ops.tecoops.linear(x, w.clamp(-1, 1), out15, None, None, "none", True)
    assert torch.equal(out15, linear64(x, w.clamp(-1, 1), None, None, None, True).to(dt))


@pytest.mark.parametrize("m,n,k", [(5, 40, 128), (100, 70, 512), (90, 33, 77)])
def test_without_the_torch_library(m, n, k, monkeypatch):
    """The Python function through the C ABI alone gives the same bits; so do
    parameters that require a gradient."""
    dt = torch.float16
    g = torch.Generator(device="cuda").manual_seed(k)
    x, w, b = whole(g, m, k, dtype=dt), whole(g, 2 * n, k, dtype=dt, most=1), whole(g, 2 * n, dtype=dt)
    r, out = whole(g, m, n, dtype=dt), torch.empty(m, n, dtype=dt, device="cuda")
    kw = dict(bias=b, residual=r, activation="silu", gated=True)
    tecoops.linear(x, w, out, **kw)
    with_grad = torch.empty_like(out)
    tecoops.linear(x, torch.nn.Parameter(w.clone()), with_grad, **kw)
    assert torch.equal(out, with_grad) and not with_grad.requires_grad
    monkeypatch.setattr(tecoops, "_linear", None)
    again = torch.empty_like(out)
    tecoops.linear(x, w, again, **kw)
    assert torch.equal(out, again)


def test_past_32_bits():
    """Weights of more than 2^32 bytes and rows of x, residual and out far apart:
    the last rows and outputs come from where they are."""
    dt, k = torch.bfloat16, 8192
    n = (1 << 32) // (2 * k) + 300
    w = torch.zeros(n, k, dtype=dt, device="cuda")
    w[-1, -1], w[n - 2, 5], w[3, 7] = 2, 3, 4
    for m in (2, 70, 300):
        x = torch.zeros(m, k, dtype=dt, device="cuda")
        x[m - 1] = 1
        out = torch.full((m, n), 9.0, dtype=dt, device="cuda")
        tecoops.linear(x, w, out)
        assert (out[:m - 1] == 0).all()
        last = out[m - 1]
        assert (last[n - 1], last[n - 2], last[3]) == (2, 3, 4) and last.count_nonzero() == 3
    del w, out
    m, n, k, apart = 1100, 96, 64, 1 << 21
    wide = torch.empty(m * apart, dtype=dt, device="cuda")
    x = wide.view(m, apart)[:, :k]
    g = torch.Generator(device="cuda").manual_seed(1)
    x.copy_(whole(g, m, k, dtype=dt))
    res = wide.view(m, apart)[:, 1000:1000 + n]
    res.copy_(whole(g, m, n, dtype=dt))
    out = wide.view(m, apart)[:, 2000:2000 + n]
    w = whole(g, n, k, dtype=dt)
    tecoops.linear(x, w, out, residual=res)
    assert torch.equal(out, linear64(x, w, None, res, None, False).to(dt))


def test_no_rows_and_refusals():
    dt = torch.float16
    x, w = torch.zeros(4, 16, dtype=dt, device="cuda"), torch.zeros(6, 16, dtype=dt, device="cuda")
    out = torch.zeros(4, 6, dtype=dt, device="cuda")
    tecoops.linear(x[:0], w, out[:0])
    good = dict(bias=None, residual=None, activation=None, gated=False)
    for a, kw in [((x, w, out[:3]), {}), ((x, w[:5], out), {}), ((x, w[:, :8], out), {}),
                  ((x, w.t().contiguous().t(), out), {}), ((x.t(), w, out), {}),
                  ((x, w, out.t().contiguous().t()), {}), ((x[0], w, out), {}),
                  ((x, w, out), dict(gated=True)), ((x, w, out), dict(activation="tanh")),
                  ((x, w, out), dict(bias=out[0, :5])), ((x, w, out), dict(residual=out[:3])),
                  ((x, w, out), dict(residual=x)), ((x.cpu(), w, out), {}),
                  ((x, w.cpu(), out), {}), ((x.expand(4, 16)[:1].expand(4, 16), w, out), {})]:
        with pytest.raises(ValueError):
            tecoops.linear(*a, **{**good, **kw})
    for a, kw in [((x.float(), w, out), {}), ((x, w.bfloat16(), out), {}),
                  ((x, w, out.float()), {}), ((x, w, out), dict(bias=torch.zeros(6, device="cuda"))),
                  ((x, w, out), dict(residual=out.bfloat16()))]:
        with pytest.raises(TypeError):
            tecoops.linear(*a, **{**good, **kw})
