"""linear and moe_layer on tensors that start off 16-byte (and off 8-byte) addresses:
slices of a buffer, each tensor alone and all together.  Whole numbers small enough
for every intermediate to be exact give the rounding of the exact value bit for bit,
and what lies around `out` stays."""
import pytest
import torch

import tecoops
from test_gpu_linear import linear64, whole
from test_gpu_moe import even_logits, layer64, route64, run, sparse_rows

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def moved(t, by):
    """t, `by` elements behind an allocation's start, 7.0 around it."""
    buf = torch.full((t.numel() + 24,), 7.0, dtype=t.dtype, device="cuda")
    buf[by:by + t.numel()] = t.flatten()
    return buf[by:by + t.numel()].view(t.shape), buf


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("k", [64, 136, 4096])
@pytest.mark.parametrize("m,n", [(1, 264), (64, 72), (200, 128), (9, 4096)])
def test_linear(m, n, k, gated, dtype):
    dt = DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(m + k)
    rows = n * (1 + gated)
    x, w = whole(g, m, k, dtype=dt), whole(g, rows, k, dtype=dt)
    w[:, 40:] = 0  # gated products stay exact
    w[:, k - 8:] = 1 - gated
    b, r = whole(g, rows, dtype=dt), whole(g, m, n, dtype=dt)
    ref = linear64(x, w, b, r, None, gated).to(dt)
    for off in (dict(x=1), dict(w=1), dict(r=1), dict(o=1), dict(b=1), dict(o=4, r=4), dict(x=8, w=8),
                dict(x=4), dict(x=1, w=3, r=5, o=7, b=1)):
        a = {name: moved(t, off.get(name, 0)) for name, t in
             dict(x=x, w=w, b=b, r=r, o=torch.zeros_like(r)).items()}
        out, buf = a["o"]
        tecoops.linear(a["x"][0], a["w"][0], out, bias=a["b"][0], residual=a["r"][0], gated=gated)
        assert torch.equal(out, ref), off
        at = off.get("o", 0)
        assert (buf[:at] == 7).all() and (buf[at + m * n:] == 7).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("T", [1, 8, 40])
@pytest.mark.parametrize("H,I,E,k", [(64, 32, 4, 2), (264, 136, 16, 4), (4096, 64, 8, 2)])
def test_moe(T, H, I, E, k, dtype):
    dt = DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(T + H)
    x = whole(g, T, H, dtype=dt, most=2)
    w_in, w_out = sparse_rows(g, E, 2 * I, H, dtype=dt), whole(g, E, H, I, dtype=dt)
    logits = even_logits(g, T, E, k)
    ids, weights = route64(logits, k, True)
    ref = layer64(x, w_in, w_out, ids, weights, "relu")[0].to(dt)
    for off in (dict(x=1), dict(w=1), dict(v=1), dict(o=1), dict(o=2), dict(l=1), dict(o=4),
                dict(x=4, w=4, v=4), dict(x=1, w=3, v=5, o=7, l=1)):
        a = {name: moved(t, off.get(name, 0)) for name, t in
             dict(x=x, w=w_in, v=w_out, l=logits, o=torch.zeros_like(x)).items()}
        out, buf = a["o"]
        tecoops.moe_layer(a["x"][0], a["w"][0], a["v"][0], a["l"][0], k, out, activation="relu")
        assert torch.equal(out, ref), off
        at = off.get("o", 0)
        assert (buf[:at] == 7).all() and (buf[at + T * H:] == 7).all()
    assert torch.equal(run(x, w_in, w_out, logits, k, act="relu")[0], ref)
