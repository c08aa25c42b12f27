"""The calls of the decoder-layer operators at their edges: an op that raises after its
launch has changed its in-place tensors once, and the error comes out; empty batches."""
import pytest
import torch

import tecoops
from tecoops import TecoopsError

pytestmark = pytest.mark.gpu


def after_launch(monkeypatch, name):
    real = getattr(tecoops, name)

    def op(*args):
        real(*args)
        raise RuntimeError("op: TECOOPS_STATUS_INTERNAL_ERROR")
    monkeypatch.setattr(tecoops, name, op)


@pytest.mark.parametrize("m", [1, 100])
def test_linear_into_its_residual(m, monkeypatch):
    x, w = torch.ones(m, 64, dtype=torch.float16, device="cuda"), torch.ones(32, 64, dtype=torch.float16,
                                                                             device="cuda")
    out = torch.ones(m, 32, dtype=torch.float16, device="cuda")
    after_launch(monkeypatch, "_linear")
    with pytest.raises(TecoopsError):
        tecoops.linear(x, w, out, residual=out)
    assert (out == 65).all()


@pytest.mark.parametrize("fused", [False, True])
def test_rotary_in_place(fused, monkeypatch):
    T, H, D, dt = 5, 2, 64, torch.float16
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(T, H * D, generator=g, device="cuda").to(dt) for _ in range(3))
    pos = torch.arange(3 * T, device="cuda").view(3, T)
    kc, vc = (torch.zeros(2, H, 16, D, dtype=dt, device="cuda") for _ in range(2))

    def call(q, k):
        if fused:
            tecoops.rotary_axes_reshape_and_cache(pos, q, k, v, torch.arange(T, device="cuda"), kc, vc, D,
                                                  [12, 10, 10], write_key=True)
        else:
            tecoops.rotary_embedding_axes(pos, q, k, D, [12, 10, 10])

    once = q.clone(), k.clone()
    call(*once)
    after_launch(monkeypatch, "_rotary_axes_cache" if fused else "_rotary_axes")
    with pytest.raises(TecoopsError):
        call(q, k)
    assert torch.equal(q, once[0]) and torch.equal(k, once[1])


@pytest.mark.parametrize("kv_heads", [1, 2, 5])
@pytest.mark.parametrize("fused", [False, True])
def test_rotary_of_no_tokens(fused, kv_heads):
    """An empty batch, through the Python functions and the torch ops alike."""
    D, dt, sec = 64, torch.float16, [12, 10, 10]
    q, k = (torch.zeros(0, h, D, dtype=dt, device="cuda") for h in (5, kv_heads))
    pos = torch.zeros(3, 0, dtype=torch.int64, device="cuda")
    kc = torch.ones(2, kv_heads, 16, D, dtype=dt, device="cuda")
    if fused:
        args = pos, q, k, k, pos[0], kc, kc, D, sec
        tecoops.rotary_axes_reshape_and_cache(*args)
        torch.ops.tecoops.rotary_axes_reshape_and_cache(*args, None, True, 1e4, D, "contiguous", False)
    else:
        tecoops.rotary_embedding_axes(pos, q, k, D, sec)
        torch.ops.tecoops.rotary_embedding_axes(pos, q, k, D, sec, None, True, 1e4, D, "contiguous")
    torch.cuda.synchronize()
    assert (kc == 1).all()


@pytest.mark.parametrize("table", [False, True])
@pytest.mark.parametrize("op", [True, False])
@pytest.mark.parametrize("T", [1, 2, 37])
def test_expanded_positions(T, op, table, monkeypatch):
    """positions.expand(3, -1), one row for all axes: as its copy, through the torch
    ops and the C functions, in place and with the cache store."""
    H, Hkv, D, dt, sec = 4, 2, 128, torch.bfloat16, [24, 20, 20]
    g = torch.Generator(device="cuda").manual_seed(T)
    q0, k0, v = (torch.randn(T, h * D, generator=g, device="cuda").to(dt) for h in (H, Hkv, Hkv))
    row = torch.randint(0, 100, (T,), generator=g, device="cuda")
    angles = torch.rand(100, D, generator=g, device="cuda") if table else None
    slots = torch.arange(T, device="cuda")
    if not op:
        monkeypatch.setattr(tecoops, "_rotary_axes", None)
        monkeypatch.setattr(tecoops, "_rotary_axes_cache", None)
    got = []
    for pos in (row.expand(3, -1), row[None].expand(3, T), row.expand(3, -1).contiguous()):
        q, k, q2 = q0.clone(), k0.clone(), q0.clone()
        kc, vc = (torch.zeros(3, Hkv, 16, D, dtype=dt, device="cuda") for _ in range(2))
        kw = dict(cos_sin_cache=angles, layout="interleaved")
        tecoops.rotary_embedding_axes(pos, q, k, D, sec, **kw)
        tecoops.rotary_axes_reshape_and_cache(pos, q2, k0, v, slots, kc, vc, D, sec, **kw)
        got.append((q, k, q2, kc, vc))
    assert not torch.equal(got[0][0], q0)
    for a in got[:2]:
        assert all(torch.equal(x, y) for x, y in zip(a, got[2]))


def test_overlapping_positions_are_refused():
    pos = torch.zeros(64, dtype=torch.int64, device="cuda").as_strided((3, 37), (1, 1))
    q = torch.zeros(37, 512, dtype=torch.float16, device="cuda")
    with pytest.raises(TecoopsError):
        tecoops.rotary_embedding_axes(pos, q, None, 128, [24, 20, 20])
