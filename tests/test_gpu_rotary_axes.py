"""Rotary positions of several axes against angles in extended precision.

Bound: the result's rounding (half a step) and, of |x1| + |x2|, 2^-21 for the
angle held as a 32-bit part of a turn (2 pi 2^-25), sin and cos (2 units), the
product and the sum; and 2^-50 of the position for 64-bit frequencies."""
import numpy as np
import pytest
import torch

import tecoops
from tecoops import TecoopsError

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def axis_of(sections, half, layout):
    if layout != "interleaved":
        return [a for a, n in enumerate(sections) for _ in range(n)]
    axes = len(sections)
    return [i % axes if i % axes and i < axes * sections[i % axes] else 0 for i in range(half)]


def angles(pos, sections, rot, base, layout):
    """[tokens, rot / 2] in extended precision."""
    half = rot // 2
    out = np.zeros((pos.shape[1], half), np.longdouble)
    for i, a in enumerate(axis_of(sections, half, layout)):
        j, n = (i - sum(sections[:a]), sections[a]) if layout == "per_axis" else (i, half)
        out[:, i] = pos[a].astype(np.longdouble) * np.longdouble(base) ** (-np.longdouble(j) / n)
    return out


def turned(x, ang, rot, neox):
    """x [T, H, D] float64 -> (turned, |x1| + |x2| of each element)."""
    half = rot // 2
    one = slice(0, half) if neox else slice(0, rot, 2)
    two = slice(half, rot) if neox else slice(1, rot, 2)
    c = np.cos(ang).astype(np.float64)[:, None]
    s = np.sin(ang).astype(np.float64)[:, None]
    y, size = x.copy(), np.zeros_like(x)
    y[..., one] = x[..., one] * c - x[..., two] * s
    y[..., two] = x[..., two] * c + x[..., one] * s
    size[..., one] = size[..., two] = np.abs(x[..., one]) + np.abs(x[..., two])
    return y, size


def check(got, x, pos, sections, rot, base, layout, neox, ang=None):
    T, D = x.shape[0], x.shape[-1]
    if ang is None:
        ang = angles(pos, sections, rot, base, layout)
    ref, size = turned(x.double().cpu().numpy(), ang, rot, neox)
    half = torch.finfo(x.dtype).eps / 2
    far = float(np.abs(pos).max()) if pos.size else 0.0
    bound = half * np.abs(ref) + (2.0 ** -21 + 2.0 ** -50 * far) * size * (1 + half) + 2.0 ** -25
    err = np.abs(got.double().cpu().numpy() - ref)
    assert (err <= bound).all(), (err / bound).max()
    rest = got[..., rot:]
    assert torch.equal(rest, x[..., rot:])


def make(seed, T, H, Hkv, D, dt):
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn(T, (H + 2 * Hkv) * D, generator=g, device="cuda").to(dt)
    return qkv, [t.unflatten(1, (-1, D)) for t in (qkv[:, :H * D], qkv[:, H * D:(H + Hkv) * D],
                                                   qkv[:, (H + Hkv) * D:])]


def positions(seed, axes, T, most):
    return torch.randint(0, most, (axes, T), generator=torch.Generator().manual_seed(seed))


CASES = [  # D, rot, sections, layout, neox
    (128, 128, [16, 24, 24], "contiguous", True), (128, 128, [24, 20, 20], "interleaved", True),
    (80, 80, [20, 20], "per_axis", True), (72, 72, [18, 18], "per_axis", True),
    (64, 32, [8, 4, 4], "contiguous", False), (128, 128, [22, 21, 21], "interleaved", False),
    (64, 64, [17, 15], "interleaved", True), (96, 96, [12, 12, 12, 12], "per_axis", False),
    (30, 22, [5, 3, 3], "contiguous", True), (30, 10, [3, 1, 1], "interleaved", False),
    (256, 256, [0, 64, 64], "contiguous", True), (2, 2, [1], "contiguous", True),
    (512, 512, [256], "interleaved", True), (128, 64, [12, 10, 10], "interleaved", True),
    (64, 64, [8, 8, 8, 8], "interleaved", True)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,rot,sections,layout,neox", CASES)
def test_rotation(D, rot, sections, layout, neox, dtype):
    """Slices of a wide product in place, near and far positions, with and
    without key; what lies between the rows stays."""
    for T, H, Hkv, most in ((1, 3, 1, 64), (37, 4, 2, 1 << 24), (5, 33, 33, 300000)):
        qkv, (q, k, v) = make(T, T, H, Hkv, D, DT[dtype])
        before = qkv.clone()
        q0, k0 = q.clone(), k.clone()
        pos = positions(T + D, len(sections), T, most)
        args = (D, sections), dict(is_neox=neox, base=500000.0, rot_dim=rot, layout=layout)
        tecoops.rotary_embedding_axes(pos.cuda(), qkv[:, :H * D], qkv[:, H * D:(H + Hkv) * D],
                                      *args[0], **args[1])
        check(q, q0, pos.numpy(), sections, rot, 500000.0, layout, neox)
        check(k, k0, pos.numpy(), sections, rot, 500000.0, layout, neox)
        assert torch.equal(v, before[:, (H + Hkv) * D:].unflatten(1, (-1, D)))
        alone = before.clone()
        tecoops.rotary_embedding_axes(pos.cuda(), alone[:, :H * D], None, *args[0], **args[1])
        assert torch.equal(alone[:, :H * D], qkv[:, :H * D])
        assert torch.equal(alone[:, H * D:], before[:, H * D:])


@pytest.mark.parametrize("D,rot,sections,layout,neox", CASES)
def test_table(D, rot, sections, layout, neox):
    """Angles from a table; a token with any position outside it is left as it
    is, whatever it holds."""
    T, H, Hkv, most, dt = 29, 4, 2, 50, torch.float16
    qkv, (q, k, _) = make(3, T, H, Hkv, D, dt)
    pos = positions(7, len(sections), T, most)
    pos[-1, 3], pos[0, 11], pos[-1, 20] = most, -1, 1 << 40
    left = [3, 11, 20]
    q[3, 0, 0] = k[11, 0, D - 1] = float("inf")
    q[20, 1] = float("nan")
    ang = np.outer(np.arange(most), 1.7 ** -np.arange(rot // 2))
    table = torch.from_numpy(np.concatenate([np.cos(ang), np.sin(ang)], 1)).float().cuda()
    q0, k0 = q.clone(), k.clone()
    tecoops.rotary_embedding_axes(pos.cuda(), q, k, D, sections, cos_sin_cache=table,
                                  is_neox=neox, layout=layout)
    for got, was in ((q, q0), (k, k0)):
        assert torch.equal(got[left].view(torch.int16), was[left].view(torch.int16))
    live = [t for t in range(T) if t not in left]
    p = pos.numpy()[:, live]
    turn = np.stack([ang[p[a], i] for i, a in enumerate(axis_of(sections, rot // 2, layout))], 1)
    for got, was in ((q, q0), (k, k0)):
        # the table's own rounding, 2^-25 of each of cos and sin, is in 2^-21
        check(got[live], was[live], p, sections, rot, 0, layout, neox, ang=turn)


@pytest.mark.parametrize("write_key", [False, True])
@pytest.mark.parametrize("with_table", [False, True])
@pytest.mark.parametrize("D,rot,sections,layout,neox", CASES)
def test_fused_equals_two_calls(D, rot, sections, layout, neox, with_table, write_key):
    """The fused kernel stores bit for bit what the two calls do: shuffled
    slots, slots outside the cache, positions outside the table."""
    T, H, Hkv, bs, nb, dt = 41, 6, 2, 5 if D == 30 else 16, 12, torch.bfloat16
    _, (q, k, v) = make(5, T, H, Hkv, D, dt)
    pos = positions(2, len(sections), T, 64)
    table = None
    if with_table:
        ang = np.outer(np.arange(64), 1.3 ** -np.arange(rot // 2))
        table = torch.from_numpy(np.concatenate([np.cos(ang), np.sin(ang)], 1)).float().cuda()
        pos[0, 9], pos[-1, 30] = 64, -5
        k[9, 0, 0], k[30, 1, D - 1] = float("inf"), float("nan")
    pos = pos.cuda()
    slots = torch.randperm(nb * bs, generator=torch.Generator().manual_seed(1))[:T].cuda()
    slots[4], slots[7], slots[8] = -1, nb * bs, 1 << 40
    kw = dict(cos_sin_cache=table, is_neox=neox, base=10000.0, rot_dim=rot, layout=layout)
    caches = [torch.full((nb, Hkv, bs, D), 3.0, dtype=dt, device="cuda") for _ in range(4)]
    q1, k1, q2, k2 = q.clone(), k.clone(), q.clone(), k.clone()
    tecoops.rotary_embedding_axes(pos, q1, k1, D, sections, **kw)
    tecoops.reshape_and_cache(k1, v.contiguous(), slots, caches[0], caches[1])
    tecoops.rotary_axes_reshape_and_cache(pos, q2, k2, v, slots, caches[2], caches[3], D, sections,
                                          write_key=write_key, **kw)

    def same(a, b):
        return torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))

    assert same(q1, q2)
    assert same(k2, k1 if write_key else k)
    assert same(caches[0], caches[2]) and same(caches[1], caches[3])


def test_one_axis_is_rotary_embedding():
    """One axis over a table is rotary_embedding, bit for bit."""
    T, H, D = 50, 4, 128
    qkv, (q, k, _) = make(1, T, H, H, D, torch.float16)
    pos = positions(1, 1, T, 99)
    ang = np.outer(np.arange(99), 10000.0 ** (-np.arange(64) / 64))
    table = torch.from_numpy(np.concatenate([np.cos(ang), np.sin(ang)], 1)).float().cuda()
    q1, k1 = q.contiguous().clone(), k.contiguous().clone()
    tecoops.rotary_embedding(pos[0].cuda(), q1, k1, D, table)
    tecoops.rotary_embedding_axes(pos.cuda(), q, k, D, [64], cos_sin_cache=table)
    assert torch.equal(q, q1) and torch.equal(k, k1)


def test_positions_of_a_larger_buffer_and_graph():
    """Rows of positions a distance apart; captured and replayed with new
    positions, each replay equal to the eager call."""
    T, H, Hkv, D, dt = 19, 8, 2, 128, torch.bfloat16
    buf = positions(3, 3, 64, 4000).cuda()
    _, (q, k, v) = make(8, T, H, Hkv, D, dt)
    slots = torch.arange(T, device="cuda")
    qs, kc, vc = q.contiguous().clone(), *(torch.zeros(4, Hkv, 16, D, dtype=dt, device="cuda")
                                           for _ in range(2))

    def step():
        tecoops.rotary_axes_reshape_and_cache(buf[:, :T], qs, k, v, slots, kc, vc, D, [24, 20, 20],
                                              layout="interleaved", base=1e6)

    qs.copy_(q)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for turn in range(4):
        buf.copy_(positions(10 + turn, 3, 64, 100000))
        qs.copy_(q)
        step()
        eager = [t.clone() for t in (qs, kc, vc)]
        check(qs, q, buf[:, :T].cpu().numpy(), [24, 20, 20], D, 1e6, "interleaved", True)
        qs.copy_(q)
        kc.zero_(), vc.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, (qs, kc, vc)))


def test_torch_ops():
    T, H, Hkv, D, dt = 9, 4, 2, 64, torch.float16
    _, (q, k, v) = make(4, T, H, Hkv, D, dt)
    pos, slots = positions(6, 3, T, 500).cuda(), torch.arange(T, device="cuda")
    caches = [torch.zeros(2, Hkv, 16, D, dtype=dt, device="cuda") for _ in range(4)]
    q1, k1, q2, k2 = q.clone(), k.clone(), q.clone(), k.clone()
    tecoops.rotary_axes_reshape_and_cache(pos, q1, k1, v, slots, caches[0], caches[1], D,
                                          [12, 10, 10], layout="interleaved", write_key=True)
    torch.ops.tecoops.rotary_axes_reshape_and_cache(pos, q2, k2, v, slots, caches[2], caches[3], D,
                                                    [12, 10, 10], None, True, 10000.0, D,
                                                    "interleaved", True)
    q3, k3 = q.clone(), k.clone()
    torch.ops.tecoops.rotary_embedding_axes(pos, q3, k3, D, [12, 10, 10], None, True, 10000.0, D,
                                            "interleaved")
    for a, b in ((q1, q2), (k1, k2), (q1, q3), (k1, k3), (caches[0], caches[2]),
                 (caches[1], caches[3])):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D", [64, 80, 128])
def test_without_the_torch_library(D, monkeypatch):
    T, H, Hkv, dt, half = 11, 4, 2, torch.bfloat16, D // 2
    _, (q, k, v) = make(4, T, H, Hkv, D, dt)
    pos, slots = positions(6, 2, T, 500).cuda(), torch.arange(T, device="cuda")
    got = []
    for _ in range(2):
        q1, k1, q2, k2 = q.clone(), k.clone(), q.clone(), k.clone()
        kc, vc = (torch.zeros(2, Hkv, 16, D, dtype=dt, device="cuda") for _ in range(2))
        sec = [half - 10, 10]
        tecoops.rotary_embedding_axes(pos, q1, k1, D, sec)
        tecoops.rotary_axes_reshape_and_cache(pos, q2, k2, v, slots, kc, vc, D, sec, write_key=True)
        assert torch.equal(q1, q2) and torch.equal(k1, k2)
        got.append((q1, k1, kc, vc))
        monkeypatch.setattr(tecoops, "_rotary_axes", None)
        monkeypatch.setattr(tecoops, "_rotary_axes_cache", None)
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_past_32_bits():
    """Cache rows and rows of q and k past 2^32 bytes."""
    T, H, Hkv, D, bs, dt = 3, 2, 2, 128, 16, torch.float16
    nb = (1 << 32) // (2 * Hkv * D * bs) + 8
    kc, vc = (torch.zeros(nb, Hkv, bs, D, dtype=dt, device="cuda") for _ in range(2))
    apart = 1 << 30
    wide = torch.zeros(T * apart, dtype=dt, device="cuda").view(T, apart)
    _, (q0, k0, v0) = make(2, T, H, Hkv, D, dt)
    q, k, v = wide[:, :H * D], wide[:, 1000:1000 + Hkv * D], wide[:, 2000:2000 + Hkv * D]
    for row, was in ((q, q0), (k, k0), (v, v0)):
        row.copy_(was.flatten(1))
    pos = positions(1, 3, T, 1000)
    slots = torch.tensor([nb * bs - 1, 5, nb * bs - 20], device="cuda")
    tecoops.rotary_axes_reshape_and_cache(pos.cuda(), q, k, v, slots, kc, vc, D, [24, 20, 20],
                                          layout="interleaved", write_key=True)
    check(q.unflatten(1, (H, D)), q0, pos.numpy(), [24, 20, 20], D, 10000.0, "interleaved", True)
    check(k.unflatten(1, (Hkv, D)), k0, pos.numpy(), [24, 20, 20], D, 10000.0, "interleaved", True)
    page, row = slots // bs, slots % bs
    assert torch.equal(kc[page, :, row].flatten(1), k) and torch.equal(vc[page, :, row].flatten(1), v)
    assert kc.count_nonzero() <= T * Hkv * D
    tecoops.rotary_embedding_axes(pos.cuda(), q, None, D, [24, 20, 20], layout="interleaved")


def test_no_tokens_and_refusals():
    T, H, D, dt = 6, 2, 64, torch.float16
    q, k = (torch.zeros(T, H, D, dtype=dt, device="cuda") for _ in range(2))
    pos = torch.zeros(3, T, dtype=torch.int64, device="cuda")
    f = tecoops.rotary_embedding_axes
    f(pos[:, :0], q[:0], k[:0], D, [12, 10, 10])
    for a in [(pos, q, k, D, [16, 16]), (pos[:2], q, k, D, [12, 10, 10]),
              (pos[:, :5], q, k, D, [12, 10, 10]), (pos, q[:5], k, D, [12, 10, 10]),
              (pos, q.transpose(1, 2), k, D, [12, 10, 10]), (pos, q, k.cpu(), D, [12, 10, 10]),
              (pos.t().contiguous().t(), q, k, D, [12, 10, 10]), (pos, q, k, 48, [12, 10, 10])]:
        with pytest.raises(ValueError):
            f(*a)
    for kw in (dict(layout="diagonal"), dict(cos_sin_cache=torch.zeros(9, D, 1, device="cuda")),
               dict(cos_sin_cache=torch.zeros(9, D, device="cuda"), rot_dim=32)):
        with pytest.raises(ValueError):
            f(pos, q, k, D, [12, 10, 10], **kw)
    with pytest.raises(TypeError):
        f(pos.int(), q, k, D, [12, 10, 10])
    with pytest.raises(TypeError):
        f(pos, q, k.bfloat16(), D, [12, 10, 10])
    with pytest.raises(TypeError):
        f(pos, q, k, D, [12, 10, 10], cos_sin_cache=torch.zeros(9, D, device="cuda").half())
    for kw in (dict(sections=[12, 10, 9]), dict(sections=[40, -4, -4]),
               dict(sections=[4, 14, 14], layout="interleaved"), dict(rot_dim=66), dict(base=0.0)):
        with pytest.raises(TecoopsError):
            f(pos, q, k, D, **{"sections": [12, 10, 10], **kw})
    c = torch.zeros(2, H, 16, D, dtype=dt, device="cuda")
    slots = torch.arange(T, device="cuda")
    g = tecoops.rotary_axes_reshape_and_cache
    for a in [(pos, q, k, k, slots[:5], c, c, D), (pos, q, k, k[:5], slots, c, c, D),
              (pos, q, None, k, slots, c, c, D), (pos, q, k, k, slots, c[:, :1], c, D),
              (pos, q, k, k, slots, c, c[:1], D), (pos, q, k, k.cpu(), slots, c, c, D)]:
        with pytest.raises(ValueError):
            g(*a, [12, 10, 10])
    with pytest.raises(TypeError):
        g(pos, q, k, k, slots.int(), c, c, D, [12, 10, 10])
