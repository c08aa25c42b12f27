"""Host checks of the decoder-layer operators' C entry points: bad arguments come
back as statuses before any device work, and how a product is cut into tiles."""
import ctypes
import os
import subprocess

import pytest

from tecoops import _lib

BAD, NOT_INIT, NOT_SUP, OK = _lib.BAD_PARAM, _lib.NOT_INITIALIZED, _lib.NOT_SUPPORTED, _lib.SUCCESS
REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(REPO, "teco-ops_amd", "csrc")
P = 0x1000  # never dereferenced: the checks come first


@pytest.fixture
def handle():
    h = ctypes.c_void_p()
    assert _lib.lib().tecoopsCreate(ctypes.byref(h)) == OK
    yield h
    assert _lib.lib().tecoopsDestroy(h) == OK


def test_linear_refusals(handle):
    f = _lib.lib().tecoopsLinear
    good = dict(h=handle, x=P, xs=64, w=P, b=P, r=P, rs=32, o=P, os=32, m=4, n=32, k=64, act=0,
                gated=0, ws=None, wb=0, dt=1)

    def call(**kw):
        a = {**good, **kw}
        return f(*(a[k] for k in good))

    assert call(h=None) == NOT_INIT
    for kw in (dict(x=None), dict(w=None), dict(o=None), dict(m=-1), dict(n=0), dict(n=-4),
               dict(k=0), dict(xs=63), dict(os=31), dict(rs=31), dict(act=5), dict(act=-1),
               dict(dt=0), dict(dt=2), dict(x=P + 1), dict(w=P + 1), dict(b=P + 1), dict(r=P + 1),
               dict(o=P + 1)):
        assert call(**kw) == BAD, kw
    assert call(k=(1 << 21) + 8, xs=(1 << 21) + 8) == NOT_SUP
    assert call(xs=(1 << 21) + 8) == NOT_SUP
    assert call(n=(1 << 23) + 4, os=1 << 31, rs=1 << 31) == NOT_SUP
    assert call(m=(1 << 31) - 1, n=2000, os=2000, rs=2000) == NOT_SUP  # too many tiles
    assert call(m=0) == OK  # no launch
    size = ctypes.c_size_t(1)
    g = _lib.lib().tecoopsGetLinearWorkspaceSize
    assert g(4, 4, 4, 0, None) == BAD and g(-1, 4, 4, 0, ctypes.byref(size)) == BAD
    assert g(4, 0, 4, 0, ctypes.byref(size)) == BAD and g(4, 4, 0, 0, ctypes.byref(size)) == BAD
    assert g(0, 4, 4, 0, ctypes.byref(size)) == OK and size.value == 0


def test_rotary_axes_refusals(handle):
    L = _lib.lib()

    def axes(sections, layout=0, n=None, half=32, **kw):
        s = (ctypes.c_int * 8)(*sections)
        a = dict(h=handle, pos=P, stride=5, q=P, k=P, T=5, H=2, Hkv=1, D=64, rot=2 * half, qs=128,
                 ks=64, table=None, most=0, base=1e4, neox=1, dt=1)
        a.update(kw)
        front = (a["h"], a["pos"], a["stride"], len(sections) if n is None else n,
                 s if kw.get("sec", True) else None, layout, a["q"], a["k"])
        size = (a["T"], a["H"], a["Hkv"], a["D"], a["rot"], a["qs"], a["ks"])
        tail = (a["table"], a["most"], a["base"], a["neox"])
        plain = L.tecoopsRotaryEmbeddingAxes(*front, *size, *tail, a["dt"])
        fused = L.tecoopsRotaryAxesReshapeAndCache(*front, P, P, P, P, *size, 64, *tail, 4, 16, 0,
                                                   a["dt"])
        assert plain == fused
        return plain

    assert axes([32], h=None) == NOT_INIT
    for sections, layout in (([16, 15], 0), ([16, 17], 0), ([33, -1], 0), ([4, 14, 14], 1),
                             ([10, 11, 11], 1), ([32], 3), ([32], -1), ([8, 8, 8, 4, 4], 0)):
        assert axes(sections, layout) == BAD, (sections, layout)
    assert axes([32], n=0) == BAD and axes([32], sec=False) == BAD
    for kw in (dict(stride=4), dict(pos=None), dict(q=None), dict(T=0), dict(T=-1), dict(H=0),
               dict(Hkv=0), dict(D=0), dict(D=63), dict(half=0), dict(qs=127), dict(ks=63),
               dict(table=P, most=0), dict(base=0.0), dict(base=float("nan")), dict(dt=0)):
        assert axes([16, 16] if kw.get("half", 1) else [0, 0], **kw) == BAD, kw
    s = (ctypes.c_int * 1)(32)
    fused = L.tecoopsRotaryAxesReshapeAndCache
    for none in (7, 8, 9, 10, 11):  # key, value, slots, caches
        a = [handle, P, 5, 1, s, 0, P, P, P, P, P, P, 5, 2, 1, 64, 64, 128, 64, 64, None, 0, 1e4, 1,
             4, 16, 0, 1]
        a[none] = None
        assert fused(*a) == BAD, none
    for at, bad in ((24, 0), (25, 0), (19, 63)):  # blocks, block size, value stride
        a = [handle, P, 5, 1, s, 0, P, P, P, P, P, P, 5, 2, 1, 64, 64, 128, 64, 64, None, 0, 1e4, 1,
             4, 16, 0, 1]
        a[at] = bad
        assert fused(*a) == BAD, at
    a[19], a[24], a[25] = 64, 1 << 20, 1 << 20
    assert fused(*a) == NOT_SUP


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text("""#include "linear.h"
extern "C" void plan(int m, int n, int k, int gated, int copy, unsigned long long ws, long long *o) {
    const auto p = tecoops::linear_plan(m, n, k, gated != 0, copy != 0, ws, 256);
    o[0] = tecoops::kLinearTiles[p.tile].bm; o[1] = tecoops::kLinearTiles[p.tile].bn;
    o[2] = p.tiles_m; o[3] = p.tiles_n; o[4] = p.splits; o[5] = p.stages;
    o[6] = static_cast<long long>(p.bytes); o[7] = p.stream; o[8] = p.tile;
}
extern "C" int first_loaded() { return tecoops::kLinearFirstLoaded; }
""")
    subprocess.run(["g++", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__=1", "-I", CSRC,
                    "-I", os.path.join(REPO, "include"), "-I", "/opt/rocm/include",
                    str(d / "plan.cpp"), "-o", str(d / "plan.so")], check=True)
    lib = ctypes.CDLL(str(d / "plan.so"))
    lib.plan.argtypes = [ctypes.c_int] * 5 + [ctypes.c_ulonglong, ctypes.c_void_p]

    def run(m, n, k, gated=0, copy=1, ws=(1 << 63)):
        o = (ctypes.c_longlong * 9)()
        lib.plan(m, n, k, gated, copy, ws, o)
        return list(o)
    run.first_loaded = lib.first_loaded()
    return run


@pytest.mark.parametrize("copy", [0, 1])
@pytest.mark.parametrize("gated", [0, 1])
def test_plan_covers_the_product(plan, gated, copy):
    """Tiles cover the rows and outputs, splits cover K with none empty, and the
    workspace holds every split's sums of every row of W."""
    for m in (1, 8, 33, 64, 65, 127, 128, 129, 333, 1000, 8192, 70000):
        for n in (1, 63, 64, 65, 300, 4096, 14336, 100000):
            for k in (1, 8, 64, 65, 512, 588, 4096, 14336, 100000):
                for ws in (0, 1 << 20, 1 << 63):
                    bm, bn, tm, tn, splits, stages, need, stream, tile = plan(m, n, k, gated, copy, ws)
                    if stream:
                        assert copy and m <= 64 and need == 0
                        continue
                    out = bn // 2 if gated else bn
                    assert (tm - 1) * bm < m <= tm * bm and (tn - 1) * out < n <= tn * out
                    total = -(-k // 64)
                    assert splits >= 1 and (splits - 1) * stages < total <= splits * stages
                    assert need == (splits * m * n * (2 if gated else 1) * 4 if splits > 1 else 0)
                    assert need <= ws
                    assert copy or tile >= plan.first_loaded


def test_plan_by_size(plan):
    """Wide products of few rows stream W, few rows of W with a long K do not;
    large products take the largest tile, unsplit."""
    assert plan(1, 4096, 4096)[7] and plan(32, 14336, 4096)[7] and plan(24, 14336, 4096, gated=1)[7]
    assert not plan(64, 1024, 14336)[7] and plan(64, 1024, 14336)[4] > 1
    assert plan(8192, 14336, 4096, gated=1)[:2] == [256, 256] and plan(8192, 14336, 4096)[4] == 1
    assert plan(512, 512, 512)[:2] == [64, 64]


def test_moe_refusals(handle):
    f = _lib.lib().tecoopsMoeLayer
    good = dict(h=handle, x=P, xs=64, wi=P, wo=P, lg=P, lt=0, o=P, ids=None, w=None, T=2, H=64, I=32,
                E=8, k=2, rn=1, act=2, ws=P, wb=1 << 40, dt=1)

    def call(**kw):
        a = {**good, **kw}
        return f(*(a[k] for k in good))

    assert call(h=None) == NOT_INIT
    for kw in (dict(x=None), dict(wi=None), dict(wo=None), dict(lg=None), dict(o=None), dict(T=-1),
               dict(H=0), dict(I=0), dict(E=0), dict(k=0), dict(k=9), dict(xs=63), dict(act=5),
               dict(act=-1), dict(dt=0), dict(lt=9), dict(lt=4), dict(x=P + 1), dict(wi=P + 1),
               dict(wo=P + 1), dict(o=P + 1), dict(lg=P + 2), dict(ids=P + 2), dict(w=P + 2),
               dict(wb=100), dict(wb=0), dict(ws=P + 8)):
        assert call(**kw) == BAD, kw
    assert call(E=1025) == NOT_SUP and call(E=64, k=33) == NOT_SUP
    assert call(H=(1 << 16) + 8, xs=1 << 21) == NOT_SUP and call(I=(1 << 16) + 8) == NOT_SUP
    assert call(T=0) == OK  # no launch
    # the next slice's first token would pass 2^31
    assert call(T=(1 << 31) - 1, H=1, I=1, E=1, k=1) == NOT_SUP and call(T=(1 << 30) + 1) == NOT_SUP
    g = _lib.lib().tecoopsGetMoeLayerWorkspaceSize
    size = ctypes.c_size_t(1)
    assert g(2, 64, 32, 8, 2, None) == BAD and g(2, 64, 32, 8, 9, ctypes.byref(size)) == BAD
    assert g(2, 64, 32, 2000, 9, ctypes.byref(size)) == NOT_SUP
    assert g(0, 64, 32, 8, 2, ctypes.byref(size)) == OK and size.value == 0


@pytest.fixture(scope="module")
def space(tmp_path_factory):
    d = tmp_path_factory.mktemp("space")
    (d / "space.cpp").write_text("""#include "moe.h"
extern "C" void space(int t, int h, int i, int e, int k, long long *o) {
    const auto s = tecoops::moe_space(t, h, i, e, k);
    const long long v[] = {s.pairs, s.items, s.rows, s.h_stride, (long long)s.items_at,
                           (long long)s.ids_at, (long long)s.token_at, (long long)s.slot_at,
                           (long long)s.weight_at, (long long)s.cols_at, (long long)s.h_at,
                           (long long)s.part_at, (long long)s.bytes};
    for (int j = 0; j < 13; ++j) o[j] = v[j];
}
extern "C" int wrows(int n, int t, int k, int e, int rows) {
    return tecoops::moe_wrows(n, t, k, e, rows, 256);
}
""")
    subprocess.run(["g++", "-std=c++17", "-fPIC", "-shared", "-I", CSRC, str(d / "space.cpp"), "-o",
                    str(d / "space.so")], check=True)
    return ctypes.CDLL(str(d / "space.so"))


def test_moe_workspace_holds_any_routing(space):
    """Parts of the workspace do not overlap; the items are enough for every
    spread of the pairs over the experts."""
    import random
    r = random.Random(1)
    for _ in range(600):
        E = r.choice([1, 2, 5, 8, 64, 128, 1000])
        k, T = r.randint(1, min(E, 32)), r.choice([1, 2, 4, 5, 9, 16, 17, 100, 511, 512, 513, 2000])
        H, I = r.choice([1, 8, 70, 4096]), r.choice([1, 8, 33, 14336])
        o = (ctypes.c_longlong * 13)()
        space.space(T, H, I, E, k, o)
        pairs, items, rows, stride, *at, total = list(o)
        assert pairs == min(T, 512) * k and stride % 8 == 0 and I <= stride < I + 8
        few = T <= 8
        sizes = [16 * items, 4 * pairs, 4 * pairs, 4 * pairs, 4 * pairs, few * 64 * items,
                 2 * pairs * stride, 4 * pairs * H]
        assert at[0] >= 4
        for a, s, nxt in zip(at, sizes, at[1:] + [total]):
            assert a % 256 == 0 and a + s <= nxt
        # the spread with the most items: one pair over a multiple of `rows` in as
        # many experts as possible
        t = min(T, 512)
        counts, left = [0] * E, pairs
        for e in range(E):
            counts[e] = min(1, left)
            left -= counts[e]
        for e in range(E):
            more = min(left, (t - counts[e]) // rows * rows)
            counts[e] += more
            left -= more
        for e in range(E):
            more = min(left, t - counts[e])
            counts[e] += more
            left -= more
        assert left == 0 and sum(-(-c // rows) for c in counts) <= items
        assert T > 4 or rows >= T
        assert space.wrows(2 * I, t, k, E, rows) in (16, 32, 64, 128)
