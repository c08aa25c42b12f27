"""Host checks of the 4-bit decode path's C entry points: bad arguments come back as
statuses before any device work, and how attention's keys are cut into splits."""
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


def caller(name, good):
    f = getattr(_lib.lib(), name)

    def call(**kw):
        a = {**good, **kw}
        assert set(a) == set(good)
        return f(*a.values())
    return call


def test_qk_norm_refusals(handle):
    sec = (ctypes.c_int * 1)(32)
    good = dict(h=handle, pos=P, ps=5, axes=1, sec=sec, lay=0, q=P, k=P, qw=P, kw=P, eps=1e-6, T=5, H=2, Hkv=1,
                D=64, rot=64, qs=128, ks=64, table=None, most=0, base=1e4, neox=1, dt=1)
    call = caller("tecoopsQkNormRotary", good)
    assert call(h=None) == NOT_INIT
    for kw in (dict(pos=None), dict(q=None), dict(qw=None), dict(kw=None), dict(T=0), dict(T=-1), dict(H=0),
               dict(Hkv=0), dict(D=0), dict(D=62), dict(rot=0), dict(rot=63), dict(rot=66), dict(qs=127),
               dict(ks=63), dict(axes=0), dict(axes=5), dict(lay=3), dict(sec=(ctypes.c_int * 1)(31)),
               dict(eps=-1e-6), dict(eps=float("nan")), dict(eps=float("inf")), dict(base=0.0),
               dict(table=P, most=0), dict(dt=0), dict(dt=2), dict(q=P + 1), dict(k=P + 1), dict(qw=P + 1),
               dict(kw=P + 1)):
        assert call(**kw) == BAD, kw
    assert call(axes=2, sec=None) == BAD
    assert call(D=1032, qs=2064, ks=1032) == NOT_SUP and call(T=1 << 24) == NOT_SUP
    assert call(D=62, rot=62, sec=None, T=(1 << 24) - 1) == NOT_SUP  # one head a wave: too many
    fused = dict(h=handle, pos=P, ps=5, axes=1, sec=None, lay=0, q=P, k=P, v=P, qw=P, kw=P, eps=1e-6, slots=P,
                 kc=P, vc=P, T=5, H=2, Hkv=1, D=64, rot=64, qs=128, ks=64, vs=64, table=None, most=0, base=1e4,
                 neox=1, nb=4, bs=16, wk=0, dt=1)
    call = caller("tecoopsQkNormRotaryReshapeAndCache", fused)
    assert call(h=None) == NOT_INIT
    for kw in (dict(k=None), dict(v=None), dict(slots=None), dict(kc=None), dict(vc=None), dict(qw=None),
               dict(kw=None), dict(vs=63), dict(nb=0), dict(bs=0), dict(eps=-1.0), dict(kc=P + 1),
               dict(v=P + 1), dict(T=0)):
        assert call(**kw) == BAD, kw
    assert call(nb=1 << 20, bs=1 << 20) == NOT_SUP


def test_append_refusals(handle):
    good = dict(h=handle, k=P, v=P, slots=P, kc=P, vc=P, ks=P, vs=P, T=5, H=2, D=64, kst=128, vst=128, nb=4,
                bs=16, dt=1)
    call = caller("tecoopsReshapeAndCacheInt4", good)
    assert call(h=None) == NOT_INIT
    for name in ("k", "v", "slots", "kc", "vc", "ks", "vs"):
        assert call(**{name: None}) == BAD, name
    for kw in (dict(T=-1), dict(H=0), dict(D=0), dict(nb=0), dict(bs=0), dict(kst=127), dict(vst=127), dict(dt=0),
               dict(k=P + 1), dict(v=P + 1), dict(kc=P + 2), dict(vc=P + 2), dict(ks=P + 2), dict(vs=P + 2)):
        assert call(**kw) == BAD, kw
    assert call(D=60) == NOT_SUP and call(D=520, kst=1040, vst=1040) == NOT_SUP
    assert call(nb=1 << 20, bs=1 << 20) == NOT_SUP and call(T=1 << 26) == NOT_SUP
    assert call(T=0) == OK  # no launch


def test_attention_refusals(handle):
    good = dict(h=handle, mq=1, mk=64, cu=P, kv=P, bt=P, bts=4, B=2, nblk=4, q=P, kc=P, vc=P, ks=P, vs=P, o=P,
                rows=2, H=8, Hkv=2, D=128, nb=16, bs=16, scale=-1.0, causal=1, ws=None, wb=0, dt=1)
    call = caller("tecoopsFlashAttentionInt4", good)
    assert call(h=None) == NOT_INIT
    for name in ("cu", "kv", "bt", "q", "kc", "vc", "ks", "vs", "o"):
        assert call(**{name: None}) == BAD, name
    for kw in (dict(B=0), dict(rows=-1), dict(nblk=-1), dict(nb=0), dict(bs=0), dict(H=0), dict(Hkv=0),
               dict(Hkv=3), dict(dt=0), dict(q=P + 8), dict(kc=P + 8), dict(vc=P + 4), dict(o=P + 2),
               dict(ks=P + 2), dict(vs=P + 2), dict(cu=P + 2), dict(kv=P + 2), dict(bt=P + 2), dict(ws=P + 8, wb=64),
               dict(bts=-1)):
        assert call(**kw) == BAD, kw
    for D in (16, 48, 224, 256):
        assert call(D=D) == NOT_SUP, D
    assert call(rows=0) == OK  # no launch
    assert call(rows=(1 << 31) - 1) == NOT_SUP  # columns past 2^31
    assert call(B=1 << 22, bts=0) == NOT_SUP    # grid
    size = ctypes.c_size_t(1)
    g = _lib.lib().tecoopsGetFlashAttentionInt4WorkspaceSize
    assert g(2, 2, 8, 2, 128, 1, 64, None) == BAD and g(2, 2, 8, 2, 128, 1, 0, ctypes.byref(size)) == BAD
    assert g(0, 2, 8, 2, 128, 1, 64, ctypes.byref(size)) == BAD
    assert g(2, 2, 8, 3, 128, 1, 64, ctypes.byref(size)) == BAD
    assert g(2, 2, 8, 2, 100, 1, 64, ctypes.byref(size)) == NOT_SUP
    assert g(2, 2, 8, 2, 128, 1, 64, ctypes.byref(size)) == OK and size.value == 0  # one split


def test_gemv_refusals(handle):
    good = dict(h=handle, w=P, s=P, z=P, x=P, y=P, B=2, n=32, k=256, g=64, ws=None, wb=0, dt=1)
    call = caller("tecoopsGemvInt4", good)
    assert call(h=None) == NOT_INIT
    for name in ("w", "s", "x", "y"):
        assert call(**{name: None}) == BAD, name
    for kw in (dict(B=-1), dict(n=0), dict(k=0), dict(g=0), dict(g=96), dict(dt=0), dict(w=P + 8), dict(s=P + 1),
               dict(z=P + 1), dict(x=P + 1), dict(y=P + 1), dict(ws=P + 2, wb=64)):
        assert call(**kw) == BAD, kw
    assert call(g=16) == NOT_SUP and call(k=48, g=48) == NOT_SUP
    assert call(n=(1 << 26) + 1) == NOT_SUP and call(B=(1 << 16) + 1) == NOT_SUP
    assert call(B=1 << 14, n=1 << 14) == NOT_SUP
    assert call(B=0) == OK  # no launch
    size = ctypes.c_size_t(1)
    g = _lib.lib().tecoopsGetGemvInt4WorkspaceSize
    assert g(2, 32, 256, None) == BAD and g(-1, 32, 256, ctypes.byref(size)) == BAD
    assert g(2, 0, 256, ctypes.byref(size)) == BAD and g(2, 32, 0, ctypes.byref(size)) == BAD
    assert g(0, 32, 256, ctypes.byref(size)) == OK and size.value == 0


@pytest.fixture(scope="module")
def parts(tmp_path_factory):
    d = tmp_path_factory.mktemp("parts")
    (d / "parts.cpp").write_text("""#include "gemv_int4.h"
extern "C" void parts(int b, int n, int k, unsigned long long room, long long *o) {
    const auto p = tecoops::gemv_int4_plan(b, n, k, room, 256);
    o[0] = p.dot; o[1] = p.parts; o[2] = (long long)p.bytes; o[3] = tecoops::gemv_int4_staged(b);
}
""")
    subprocess.run(["g++", "-std=c++17", "-fPIC", "-shared", "-I", CSRC, str(d / "parts.cpp"), "-o",
                    str(d / "parts.so")], check=True)
    lib = ctypes.CDLL(str(d / "parts.so"))
    lib.parts.argtypes = [ctypes.c_int] * 3 + [ctypes.c_ulonglong, ctypes.c_void_p]

    def run(b, n, k, room=(1 << 63)):
        o = (ctypes.c_longlong * 4)()
        lib.parts(b, n, k, room, o)
        return list(o)
    return run


def test_parts_of_k(parts):
    """No more parts than stages of K, and their sums fit the workspace."""
    for b in (1, 2, 3, 8, 9, 33, 64, 65, 1000):
        for n in (1, 64, 65, 1000, 4096, 28672, 1 << 20):
            for k in (32, 512, 513, 1024, 4096, 14336, 1 << 20):
                for room in (0, 1 << 20, 1 << 63):
                    dot, count, need, staged = parts(b, n, k, room)
                    assert staged >= min(b, 64) and staged in (8, 16, 32, 48, 64)
                    assert 1 <= count <= max(1, k // 1024) and need <= room
                    assert need == (b * n * 4 * count if count > 1 else 0)
                    assert count == 1 or not dot


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan4")
    (d / "plan.cpp").write_text("""#include "fa_int4.h"
extern "C" void plan(int b, int h, int hkv, int d, int rows, int keys, unsigned long long room, long long *o) {
    const auto p = tecoops::fa4::make_plan(b, h, hkv, d, rows, keys, room, 256);
    o[0] = p.split; o[1] = p.split ? p.ct * 16 : p.waves * 32; o[2] = p.tiles; o[3] = p.cols;
    o[4] = p.split_len; o[5] = p.splits; o[6] = (long long)p.bytes;
}
""")
    subprocess.run(["g++", "-std=c++17", "-fPIC", "-shared", "-I", CSRC, str(d / "plan.cpp"), "-o",
                    str(d / "plan.so")], check=True)
    lib = ctypes.CDLL(str(d / "plan.so"))
    lib.plan.argtypes = [ctypes.c_int] * 6 + [ctypes.c_ulonglong, ctypes.c_void_p]

    def run(b, h, hkv, d, rows, keys, room=(1 << 63)):
        o = (ctypes.c_longlong * 7)()
        lib.plan(b, h, hkv, d, rows, keys, room, o)
        return list(o)
    return run


@pytest.mark.parametrize("room", [0, 1000, 1 << 20, 1 << 63])
def test_splits_cover_the_keys(plan, room):
    """Tiles hold the columns, splits the keys, none empty, and the states fit the
    workspace."""
    for b in (1, 3, 64, 1000):
        for h, hkv in ((1, 1), (8, 1), (32, 8), (64, 1), (40, 8)):
            for rows in (1, 2, 5, 17, 64, 1000):
                for keys in (1, 31, 32, 128, 129, 777, 8192, 100000, (1 << 31) - 4097):
                    split, tile, tiles, cols, length, splits, need = plan(b, h, hkv, 128, rows, keys, room)
                    assert cols == h // hkv * rows and (tiles - 1) * tile < cols <= tiles * tile
                    # whole rounds of a workgroup's waves, whole tiles of keys
                    assert length % (128 if split else 96) == 0 or splits == 1
                    assert need <= room
                    assert splits >= 1 and (splits - 1) * length < keys
                    assert splits * length >= keys or splits == 1
                    assert need == (0 if splits == 1 else b * hkv * splits * cols * (128 + 2) * 4)
