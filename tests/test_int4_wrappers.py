"""The 4-bit decode path's Python functions: arguments that they refuse (checked
without the torch ops too, whose checks are the same), and that a torch op which
raised is not called again (no GPU: ops and checks of the device are stubs)."""
import pytest
import torch

import tecoops
from tecoops import TecoopsError, _lib

F16, U8, I32, I64 = torch.float16, torch.uint8, torch.int32, torch.int64
T, H, HKV, D, NB, BS = 3, 4, 2, 64, 4, 16


def z(*shape, dtype=F16):
    return torch.zeros(shape, dtype=dtype)


def args():
    cache = dict(kc=z(NB, HKV, BS, D // 2, dtype=U8), vc=z(NB, HKV, BS, D // 2, dtype=U8), ks=z(NB, HKV, BS, 2),
                 vs=z(NB, HKV, BS, 2))
    return {
        "_qk_norm": dict(pos=z(T, dtype=I64), q=z(T, H * D), k=z(T, HKV * D), qw=z(D), kw=z(D), D=D),
        "_qk_norm_cache": dict(pos=z(T, dtype=I64), q=z(T, H * D), k=z(T, HKV * D), v=z(T, HKV * D), qw=z(D), kw=z(D),
                               slots=z(T, dtype=I64), kc=z(NB, HKV, BS, D), vc=z(NB, HKV, BS, D), D=D),
        "_cache_int4": dict(k=z(T, HKV, D), v=z(T, HKV, D), slots=z(T, dtype=I64), **cache),
        "_attn_int4": dict(q=z(T, H, D), **cache, mq=1, cu=z(T + 1, dtype=I32), mk=64, used=z(T, dtype=I32),
                           scale=None, causal=True, table=z(T, 4, dtype=I32), out=z(T, H, D)),
        "_gemv_int4": dict(w=z(32, 64, dtype=U8), s=z(32, 2), x=z(T, 128), out=z(T, 32), zeros=z(32, 2)),
    }


FUNCTIONS = {"_qk_norm": tecoops.qk_norm_rotary, "_qk_norm_cache": tecoops.qk_norm_rotary_reshape_and_cache,
             "_cache_int4": tecoops.reshape_and_cache_int4, "_attn_int4": tecoops.flash_attn_varlen_int4,
             "_gemv_int4": tecoops.gemv_int4}
NAMES = list(FUNCTIONS)


def call(name, **change):
    a = args()[name]
    assert set(change) <= set(a)
    return FUNCTIONS[name](*{**a, **change}.values())


@pytest.fixture
def launched(monkeypatch):
    got = []
    monkeypatch.setattr(tecoops, "_check_cuda", lambda *ts: None)
    monkeypatch.setattr(tecoops, "_handle", lambda device: None)
    monkeypatch.setattr(tecoops, "_workspace", lambda *a: torch.empty(1, dtype=U8))
    monkeypatch.setattr(tecoops, "_call_on", lambda device, name, *a: got.append(name))
    for name in NAMES:
        monkeypatch.setattr(tecoops, name, None)
    return got


@pytest.mark.parametrize("name", NAMES)
def test_good_arguments_launch(name, launched):
    call(name)
    assert len(launched) == 1


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("error", [RuntimeError("x: TECOOPS_STATUS_INTERNAL_ERROR"), RuntimeError("no memory"),
                                   ValueError("something")])
def test_an_op_that_raised_is_not_called_again(name, error, launched, monkeypatch):
    def op(*a):
        launched.append("op")
        raise error
    monkeypatch.setattr(tecoops, name, op)
    with pytest.raises((TecoopsError, type(error))) as e:
        call(name)
    assert launched == ["op"]
    if "INTERNAL" in str(error):
        assert e.value.status == _lib.INTERNAL_ERROR


def wide(*shape, dtype=F16):
    """A tensor of this shape whose last dimension is not packed."""
    return torch.zeros(*shape[:-1], 2 * shape[-1], dtype=dtype)[..., ::2]


REFUSED = [
    ("_qk_norm", dict(pos=z(T + 1, dtype=I64)), dict(pos=z(T, dtype=I32)), dict(pos=z(2, T, dtype=I64)),
     dict(q=z(T, H * D + 1)), dict(q=wide(T, H * D)), dict(k=z(T + 1, HKV * D)), dict(qw=z(D + 1)), dict(kw=None),
     dict(kw=z(1, D)), dict(qw=z(D, dtype=torch.bfloat16)), dict(k=z(T, HKV * D, dtype=torch.bfloat16)),
     dict(q=z(T, H * D, dtype=torch.float32)), dict(qw=wide(D))),
    ("_qk_norm_cache", dict(slots=z(T + 1, dtype=I64)), dict(slots=z(T, dtype=I32)), dict(v=z(T, H * D)),
     dict(v=wide(T, HKV * D)), dict(kc=z(NB, H, BS, D)), dict(vc=z(NB, HKV, BS, D + 8)), dict(k=None),
     dict(kc=z(NB, HKV, BS, D, dtype=torch.bfloat16)), dict(kw=z(D - 1))),
    ("_cache_int4", dict(k=z(T, HKV * D)), dict(v=z(T, H, D)), dict(k=wide(T, HKV, D)), dict(slots=z(T - 1, dtype=I64)),
     dict(slots=z(T, dtype=I32)), dict(kc=z(NB, HKV, BS, D, dtype=U8)), dict(vc=z(NB + 1, HKV, BS, D // 2, dtype=U8)),
     dict(ks=z(NB, HKV, BS)), dict(vs=z(NB, HKV, BS, 2, dtype=torch.bfloat16)), dict(kc=z(NB, HKV, BS, D // 2)),
     dict(k=z(T, HKV, D, dtype=torch.bfloat16)), dict(ks=wide(NB, HKV, BS, 2)),
     dict(kc=z(NB, H, BS, D // 2, dtype=U8), vc=z(NB, H, BS, D // 2, dtype=U8), ks=z(NB, H, BS, 2), vs=z(NB, H, BS, 2))),
    ("_attn_int4", dict(q=z(T, H * D)), dict(out=z(T, H, D + 8)), dict(q=wide(T, H, D)), dict(cu=z(T, dtype=I32)),
     dict(cu=z(T + 1, dtype=I64)), dict(used=z(T + 1, dtype=I32)), dict(table=z(T + 1, 4, dtype=I32)),
     dict(table=wide(T, 4, dtype=I32)), dict(table=z(T, 4, dtype=I64)), dict(out=z(T, H, D, dtype=torch.bfloat16)),
     dict(ks=z(NB, HKV, BS, 2, dtype=torch.bfloat16)), dict(kc=z(NB, HKV, BS, D, dtype=U8))),
    ("_gemv_int4", dict(x=z(T, 127)), dict(out=z(T, 31)), dict(s=z(31, 2)), dict(s=z(32, 3)), dict(s=z(32, 0)),
     dict(zeros=z(32, 1)), dict(w=z(32, 64, dtype=torch.int8)), dict(x=wide(T, 128)), dict(w=wide(32, 64, dtype=U8)),
     dict(s=z(32, 2, dtype=torch.bfloat16)), dict(x=z(T, 1, 128)), dict(out=z(T, 32, dtype=torch.bfloat16))),
]


@pytest.mark.parametrize("name,change", [(n, c) for n, *cs in REFUSED for c in cs])
def test_refused(name, change, launched):
    with pytest.raises((ValueError, TypeError)):
        call(name, **change)
    assert launched == []


def test_nothing_to_do(launched):
    e = z(0, HKV * D)
    tecoops.qk_norm_rotary(z(0, dtype=I64), z(0, H * D), e, z(D), z(D), D)
    call("_qk_norm_cache", pos=z(0, dtype=I64), q=z(0, H * D), k=e, v=e, slots=z(0, dtype=I64))
    call("_cache_int4", k=z(0, HKV, D), v=z(0, HKV, D), slots=z(0, dtype=I64))
    call("_attn_int4", q=z(0, H, D), out=z(0, H, D))
    call("_gemv_int4", x=z(0, 128), out=z(0, 32))
    assert launched == []


def test_several_axes_and_a_query_alone(launched):
    tecoops.qk_norm_rotary(z(3, T, dtype=I64), z(T, H, D), None, z(D), None, D, sections=[12, 10, 10],
                           layout="interleaved")
    with pytest.raises(ValueError):
        tecoops.qk_norm_rotary(z(3, T, dtype=I64), z(T, H, D), None, z(D), None, D, sections=[12, 20])
    assert launched == ["tecoopsQkNormRotary"]
