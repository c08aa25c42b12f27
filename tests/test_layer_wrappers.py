"""The decoder-layer operators' Python functions when the torch op below raises: the
op may have launched by then and some outputs are inputs too, so it is never called
again, nor is the C function in its place (no GPU: the op is a stub)."""
import pytest
import torch

import tecoops
from tecoops import TecoopsError, _lib

T, H, D, E, K = 3, 2, 64, 4, 2
F16 = torch.float16


def tensors():
    def z(*shape, dtype=F16):
        return torch.zeros(shape, dtype=dtype)
    return dict(x=z(T, 64), w=z(32, 64), out=z(T, 32), w_in=z(E, 64, 64), w_out=z(E, 64, 32),
                logits=z(T, E, dtype=torch.float32), y=z(T, 64), pos=z(3, T, dtype=torch.int64),
                q=z(T, H * D), k=z(T, H * D), v=z(T, H * D), slots=z(T, dtype=torch.int64),
                kc=z(2, H, 16, D), vc=z(2, H, 16, D))


def calls(t):
    sec = [12, 10, 10]
    return {
        "_linear": lambda **kw: tecoops.linear(t["x"], t["w"], t["out"], residual=t["out"], **kw),
        "_moe_layer": lambda **kw: tecoops.moe_layer(t["x"], t["w_in"], t["w_out"], t["logits"], K,
                                                     t["y"], **kw),
        "_rotary_axes": lambda **kw: tecoops.rotary_embedding_axes(t["pos"], t["q"], t["k"], D, sec, **kw),
        "_rotary_axes_cache": lambda **kw: tecoops.rotary_axes_reshape_and_cache(
            t["pos"], t["q"], t["k"], t["v"], t["slots"], t["kc"], t["vc"], D, sec, **kw)}


@pytest.fixture
def stub(monkeypatch):
    """stub(name, error): op `name` counts its calls and raises `error`; the list of
    all launches, the C functions' among them."""
    launched = []
    monkeypatch.setattr(tecoops, "_check_cuda", lambda *ts: None)
    monkeypatch.setattr(tecoops, "_handle", lambda device: None)
    monkeypatch.setattr(tecoops, "_workspace", lambda *a: torch.empty(1, dtype=torch.uint8))
    monkeypatch.setattr(tecoops, "_call_on", lambda device, name, *a: launched.append(name))

    def put(name, error):
        def op(*args):
            launched.append("op")
            raise error
        monkeypatch.setattr(tecoops, name, op)
        return launched
    return put


NAMES = ["_linear", "_moe_layer", "_rotary_axes", "_rotary_axes_cache"]


@pytest.mark.parametrize("name", NAMES)
def test_launch_error_is_raised_once(name, stub):
    launched = stub(name, RuntimeError("x: TECOOPS_STATUS_INTERNAL_ERROR"))
    with pytest.raises(TecoopsError) as e:
        calls(tensors())[name]()
    assert e.value.status == _lib.INTERNAL_ERROR and launched == ["op"]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("error", [RuntimeError("no memory"), torch.OutOfMemoryError("no memory"),
                                   TypeError("something"), ValueError("something")])
def test_other_errors_stay_what_they_are(name, error, stub):
    launched = stub(name, error)
    with pytest.raises(type(error)) as e:
        calls(tensors())[name]()
    assert e.value is error and launched == ["op"]


@pytest.mark.parametrize("name", NAMES)
def test_no_tokens(name, stub):
    """An error without any work to do is still one."""
    t = tensors()
    for k in ("x", "out", "logits", "y", "q", "k", "v", "slots"):
        t[k] = t[k][:0]
    t["pos"] = t["pos"][:, :0]
    launched = stub(name, RuntimeError("something"))
    with pytest.raises(RuntimeError):
        calls(t)[name]()
    assert launched == ["op"]


@pytest.mark.parametrize("heads", [(H * D,), (H, D)])
def test_empty_batch_of_several_heads(heads, stub, monkeypatch):
    """No tokens, any number of heads: nothing to do (the checks alone, without the op)."""
    launched = stub("_rotary_axes", RuntimeError("not called"))
    t = tensors()
    q = torch.zeros(0, *heads, dtype=F16)
    monkeypatch.setattr(tecoops, "_rotary_axes", None)
    monkeypatch.setattr(tecoops, "_rotary_axes_cache", None)
    tecoops.rotary_embedding_axes(t["pos"][:, :0], q, q, D, [12, 10, 10])
    args = (t["slots"][:0], t["kc"], t["vc"], D, [12, 10, 10])
    tecoops.rotary_axes_reshape_and_cache(t["pos"][:, :0], q, q, q, *args)
    assert launched == []
    with pytest.raises(ValueError):  # one kv head of value, two of key
        tecoops.rotary_axes_reshape_and_cache(t["pos"][:, :0], q, q, torch.zeros(0, D, dtype=F16), *args)


def test_refused_arguments_keep_their_errors(stub):
    for name, key, bad in (("_linear", "x", torch.zeros(T, 63, dtype=F16)),
                           ("_linear", "w", torch.zeros(31, 64, dtype=F16)),
                           ("_moe_layer", "logits", torch.zeros(T, E + 1)),
                           ("_rotary_axes", "q", torch.zeros(T + 1, D, dtype=F16)),
                           ("_rotary_axes_cache", "slots", torch.zeros(T + 1, dtype=torch.int64))):
        t = tensors()
        t[key] = bad
        launched = stub(name, RuntimeError("refused"))
        with pytest.raises(ValueError):
            calls(t)[name]()
        assert set(launched) == {"op"}
    t = tensors()
    t["x"] = t["x"].float()
    for name in NAMES[:2]:
        stub(name, RuntimeError("refused"))
        with pytest.raises(TypeError):
            calls(t)[name]()


def test_arguments_of_other_types(monkeypatch):
    """What int(), bool() and float() take is passed on as such, so that the op does
    not refuse it."""
    import numpy as np
    seen = []
    for name in NAMES:
        monkeypatch.setattr(tecoops, name, lambda *a: seen.append(a))
    t = tensors()
    tecoops.linear(t["x"], t["w"], t["out"], gated=np.bool_(True))
    tecoops.moe_layer(t["x"], t["w_in"], t["w_out"], t["logits"], np.int64(2), t["y"], renormalize=1)
    for f, front in ((tecoops.rotary_embedding_axes, ("pos", "q", "k")),
                     (tecoops.rotary_axes_reshape_and_cache, ("pos", "q", "k", "v", "slots", "kc", "vc"))):
        f(*(t[n] for n in front), np.int64(D), np.array([12, 10, 10]), is_neox=np.bool_(False), base=10000,
          rot_dim=np.int32(64))
    types = {bool, int, float, str, list, type(None), torch.Tensor}
    assert all(type(a) in types for args in seen for a in args)
    assert seen[0][-1] is True and seen[1][4] == 2 and seen[1][6] is True
    assert all(type(n) is int for args in seen[2:] for a in args if type(a) is list for n in a)
    with pytest.raises(ValueError):
        tecoops.rotary_embedding_axes(t["pos"], t["q"], t["k"], D, ["a"])


def test_status_of_a_message():
    assert _lib.status_of("linear: TECOOPS_STATUS_NOT_SUPPORTED\nraised from here") == _lib.NOT_SUPPORTED
    assert _lib.status_of("tensors must be contiguous") is None


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("error", ["no memory", "x: TECOOPS_STATUS_INTERNAL_ERROR"])
def test_a_failed_call_keeps_no_tensors(name, error, stub, monkeypatch):
    """A caller that catches the error and lets go of its tensors gets their memory
    back, without waiting for a collection of cycles."""
    import gc
    import weakref
    t = tensors()
    held = [weakref.ref(v) for v in t.values()]
    call = calls(t)[name]
    stub(name, None)

    def op(*args):
        raise RuntimeError(error)
    monkeypatch.setattr(tecoops, name, op)
    gc.disable()
    try:
        try:
            call()
        except RuntimeError:
            pass
        del call, t
        assert all(ref() is None for ref in held)
    finally:
        gc.enable()
