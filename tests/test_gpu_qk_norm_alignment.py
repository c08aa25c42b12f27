"""The norm with the rotation and the store gives the bits of the two calls in turn
where only value, or only a cache, is off 16-byte addresses or strides (q and k alone
decide how the call in place is done)."""
import pytest
import torch

import tecoops
from int4_reference import DTYPES, rand

pytestmark = pytest.mark.gpu


def placed(t, off, width=None):
    """t's elements from `off` elements behind a 16-byte address on, its rows `width` apart."""
    width = t[0].numel() if width is None else width
    flat = torch.zeros(off + t.shape[0] * width + 8, dtype=t.dtype, device="cuda")
    rows = flat[off:off + t.shape[0] * width].view(t.shape[0], width)[:, :t[0].numel()]
    rows.copy_(t.reshape(t.shape[0], -1))
    return rows if t.dim() == 2 else rows.view(t.shape)


@pytest.mark.parametrize("what", ["value", "value stride", "key cache", "value cache", "all"])
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("D,rot", [(128, 128), (64, 64), (80, 32), (96, 96), (256, 128), (512, 512), (8, 8), (200, 64)])
def test_only_one_tensor_off(D, rot, dt, neox, what):
    dtype, T, H, Hkv, NB, bs = DTYPES[dt], 67, 4, 2, 9, 16
    q, k, v = (rand(T, h * D, dtype=dtype, scale=3.0, seed=i).cuda() for i, h in enumerate((H, Hkv, Hkv)))
    qw, kw = (rand(D, dtype=dtype, seed=5) + 1).cuda(), (rand(D, dtype=dtype, seed=6) + 1).cuda()
    pos = (torch.arange(T) * 977).cuda()
    slots = torch.randperm(NB * bs, generator=torch.Generator().manual_seed(1))[:T].cuda()
    one_q, one_k = q.clone(), k.clone()
    tecoops.qk_norm_rotary(pos, one_q, one_k, qw, kw, D, rot_dim=rot, is_neox=neox)
    empty = torch.full((NB, Hkv, bs, D), 7.0, dtype=dtype, device="cuda")
    kc1, vc1 = empty.clone(), empty.clone()
    tecoops.reshape_and_cache(one_k.view(T, Hkv, D), v.view(T, Hkv, D), slots, kc1, vc1)
    off = {n: int(what in (n, "all")) for n in ("value", "key cache", "value cache")}
    kc2, vc2 = placed(empty, off["key cache"]), placed(empty, off["value cache"])
    v2 = placed(v, off["value"], Hkv * D + (3 if what in ("value stride", "all") else 0))
    two_q, two_k = q.clone(), k.clone()
    tecoops.qk_norm_rotary_reshape_and_cache(pos, two_q, two_k, v2, qw, kw, slots, kc2, vc2, D, rot_dim=rot,
                                             is_neox=neox, write_key=True)
    for a, b in ((one_q, two_q), (one_k, two_k), (kc1, kc2), (vc1, vc2)):
        assert torch.equal(a, b)
