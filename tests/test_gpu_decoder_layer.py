"""The operators of a decoder layer of a multimodal mixture-of-experts model run
together, as a server uses them: prefill of a ragged batch, then decode steps
from a captured graph, against the same layer in 64 bits.

Bound: each operator's output is rounded once to 16 bits (u, half a step) and
the errors add up along the layer; a row's distance from the reference, relative
to its 2-norm, is at most u for each of the operators between (norm, qkv,
rotary, attention: its probabilities and its output, output product, residual,
norm, gate and up, h, down and the sum) times the gain of the ones behind it,
which normalised random weights keep near 1.  16 u is asserted."""
import math

import pytest
import torch

import tecoops

pytestmark = pytest.mark.gpu

HID, H, HKV, D, BS, E, K, INTER = 512, 8, 2, 64, 16, 8, 2, 192
SEC, BASE, EPS = [12, 10, 10], 1e6, 1e-6
QKV = (H + 2 * HKV) * D


class Layer:
    def __init__(self, dt, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def w(*shape, scale):
            return (torch.randn(shape, generator=g, device="cuda") * scale).to(dt)

        self.dt, self.g = dt, g
        self.norm1, self.norm2 = (w(HID, scale=0.1) + 1 for _ in range(2))
        self.wqkv, self.bqkv = w(QKV, HID, scale=HID ** -0.5), w(QKV, scale=0.3)
        self.wo = w(HID, H * D, scale=(H * D) ** -0.5)
        self.router = w(E, HID, scale=4 * HID ** -0.5)
        self.w_in = w(E, 2 * INTER, HID, scale=HID ** -0.5)
        self.w_out = w(E, HID, INTER, scale=2 * INTER ** -0.5)

    def buffers(self, T):
        def e(*shape, dtype=self.dt):
            return torch.zeros(shape, dtype=dtype, device="cuda")
        return dict(n1=e(T, HID), qkv=e(T, QKV), o=e(T, H, D), r=e(T, HID), n2=e(T, HID),
                    logits=e(T, E), out=e(T, HID), ids=e(T, K, dtype=torch.int32))

    def run(self, b, x, pos, slots, kc, vc, cu, kv_lens, table, max_q, max_k):
        tecoops.rms_norm(x, self.norm1, None, b["n1"], None, EPS)
        tecoops.linear(b["n1"], self.wqkv, b["qkv"], bias=self.bqkv)
        q, k, v = b["qkv"].split([H * D, HKV * D, HKV * D], 1)
        tecoops.rotary_axes_reshape_and_cache(pos, q, k, v, slots, kc, vc, D, SEC,
                                              layout="interleaved", base=BASE)
        torch.ops.tecoops.flash_attn_varlen_func(q.unflatten(1, (H, D)).contiguous(), kc, vc, max_q,
                                                 cu, max_k, None, kv_lens, D ** -0.5, True, None,
                                                 table, False, b["o"])
        tecoops.linear(b["o"].flatten(1), self.wo, b["r"], residual=x)
        tecoops.rms_norm(b["r"], self.norm2, None, b["n2"], None, EPS)
        tecoops.linear(b["n2"], self.router, b["logits"])
        tecoops.moe_layer(b["n2"], self.w_in, self.w_out, b["logits"], K, b["out"], topk_ids=b["ids"])

    def ref(self, x, pos, ids, ks, vs, lens):
        """64 bits; ks / vs: each sequence's earlier keys and values (lists that
        grow); ids: the experts taken (a near tie may fall either way)."""
        def norm(t, w):
            return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + EPS) * w.double()
        x = x.double()
        qkv = norm(x, self.norm1) @ self.wqkv.double().t().contiguous() + self.bqkv.double()
        T = x.shape[0]
        half = D // 2
        axis = torch.tensor([i % 3 if i % 3 and i < 3 * SEC[i % 3] else 0 for i in range(half)],
                            device="cuda")
        ang = pos[axis].t().double() * BASE ** (-torch.arange(half, device="cuda").double() / half)
        c, s = ang.cos()[:, None], ang.sin()[:, None]

        def turn(t, heads):
            t = t.reshape(T, heads, D)
            a, b = t[..., :half], t[..., half:]
            return torch.cat([a * c - b * s, b * c + a * s], -1)
        q, k = turn(qkv[:, :H * D], H), turn(qkv[:, H * D:(H + HKV) * D], HKV)
        v = qkv[:, (H + HKV) * D:].reshape(T, HKV, D)
        o, at = torch.empty(T, H, D, dtype=torch.float64, device="cuda"), 0
        for i, n in enumerate(lens):
            ks[i] = torch.cat([ks[i], k[at:at + n]])
            vs[i] = torch.cat([vs[i], v[at:at + n]])
            m = ks[i].shape[0]
            hide = torch.arange(m, device="cuda")[None] > torch.arange(n, device="cuda")[:, None] + m - n
            for h in range(H):
                p = q[at:at + n, h] @ ks[i][:, h // 4].t().contiguous() * D ** -0.5
                o[at:at + n, h] = p.masked_fill(hide, -math.inf).softmax(-1) @ vs[i][:, h // 4].contiguous()
            at += n
        r = x + o.flatten(1) @ self.wo.double().t().contiguous()
        n2 = norm(r, self.norm2)
        logits = n2 @ self.router.double().t().contiguous()
        chosen = logits.gather(1, ids.long())
        weights = chosen.softmax(-1)
        out = torch.zeros_like(x)
        for t in range(T):
            for j in range(K):
                e = int(ids[t, j])
                y = self.w_in[e].double() @ n2[t]
                h = y[:INTER] * torch.sigmoid(y[:INTER]) * y[INTER:]
                out[t] += weights[t, j] * (self.w_out[e].double() @ h)
        return r, logits, out


def close(got, ref, dt, what):
    u = torch.finfo(dt).eps / 2
    err = (got.double() - ref).norm(dim=-1) / ref.norm(dim=-1)
    assert (err <= 16 * u).all(), (what, err.max().item() / u)


def check_routing(ids, logits, dt):
    """The chosen experts' logits are the largest up to what 16-bit errors of
    rows of this size can swap."""
    best = logits.sort(-1, descending=True).values[:, :K]
    slack = 32 * torch.finfo(dt).eps / 2 * logits.norm(dim=-1, keepdim=True)
    assert (logits.gather(1, ids.long()) >= best - slack).all()
    assert (ids[:, 0] != ids[:, 1]).all()


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_prefill_then_decode_graph(dt):
    layer = Layer(dt, 1)
    lens, nb = [70, 1, 33], 32
    B, T = len(lens), sum(lens)
    perm = torch.randperm(nb, generator=torch.Generator().manual_seed(1))
    table = perm[:B * 6].reshape(B, 6).int().cuda()
    kc, vc = (torch.zeros(nb, HKV, BS, D, dtype=dt, device="cuda") for _ in range(2))

    def slot(i, t):
        return int(table[i, t // BS]) * BS + t % BS

    x = torch.randn(T, HID, generator=layer.g, device="cuda").to(dt)
    pos = torch.randint(0, 5000, (3, T), generator=layer.g, device="cuda")
    slots = torch.tensor([slot(i, t) for i, n in enumerate(lens) for t in range(n)], device="cuda")
    cu = torch.tensor([0, 70, 71, 104], dtype=torch.int32, device="cuda")
    b = layer.buffers(T)
    layer.run(b, x, pos, slots, kc, vc, cu, torch.tensor(lens, dtype=torch.int32, device="cuda"),
              table, 70, 70)
    ks = [torch.zeros(0, HKV, D, dtype=torch.float64, device="cuda") for _ in lens]
    vs = [t.clone() for t in ks]
    r, logits, out = layer.ref(x, pos, b["ids"], ks, vs, lens)
    check_routing(b["ids"], logits, dt)
    close(b["r"], r, dt, "after attention")
    close(b["out"], out, dt, "experts")

    # decode, replayed from a graph with new inputs
    kv = torch.tensor(lens, dtype=torch.int32, device="cuda")
    x1, pos1 = x[:B].clone(), pos[:, :B].clone()
    slot1 = torch.zeros(B, dtype=torch.int64, device="cuda")
    cu1 = torch.arange(B + 1, dtype=torch.int32, device="cuda")
    b1 = layer.buffers(B)
    scratch = [t.clone() for t in (kc, vc)]  # the warm-up and capture steps' stores

    def step():
        layer.run(b1, x1, pos1, slot1, kc, vc, cu1, kv, table, 1, 96)

    slot1.fill_(-1)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    assert torch.equal(scratch[0], kc) and torch.equal(scratch[1], vc)
    for n in range(3):
        at = [m + n for m in lens]
        slot1.copy_(torch.tensor([slot(i, t) for i, t in enumerate(at)]))
        kv.copy_(torch.tensor([t + 1 for t in at], dtype=torch.int32))
        x1.copy_(torch.randn(B, HID, generator=layer.g, device="cuda"))
        pos1.copy_(torch.randint(0, 100000, (3, B), generator=layer.g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        replayed = {k: t.clone() for k, t in b1.items()}
        r, logits, out = layer.ref(x1, pos1, b1["ids"], ks, vs, [1] * B)
        check_routing(b1["ids"], logits, dt)
        close(b1["r"], r, dt, f"after attention, step {n}")
        close(b1["out"], out, dt, f"experts, step {n}")
        step()  # eagerly: the same bits
        torch.cuda.synchronize()
        assert all(torch.equal(replayed[k], t) for k, t in b1.items())
