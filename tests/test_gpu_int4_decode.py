"""An attention block with 4-bit weights and a 4-bit cache as a server runs it:
prefill of a ragged batch, then decode steps from a captured graph, each against the
same block in 64 bits over the cache that the kernels have written.

Bound: the outputs of the operators between (norm, qkv, norm with rotation,
attention, output product) are each rounded once to 16 bits, at most u = half a step
each, attention's weights (and in prefill its keys and values) to fp16, at most 2^-11
each; normalised random weights keep the gain of the ones behind near 1.  16 u is
asserted of each row, relative to its 2-norm.  The rows that a step stores in 4 bits
are the exact codes of its rounded key and value."""
import pytest
import torch

import tecoops
from int4_reference import DTYPES, HALF_STEP, attention, norm_rotary, pack, quantised, rand, weights

pytestmark = pytest.mark.gpu

HID, H, HKV, D, BS, NB, G = 512, 8, 2, 128, 16, 32, 64
QKV, EPS, BASE = (H + 2 * HKV) * D, 1e-6, 1e6


class Block:
    def __init__(self, dtype):
        self.dtype = dtype
        g = torch.Generator().manual_seed(7)
        self.host = {}
        for name, n, k in (("qkv", QKV, HID), ("o", HID, H * D)):
            codes = torch.randint(0, 16, (n, k), generator=g)
            scales = ((torch.rand(n, k // G, generator=g) + 0.5) * 0.22 * k ** -0.5).to(dtype)
            zeros = (torch.rand(n, k // G, generator=g) + 7).to(dtype)
            self.host[name] = (codes, scales, zeros)
        self.w = {k: (pack(c).cuda(), s.cuda(), z.cuda()) for k, (c, s, z) in self.host.items()}
        self.norm, self.qw, self.kw = (rand(n, dtype=dtype, scale=0.2, seed=i) + 1
                                       for i, n in enumerate((HID, D, D)))
        self.nd, self.qd, self.kd = self.norm.cuda(), self.qw.cuda(), self.kw.cuda()
        self.cache = [torch.zeros(NB, HKV, BS, D // 2, dtype=torch.uint8, device="cuda") for _ in range(2)] + \
            [torch.zeros(NB, HKV, BS, 2, dtype=dtype, device="cuda") for _ in range(2)]

    def buffers(self, T):
        return [torch.zeros(*s, dtype=self.dtype, device="cuda")
                for s in ((T, HID), (T, QKV), (T, H, D), (T, H, D), (T, HID))]

    def run(self, b, x, pos, slots, cu, lens, table, most_q, most_k):
        n, qkv, qc, o, out = b
        kc, vc, ks, vs = self.cache
        tecoops.rms_norm(x, self.nd, None, n, None, EPS)
        w, s, z = self.w["qkv"]
        tecoops.gemv_int4(w, s, n, qkv, zeros=z)
        q, k, v = qkv.split([H * D, HKV * D, HKV * D], 1)
        tecoops.qk_norm_rotary(pos, q, k, self.qd, self.kd, D, eps=EPS, base=BASE)
        tecoops.reshape_and_cache_int4(k.unflatten(1, (HKV, D)), v.unflatten(1, (HKV, D)), slots, kc, vc, ks, vs)
        qc.copy_(q.unflatten(1, (H, D)))
        tecoops.flash_attn_varlen_int4(qc, kc, vc, ks, vs, most_q, cu, most_k, lens, None, True, table, o)
        w, s, z = self.w["o"]
        tecoops.gemv_int4(w, s, o.flatten(1), out, zeros=z)

    def reference(self, x, pos, cu, lens, table):
        """Output in 64 bits, over the cache as it is."""
        f = x.double()
        f = f / torch.sqrt((f * f).mean(-1, keepdim=True) + EPS) * self.norm.double()
        qkv = f @ weights(*self.host["qkv"], G).t()
        a = pos.double()[:, None] * BASE ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
        q, _ = norm_rotary(qkv[:, :H * D].view(-1, H, D), self.qw, EPS, a.cos(), a.sin(), D, True)
        kc, vc, ks, vs = [t.cpu() for t in self.cache]
        o, _, _ = attention(q, kc, vc, ks, vs, cu, lens, table)
        return o.flatten(1) @ weights(*self.host["o"], G).t()


def close(got, ref, dtype):
    got = got.cpu().double()
    off = (got - ref).norm(dim=-1) / ref.norm(dim=-1)
    assert float(off.max()) < 16 * HALF_STEP[dtype], off.max()


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("lens", [[37, 1, 90], [5, 20, 16]])
def test_prefill_then_decode(dt, lens):
    dtype = DTYPES[dt]
    m = Block(dtype)
    table = torch.randperm(NB, generator=torch.Generator().manual_seed(1))[:3 * 8].view(3, 8).int()

    def slots_at(b, p):
        return int(table[b, p // BS]) * BS + p % BS

    def inputs(first, count, seed):
        """x, positions, slots and offsets of `count` tokens of each sequence."""
        T = sum(count)
        x = rand(T, HID, dtype=dtype, seed=seed)
        at = [(b, p) for b in range(3) for p in range(first[b], first[b] + count[b])]
        cu = [sum(count[:b]) for b in range(4)]
        return (x, torch.tensor([p for _, p in at]), torch.tensor([slots_at(b, p) for b, p in at]),
                torch.tensor(cu, dtype=torch.int32))

    x, pos, slots, cu = inputs([0, 0, 0], lens, 3)
    bufs = m.buffers(len(pos))
    m.run(bufs, x.cuda(), pos.cuda(), slots.cuda(), cu.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
          table.cuda(), max(lens), max(lens))
    close(bufs[4], m.reference(x, pos, cu.tolist(), lens, table), dtype)

    # decode: one graph, replayed with new inputs
    x, pos, slots, cu = [t.cuda() for t in inputs(lens, [1, 1, 1], 4)]
    used, td = torch.tensor([n + 1 for n in lens], dtype=torch.int32).cuda(), table.cuda()
    bufs = m.buffers(3)
    saved = [t.clone() for t in m.cache]
    m.run(bufs, x, pos, slots, cu, used, td, 1, 128)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.run(bufs, x, pos, slots, cu, used, td, 1, 128)
    for t, s in zip(m.cache, saved):
        t.copy_(s)
    for step in range(3):
        now = [n + step for n in lens]
        for dst, src in zip((x, pos, slots, cu), inputs(now, [1, 1, 1], 10 + step)):
            dst.copy_(src)
        used.copy_(torch.tensor([n + 1 for n in now], dtype=torch.int32))
        for b in bufs:
            b.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        # what was stored are the codes of the rounded rows
        k, v = (t.cpu().view(3, HKV, D) for t in bufs[1].split([H * D, HKV * D, HKV * D], 1)[1:])
        for rows, codes, pairs in ((k, m.cache[0], m.cache[2]), (v, m.cache[1], m.cache[3])):
            n, pair = quantised(rows)
            for b in range(3):
                s = slots_at(b, now[b])
                assert torch.equal(codes[s // BS, :, s % BS].cpu(), pack(n[b]))
                assert torch.equal(pairs[s // BS, :, s % BS].cpu(), pair[b])
        close(bufs[4], m.reference(x.cpu(), pos.cpu(), [0, 1, 2, 3], [n + 1 for n in now], table), dtype)
