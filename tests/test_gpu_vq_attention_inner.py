"""VQAttention step by step, each part against 64 bits on the very numbers that the module gave it, so
that no error of an earlier part has to be allowed for in a later one.

Tolerances, before any run; u = 2^-8 (bf16):
  * rotated q, and k in the cache: one rounding and 2^-20 (|a| + |b|) amplitude of the pair; v in the cache: equal;
  * attention, from the rotated q and the cache's k and v: u |o| + (u + 2 ds + 2^-16) A, A = sum p |v|,
    ds = D 2^-23 scale sum |q k| + 2^-22 |s|, as for the call alone;
  * the layer's result: the output projection of that attention, bit for bit.
Each bound has to refuse a reference with a mistake in it: nothing attended to, the prefix left out, no
causal mask, keys in another order, heads in another order, positions off by one.
"""
import numpy as np
import pytest
import torch

from test_gpu_vq_attention import U, Layer
from vqlab_b200 import PagedKVCache, attention

pytestmark = pytest.mark.gpu


def rotated(layer, x, pos):
    """(rotated x in float64, |a| + |b| of each element's pair times the amplitude)"""
    m, rot = layer.mod, layer.rot
    turns = np.array([[((int(p) * int(f)) % (1 << 64)) / 2.0 ** 64 for f in m.freq.tolist()] for p in pos])
    c = torch.from_numpy(np.cos(2 * np.pi * turns)).cuda()[:, None] * m.amplitude
    s = torch.from_numpy(np.sin(2 * np.pi * turns)).cuda()[:, None] * m.amplitude
    i0, i1 = ((slice(0, rot, 2), slice(1, rot, 2)) if layer.inter else (slice(0, rot // 2), slice(rot // 2, rot)))
    y, size = x.double().clone(), torch.zeros_like(x, dtype=torch.double)
    a, b = x[..., i0].double(), x[..., i1].double()
    y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
    size[..., i0] = size[..., i1] = (a.abs() + b.abs()) * m.amplitude
    return y, size


def attended(q, k, v, seen, D):
    """(softmax attention in float64 [n, H, D], bound); q [n, H, D], k and v [T, H, D], seen [n, T]."""
    s = torch.einsum("nhd,thd->nht", q, k) * D ** -0.5
    ds = (torch.einsum("nhd,thd->nht", q.abs(), k.abs()) * D ** 0.5 * 2.0 ** -23 + s.abs() * 2.0 ** -22)
    ds = ds.masked_fill(~seen[:, None], 0).amax(-1, keepdim=True)
    p = torch.softmax(s.masked_fill(~seen[:, None], -torch.inf), -1)
    o, A = torch.einsum("nht,thd->nhd", p, v), torch.einsum("nht,thd->nhd", p, v.abs())
    return o, U * o.abs() + (U + 2 * ds + 2.0 ** -16) * A + 1e-38


@pytest.mark.parametrize("heads,kv_heads,dim,rot,interleaved", [(8, 2, 64, 64, False), (5, 1, 128, 64, True)])
def test_each_part_of_the_layer(heads, kv_heads, dim, rot, interleaved, monkeypatch):
    hidden, page, R, G = 512, 16, 3, heads // kv_heads
    layer = Layer(hidden, heads, kv_heads, dim, rot, interleaved, 11)
    cache = PagedKVCache(1, 48, page, kv_heads, dim, R, 512)
    g = torch.Generator(device="cuda").manual_seed(2)
    call, inner = attention.prefix_attention, {}

    def recorded(q, *a, **kw):
        inner["q"] = q.clone()
        inner["o"] = call(q, *a, **kw)
        return inner["o"]
    monkeypatch.setattr(attention, "prefix_attention", recorded)
    lens = [0] * R
    refused = {}

    def wrong(name, got, o, lim):
        """A reference with a mistake: some element has to be off by more than the bound allows."""
        refused[name] = refused.get(name, 0) + 1
        assert not bool(((got - o).abs() <= lim).all()), name

    def step(new):
        n = [max(v, 0) for v in new]
        tables = cache.step(torch.tensor(new, dtype=torch.int32, device="cuda"), max(sum(n), 1))
        for r in range(R):
            lens[r] = 0 if new[r] < 0 else lens[r] + n[r]
        x = torch.randn((sum(n), hidden), device="cuda", generator=g).to(torch.bfloat16)
        y = layer.mod(x, cache, 0, tables, max(n), max(lens))
        q, o = inner["q"].double(), inner["o"]
        assert torch.equal(y, layer.mod.o_proj(o.view(sum(n), -1)))
        # of all tokens together, as the module projects them (fewer rows may take another kernel)
        projected = [p(x).view(sum(n), -1, dim) for p in (layer.mod.q_proj, layer.mod.k_proj, layer.mod.v_proj)]
        at = 0
        for r in range(R):
            if n[r] == 0:
                continue
            rows = slice(at, at + n[r])
            at += n[r]
            pre = cache.prefix_len
            pages = cache.block_table[r, :-(-lens[r] // page)]
            flat = lambda c, p, m: c[p.long()].transpose(1, 2).reshape(-1, kv_heads, dim)[:m].double()  # noqa: E731
            k, v = (flat(c[0], pages, lens[r]) for c in (cache.k, cache.v))
            pos = pre + np.arange(lens[r] - n[r], lens[r])
            plain_q, new_k, new_v = (t[rows] for t in projected)
            for name, got, plain in (("q", q[rows], plain_q), ("k", k[-n[r]:], new_k)):
                want, size = rotated(layer, plain, pos)
                assert bool(((got - want).abs() <= U * want.abs() + 2.0 ** -20 * size + 1e-38).all()), (name, r)
                off, size = rotated(layer, plain, pos + 1)
                wrong("position of " + name, got, off, U * off.abs() + 2.0 ** -20 * size + 1e-38)
            assert torch.equal(v[-n[r]:], new_v.double())
            if pre:
                k, v = (torch.cat([flat(c[0], cache.prefix_pages, pre), own]) for c, own in ((cache.k, k), (cache.v, v)))
            T = k.shape[0]
            k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
            seen = torch.arange(T, device="cuda")[None] <= (T - n[r] + torch.arange(n[r], device="cuda"))[:, None]
            got = o[rows].double()
            want, lim = attended(q[rows], k, v, seen, dim)
            assert bool(((got - want).abs() <= lim).all()), (r, float(((got - want).abs() / lim).max()))
            wrong("nothing", got, torch.zeros_like(want), lim)
            if pre:
                wrong("no prefix", got, *attended(q[rows], k[pre:], v[pre:], seen[:, pre:], dim))
            if n[r] > 1:
                wrong("no causal mask", got, *attended(q[rows], k, v, torch.ones_like(seen), dim))
            if T > 1:
                wrong("keys in another order", got, *attended(q[rows], k.roll(1, 0), v, seen, dim))
            wrong("heads in another order", got, *attended(q[rows].flip(1), k, v, seen, dim))

    step([70, 0, 0])
    step([1, 0, 0])
    cache.share(0)
    lens[0] = 0
    step([33, 1, 5])
    step([1, 1, 1])
    step([1, -1, 40])
    for _ in range(3):
        step([1, 2, 1])
    assert len(refused) == 7 and min(refused.values()) >= 3
