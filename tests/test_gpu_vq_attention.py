"""VQAttention over PagedKVCache: a shared prompt, requests joining and leaving,
prompts and single tokens, against the same projections with rotary and softmax
attention in 64 bits.

Tolerance, before any run: the 64-bit reference takes the module's own q, k and v
(bf16) and rounds where the module must: rotated q and k once (u = 2^-8), so each
score moves by at most 2 u scale sum |q k|, which moves the attention output by at
most 2 (2 u scale sum |q k|) A, A = sum p |v|; the weights' and the output's
rounding add u (A + |o|).  The output projection is linear: its result moves by at
most |W| times that, taken from the projection of unit vectors.
"""
import numpy as np
import pytest
import torch

from oracle import oracle as orc
from vqlab_b200 import PagedKVCache, VQAttention, VQLinear, rotary_frequencies

pytestmark = pytest.mark.gpu
U = 2.0 ** -8


def linear(rng, out, inn, scale):
    K, D, bits = 256, 2, 8
    codes = rng.integers(0, K, (1, out, inn // D)).astype(np.uint16)
    cb = (rng.standard_normal((K, D)) * scale).astype(np.float16)
    sc = rng.uniform(0.5, 1.5, (out, inn // 64)).astype(np.float16)
    t = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    return VQLinear(t(orc.pack(codes, bits)[0].view(np.int32)), t(cb), t(sc), group_size=64, pack_bits=bits, in_features=inn)


class Layer:
    def __init__(self, hidden, heads, kv_heads, dim, rot, interleaved, seed):
        rng = np.random.default_rng(seed)
        self.H, self.KH, self.D, self.rot, self.inter = heads, kv_heads, dim, rot, interleaved
        freq, amp = rotary_frequencies(rot, 10000.0, "ramp", 4.0, original_length=512)
        s = 1.0 / hidden ** 0.5
        self.mod = VQAttention(linear(rng, heads * dim, hidden, s), linear(rng, kv_heads * dim, hidden, s),
                               linear(rng, kv_heads * dim, hidden, s), linear(rng, hidden, heads * dim, s), heads,
                               kv_heads, dim, freq, amp, interleaved)
        eye = torch.eye(heads * dim, dtype=torch.bfloat16, device="cuda")
        self.o_abs = self.mod.o_proj(eye).double().abs()  # [heads * dim, hidden]

    def rotate(self, x, pos):
        """x [N, heads, D] at positions, float64, rounded once to bf16."""
        m = self.mod
        turns = np.array([[((int(p) * int(f)) % (1 << 64)) / 2.0 ** 64 for f in m.freq.tolist()] for p in pos])
        c = torch.from_numpy(np.cos(2 * np.pi * turns)).cuda()[:, None] * m.amplitude
        s = torch.from_numpy(np.sin(2 * np.pi * turns)).cuda()[:, None] * m.amplitude
        y = x.double().clone()
        i0, i1 = ((slice(0, self.rot, 2), slice(1, self.rot, 2)) if self.inter else
                  (slice(0, self.rot // 2), slice(self.rot // 2, self.rot)))
        a, b = x[..., i0].double(), x[..., i1].double()
        y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
        return y.to(torch.bfloat16)

    def reference(self, x, pos, past):
        """(output [N, hidden], bound) of one request's new tokens; past: its (and the prefix's) rotated k and v,
        to which the new ones are added."""
        m, G = self.mod, self.H // self.KH
        n = x.shape[0]
        q = self.rotate(m.q_proj(x).view(n, self.H, self.D), pos)
        past[0] = torch.cat([past[0], self.rotate(m.k_proj(x).view(n, self.KH, self.D), pos)])
        past[1] = torch.cat([past[1], m.v_proj(x).view(n, self.KH, self.D)])
        k, v = past[0].double(), past[1].double()
        T = k.shape[0]
        out, lim = torch.empty((n, self.H, self.D), device="cuda", dtype=torch.double), None
        lim = torch.empty_like(out)
        last = T - n + torch.arange(n, device="cuda")
        seen = torch.arange(T, device="cuda")[None] <= last[:, None]
        for h in range(self.H):
            kh, vh = k[:, h // G], v[:, h // G]
            s = q[:, h].double() @ kh.T * self.D ** -0.5
            ds = (2 * U * (q[:, h].double().abs() @ kh.abs().T) * self.D ** -0.5).masked_fill(~seen, 0).amax(-1, keepdim=True)
            p = torch.softmax(s.masked_fill(~seen, -torch.inf), -1)
            out[:, h] = p @ vh
            A = p @ vh.abs()
            lim[:, h] = 2 * torch.expm1(2 * ds) / 2 * A + U * (A + out[:, h].abs()) + 2.0 ** -16 * A
        y = m.o_proj(out.to(torch.bfloat16).view(n, -1)).double()
        return y, (lim.view(n, -1) @ self.o_abs) + U * y.abs() + U * (out.abs().view(n, -1) @ self.o_abs)


@pytest.mark.parametrize("heads,kv_heads,dim,rot,interleaved", [(8, 2, 64, 64, False), (5, 1, 128, 64, True)])
def test_batch_life(heads, kv_heads, dim, rot, interleaved):
    hidden, page, R, layers = 512, 16, 4, 2
    L = [Layer(hidden, heads, kv_heads, dim, rot, interleaved, 7 + i) for i in range(layers)]
    cache = PagedKVCache(layers, 64, page, kv_heads, dim, R, 512)
    g = torch.Generator(device="cuda").manual_seed(1)
    empty = lambda: [torch.empty((0, kv_heads, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2)]  # noqa: E731
    past = {(r, i): empty() for r in range(R) for i in range(layers)}
    lens = [0] * R

    def step(new):
        """One step of all layers for the requests' new token counts (-1: finished), checked layer by layer."""
        n = [max(v, 0) for v in new]
        tables = cache.step(torch.tensor(new, dtype=torch.int32, device="cuda"), sum(n) + 2)
        assert cache.refused() == 0
        for r in range(R):
            if new[r] < 0:
                lens[r] = 0
                for i in range(layers):
                    past[r, i] = [t[:cache.prefix_len] for t in shared[i]] if cache.prefix_len else empty()
            else:
                lens[r] += new[r]
        assert tables.kv_lens.tolist() == lens
        for i, layer in enumerate(L):
            x = torch.randn((sum(n), hidden), device="cuda", generator=g).to(torch.bfloat16)
            got = layer.mod(x, cache, i, tables, max(n), max(lens)).double()
            at = 0
            for r in range(R):
                if n[r] == 0:
                    continue
                pos = cache.prefix_len + np.arange(lens[r] - n[r], lens[r])
                want, lim = layer.reference(x[at:at + n[r]], pos, past[r, i])
                err = (got[at:at + n[r]] - want).abs()
                assert bool((err <= lim).all()), (i, r, float((err / lim).max()))
                at += n[r]

    shared = None
    step([70, 0, 0, 0])            # the prompt that all will share
    step([1, 0, 0, 0])
    shared = [[t.clone() for t in past[0, i]] for i in range(layers)]
    cache.share(0)
    assert cache.prefix_len == 71
    lens[0] = 0
    for r in range(R):
        for i in range(layers):
            past[r, i] = [t.clone() for t in shared[i]]
    step([33, 1, 0, 5])            # prompts of three requests behind it
    step([1, 1, 0, 1])
    step([1, -1, 40, 1])           # one leaves, another joins
    step([1, 2, 1, 1])
    for _ in range(3):
        step([1, 1, 1, 1])
    step([-1, -1, -1, -1])
    used = -(-71 // page)
    assert int(cache.state[1] - cache.state[0]) == 64 - used  # every page but the prefix's is free again
    assert sorted(cache.free_pages[[(int(cache.state[0]) + i) % 64 for i in range(64 - used)]].tolist()
                  + cache.prefix_pages.tolist()) == list(range(64))


def test_share_refusals():
    cache = PagedKVCache(1, 8, 16, 1, 64, 2, 64)
    with pytest.raises(ValueError):
        cache.share(0)
    cache.step(torch.tensor([5, 3], dtype=torch.int32, device="cuda"), 8)
    with pytest.raises(ValueError):
        cache.share(0)
    cache.step(torch.tensor([0, -1], dtype=torch.int32, device="cuda"), 8)
    cache.share(0)
    assert cache.prefix_len == 5 and cache.kv_lens.tolist() == [0, 0]
    with pytest.raises(ValueError):
        cache.share(0)
