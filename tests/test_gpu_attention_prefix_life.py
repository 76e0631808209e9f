"""A shared prefix that is given back and replaced: no page is lost, and the next prefix is read."""
import pytest
import torch

from vqlab_b200 import PagedKVCache, prefix_attention, rotary_append, rotary_frequencies

pytestmark = pytest.mark.gpu
H, KH, D, PAGE, PAGES = 8, 2, 64, 16, 12


def test_prefixes_one_after_another():
    """Tolerance, before any run: keys and values are compared bit for bit; the result with one of the exact softmax
    within u (|o| + A) + 2^-16 A, u = 2^-8, and twice the scores' error, D 2^-23 of sum |q k| (under 2^-12 here)."""
    cache = PagedKVCache(1, PAGES, PAGE, KH, D, 2, 96)
    freq, amp = rotary_frequencies(D)
    kc, vc = cache.k[0], cache.v[0]
    g = torch.Generator(device="cuda").manual_seed(4)

    def step(new):
        t = cache.step(torch.tensor(new, dtype=torch.int32, device="cuda"), max(sum(max(n, 0) for n in new), 1))
        n = sum(max(v, 0) for v in new)
        x = torch.randn((n, H + 2 * KH, D), device="cuda", generator=g).to(torch.bfloat16)
        if n == 0:
            return x, None
        q = rotary_append(x[:, :H], x[:, H:H + KH], x[:, H + KH:], t.positions, freq, kc, vc, t.slots, amplitude=amp)
        return q, prefix_attention(q, kc, vc, t.block_table, t.kv_lens, t.cu_q, max_q_len=max(new), max_kv_len=96,
                                   prefix_pages=cache.prefix_pages, prefix_len=cache.prefix_len)

    for length in (40, 17, 90, 64):  # 90 tokens and their followers need pages of the prefixes before
        step([length, 0])
        cache.share(0)
        with pytest.raises(ValueError):
            cache.share(0)
        q, out = step([5, 30])
        assert cache.refused() == 0
        flat = lambda c, pages, n: c[pages.long()].transpose(1, 2).reshape(-1, KH, D)[:n].double()  # noqa: E731
        for h in range(H):
            k, v = (torch.cat([flat(c, cache.prefix_pages, length), flat(c, cache.block_table[1, :2], 30)])[:, h // 4] for c in (kc, vc))
            p = torch.softmax(k @ q[-1, h].double() * D ** -0.5, 0)
            o, A = p @ v, p @ v.abs()
            assert bool(((out[-1, h].double() - o).abs() <= 2.0 ** -8 * (o.abs() + A) + 2.0 ** -11 * A).all())
        with pytest.raises(ValueError):
            cache.unshare()  # requests hold tokens behind it
        step([-1, -1])
        cache.unshare()
        assert cache.prefix_len == 0 and cache.prefix_pages is None
        start, end = cache.state[:2].tolist()
        assert end - start == PAGES
        assert sorted(cache.free_pages[[(start + i) % PAGES for i in range(PAGES)]].tolist()) == list(range(PAGES))
        with pytest.raises(ValueError):
            cache.unshare()
