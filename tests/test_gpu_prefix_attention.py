"""vqb_prefix_attention against softmax attention in 64 bits.

Tolerance, before any run.  With A = sum p |v| / sum p of the exact weights, u
the half unit of the type (2^-8 bf16, 2^-11 fp16):
  * the result is rounded once: u |o| (and 2^-25 among fp16 subnormals);
  * the weights may take one rounding to the type before they meet the values: u A;
  * a score is a sum of D products in fp32: its error is at most
    ds = D 2^-23 scale sum |q k| + 2^-22 |s|, which moves o by at most 2 ds A;
  * exponential, sums and joins: 2^-16 A.
The log-sum-exp is off by at most ds + 2^-16 + 2^-22 |lse|.
"""
import numpy as np
import pytest
import torch

from vqlab_b200 import prefix_attention

pytestmark = pytest.mark.gpu
HALF_UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16)}  # 2^-8, 2^-11


class Case:
    def __init__(self, q_lens, kv_lens, prefix, H, KH, D, page, dtype, seed=0, layout="head", spare=3, magnitude=1.0):
        rng = np.random.default_rng(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.q_lens, self.lens, self.prefix = list(q_lens), list(kv_lens), prefix
        self.H, self.KH, self.D, self.page, self.dtype = H, KH, D, page, dtype
        held = [-(-n // page) for n in kv_lens]
        shared = -(-prefix // page)
        pages = sum(held) + shared + spare
        order = rng.permutation(pages)
        W = max(held + [1]) + 1
        table = np.full((len(held), W), -1, np.int64)
        at = shared
        for r, n in enumerate(held):
            table[r, :n] = order[at:at + n]
            at += n
        self.prefix_pages = torch.from_numpy(order[:shared].copy()).to("cuda", torch.int32)
        self.table = torch.from_numpy(table).to("cuda", torch.int32)
        rnd = lambda *s: (torch.randn(s, device="cuda", generator=g) * magnitude).to(dtype)  # noqa: E731
        self.q = rnd(sum(q_lens), H, D)
        if layout == "head":  # [pages, heads, page, D]
            self.k, self.v = rnd(pages, KH, page, D), rnd(pages, KH, page, D)
        else:                 # [pages, page, 2, heads, D]: one pool of both, token-major
            kv = rnd(pages, page, 2, KH, D)
            self.k, self.v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
        # what no request holds is NaN: it must not be used
        used = torch.zeros((pages, page), dtype=torch.bool, device="cuda")
        for pg, n in [(self.prefix_pages, prefix)] + [(self.table[r, :held[r]], self.lens[r]) for r in range(len(held))]:
            for i, p in enumerate(pg.tolist()):
                used[p, :max(min(page, n - i * page), 0)] = True
        dead = ~used[:, None, :, None].expand(pages, KH, page, D)
        self.k.masked_fill_(dead, float("nan"))
        self.v.masked_fill_(dead, float("nan"))
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        self.cu = i32(np.concatenate([[0], np.cumsum(self.q_lens)]).tolist())
        self.kv_lens = i32(self.lens)

    def rows(self, cache, pages, n, h):
        return cache[pages.long(), h].double().reshape(-1, self.D)[:n]

    def run(self, **kw):
        a = dict(max_q_len=max(self.q_lens + [0]), max_kv_len=max(self.lens + [0]), prefix_len=self.prefix,
                 prefix_pages=self.prefix_pages if self.prefix else None)
        a.update(kw)
        q = a.pop("q", self.q)
        return prefix_attention(q, self.k, self.v, self.table, self.kv_lens, self.cu, **a)

    def check(self, causal=True, scale=None, **kw):
        got, lse = self.run(causal=causal, scale=scale, return_lse=True, **kw)
        assert got.shape == self.q.shape and got.dtype == self.dtype
        scale = self.D ** -0.5 if scale is None else scale
        u, G = HALF_UNIT[self.dtype], self.H // self.KH
        cu = self.cu.tolist()
        worst = 0.0
        for r, length in enumerate(self.lens):
            a, b = cu[r], cu[r + 1]
            if a == b:
                continue
            for h in range(self.KH):
                own = self.table[r, :-(-length // self.page)]
                k = torch.cat([self.rows(self.k, self.prefix_pages, self.prefix, h), self.rows(self.k, own, length, h)])
                v = torch.cat([self.rows(self.v, self.prefix_pages, self.prefix, h), self.rows(self.v, own, length, h)])
                x = self.q[a:b, h * G:(h + 1) * G].double().reshape(-1, self.D)
                s = x @ k.T * scale
                ds = (x.abs() @ k.abs().T * scale * self.D * 2.0 ** -23 + s.abs() * 2.0 ** -22)
                ds = ds.amax(-1, keepdim=True) if k.shape[0] else s.new_zeros((x.shape[0], 1))
                if causal:
                    last = self.prefix + length - (b - a) + torch.arange(b - a, device="cuda").repeat_interleave(G)
                    # a query placed before the request's first token still sees the whole prefix
                    last = last.clamp(min=self.prefix - 1)
                    s = s.masked_fill(torch.arange(k.shape[0], device="cuda")[None] > last[:, None], -torch.inf)
                L = torch.logsumexp(s, -1, keepdim=True) if k.shape[0] else s.new_full((x.shape[0], 1), -torch.inf)
                w = torch.exp(s - torch.where(torch.isinf(L), 0.0, L))
                o, A = w @ v, w @ v.abs()
                lim = u * o.abs() + (u + 2 * ds + 2.0 ** -16) * A + (2.0 ** -25 if self.dtype == torch.float16 else 1e-38)
                mine = got[a:b, h * G:(h + 1) * G].double().reshape(-1, self.D)
                err = (mine - o).abs()
                assert torch.isfinite(mine).all(), (r, h)
                worst = max(worst, float((err / lim).max()))
                assert bool((err <= lim).all()), (r, h, worst)
                ml, L, ds = lse[a:b, h * G:(h + 1) * G].double().reshape(-1), L[:, 0], ds[:, 0]
                inf = torch.isinf(L)
                assert torch.equal(torch.isinf(ml) & (ml < 0), inf)
                assert bool(((ml - L).abs()[~inf] <= (ds + 2.0 ** -16 + 2.0 ** -22 * L.abs())[~inf]).all())
        return got

    def reference(self):
        """(result, bound) [N, heads, D] in 64 bits of a causal call at the default scale."""
        u, G, cu = HALF_UNIT[self.dtype], self.H // self.KH, self.cu.tolist()
        out = torch.zeros(self.q.shape, dtype=torch.double, device="cuda")
        lim = torch.zeros_like(out)
        for r, length in enumerate(self.lens):
            n = cu[r + 1] - cu[r]
            for h in range(self.KH):
                own = self.table[r, :-(-length // self.page)]
                k = torch.cat([self.rows(self.k, self.prefix_pages, self.prefix, h), self.rows(self.k, own, length, h)])
                v = torch.cat([self.rows(self.v, self.prefix_pages, self.prefix, h), self.rows(self.v, own, length, h)])
                x = self.q[cu[r]:cu[r + 1], h * G:(h + 1) * G].double().reshape(-1, self.D)
                s = x @ k.T * self.D ** -0.5
                ds = ((x.abs() @ k.abs().T) * self.D ** 0.5 * 2.0 ** -23 + s.abs() * 2.0 ** -22).amax(-1, keepdim=True)
                last = self.prefix + length - n + torch.arange(n, device="cuda").repeat_interleave(G)
                w = torch.softmax(s.masked_fill(torch.arange(k.shape[0], device="cuda")[None] > last[:, None], -torch.inf), -1)
                o, A = w @ v, w @ v.abs()
                out[cu[r]:cu[r + 1], h * G:(h + 1) * G] = o.view(n, G, self.D)
                lim[cu[r]:cu[r + 1], h * G:(h + 1) * G] = (u * o.abs() + (u + 2 * ds + 2.0 ** -16) * A + 2.0 ** -25).view(n, G, self.D)
        return out, lim


BF, FP = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,KH", [(40, 8), (4, 4), (8, 1), (16, 1), (3, 1), (24, 1)])
def test_decode_heads(H, KH, D, dtype):
    Case([1] * 5, [1, 17, 64, 333, 130], 0, H, KH, D, 16, dtype, seed=H + D).check()


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("prefix", [0, 1, 127, 128, 129, 1000])
def test_pages_and_prefixes(page, prefix):
    Case([1, 1, 1, 1], [1, page, page + 1, 500], prefix, 8, 2, 128, page, BF, seed=page + prefix).check()


@pytest.mark.parametrize("layout", ["head", "token"])
@pytest.mark.parametrize("q_lens,kv_lens,prefix,H,KH,D", [
    ([1, 7, 130, 0, 33], [90, 7, 300, 0, 64], 0, 10, 2, 128),
    ([1, 7, 130, 0, 33], [90, 7, 300, 11, 64], 333, 10, 2, 64),
    ([257], [257], 0, 8, 2, 128), ([64, 65, 63], [64, 65, 63], 129, 4, 4, 64),
    ([300], [1300], 0, 5, 1, 128), ([1], [1], 0, 1, 1, 128), ([16] * 9, [16] * 9, 700, 16, 2, 128),
    ([2] * 40, [30] * 40, 2000, 15, 3, 64), ([700, 1, 700], [1000, 700, 700], 64, 4, 1, 128)])
def test_ragged_queries(q_lens, kv_lens, prefix, H, KH, D, layout):
    for dtype in (BF, FP):
        Case(q_lens, kv_lens, prefix, H, KH, D, 16, dtype, seed=sum(kv_lens), layout=layout).check()


def test_not_causal():
    Case([5, 40, 1], [70, 40, 0], 100, 6, 2, 128, 32, BF, seed=1).check(causal=False)
    Case([300], [40], 0, 6, 2, 64, 32, FP, seed=2).check(causal=False)
    Case([1] * 3, [0, 5, 200], 0, 6, 2, 64, 32, FP, seed=3).check(causal=False)


@pytest.mark.parametrize("q_lens,kv_lens,prefix", [
    ([1, 1], [0, 0], 0), ([1, 1], [0, 5], 0), ([4, 4], [2, 0], 0), ([4, 4], [2, 0], 50), ([200, 3], [100, 0], 0),
    ([200, 3], [100, 0], 130), ([0, 0], [3, 4], 10)])
def test_empty_rows(q_lens, kv_lens, prefix):
    """Requests that hold nothing, and more queries than tokens: rows that see nothing are 0."""
    for D, dtype in ((128, BF), (64, FP)):
        got = Case(q_lens, kv_lens, prefix, 10, 2, D, 16, dtype, seed=3).check()
        if prefix == 0 and sum(q_lens):
            assert bool((got[:max(q_lens[0] - kv_lens[0], 0)] == 0).all())


@pytest.mark.parametrize("R,prefix,context", [(64, 3000, 40), (150, 700, 100), (3, 20000, 10), (33, 2049, 1)])
def test_shared_prefix_batches(R, prefix, context):
    rng = np.random.default_rng(R)
    Case([1] * R, rng.integers(1, context + 1, R).tolist(), prefix, 10, 2, 128, 64, BF, seed=R).check()
    Case([2] * R, rng.integers(2, context + 2, R).tolist(), prefix, 8, 2, 64, 16, FP, seed=R).check()


@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("prefix", [0, 1, 15, 17, 31, 33, 47, 1000])
def test_ends_inside_a_stage(prefix, page):
    """Lengths of keys around the 16 and 32 of a stage, the prefix's end and the request's own."""
    for length in (0, 1, 15, 16, 17, 31, 32, 33, 49, 500):
        Case([1], [length], prefix, 8, 2, 64, page, FP, seed=prefix + length).check()
        Case([min(length, 3)], [length], prefix, 8, 2, 128, page, BF, seed=prefix + length).check()


@pytest.mark.parametrize("R,KH,length", [(16, 8, 2000), (13, 8, 2000), (74, 8, 300), (74, 8, 450), (150, 4, 300), (40, 8, 2000)])
def test_small_heads_in_one_round_and_in_several(R, KH, length):
    rng = np.random.default_rng(R)
    Case([1] * R, rng.integers(1, length, R, endpoint=True).tolist(), 0, 2 * KH, KH, 64, 32, BF, seed=R).check()


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("R,H,KH,q_len,length,prefix,page", [
    (64, 40, 8, 5, 200, 0, 16), (90, 10, 2, 4, 90, 0, 64), (150, 20, 4, 6, 40, 333, 32), (64, 17, 1, 1, 500, 0, 16), (200, 4, 4, 32, 60, 0, 16),
    (40, 24, 8, 7, 64, 1000, 16)])
def test_between_16_and_32_rows(R, H, KH, q_len, length, prefix, page, D, dtype):
    """A request's rows in two tiles of 16, the second one full, ragged or empty."""
    rng = np.random.default_rng(R + q_len)
    lens = rng.integers(0, length, R, endpoint=True)
    q_lens = np.minimum(rng.integers(0, q_len, R, endpoint=True), lens)
    q_lens[0], lens[0] = q_len, length
    c = Case(q_lens.tolist(), lens.tolist(), prefix, H, KH, D, page, dtype, seed=R)
    first = c.check()
    for _ in range(5):
        assert torch.equal(first, c.run())


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("R,H,KH,q_len,length,prefix,page", [
    (60, 24, 3, 16, 600, 0, 16), (40, 20, 4, 25, 300, 200, 64), (75, 4, 2, 64, 129, 0, 32), (160, 35, 1, 3, 1000, 0, 128), (20, 16, 8, 33, 2000, 0, 16)])
def test_one_tile_of_rows_each(R, H, KH, q_len, length, prefix, page, causal, dtype):
    """More (request, head)s than SMs, each with up to 128 rows: none, a few, a whole tile; keys from none to many tiles."""
    rng = np.random.default_rng(R + q_len)
    lens = rng.integers(0, length, R, endpoint=True)
    q_lens = np.minimum(rng.integers(0, q_len, R, endpoint=True), lens)
    q_lens[0], lens[0] = q_len, length
    c = Case(q_lens.tolist(), lens.tolist(), prefix, H, KH, 128, page, dtype, seed=R)
    first = c.check(causal=causal)
    for _ in range(5):
        assert torch.equal(first, c.run(causal=causal))


def test_long_context_splits():
    """One request over tens of thousands of tokens (split and joined), ragged beside short ones."""
    Case([1], [40001], 0, 8, 2, 128, 64, BF, seed=1).check()
    Case([1, 1, 1], [30011, 3, 0], 0, 8, 2, 64, 32, FP, seed=2).check()
    Case([20, 1], [9000, 8000], 5000, 8, 2, 128, 128, BF, seed=3).check()


@pytest.mark.parametrize("q_len", [1, 40])
def test_growing_scores(q_len):
    """Scores that rise and fall by hundreds over the keys: the running maximum moves, early sums vanish."""
    for up in (True, False):
        c = Case([q_len] * 2, [900, 640], 300, 4, 2, 64, 16, BF, seed=5)
        ramp = torch.linspace(-6, 6, c.k.shape[0], device="cuda")
        order = torch.argsort(torch.cat([c.prefix_pages, c.table[c.table >= 0]]).long())
        ramp = ramp if up else ramp.flip(0)
        full = torch.zeros_like(ramp)
        full[:order.numel()] = ramp[:order.numel()][order]
        c.k.mul_(full[:, None, None, None].to(c.dtype))
        c.q.copy_(c.q.abs() + 1)
        c.check(scale=0.6)


def test_large_and_small_scales():
    Case([1, 3], [200, 300], 50, 4, 2, 128, 16, BF, seed=6, magnitude=8.0).check(scale=1.0)
    Case([1, 300], [200, 300], 50, 4, 2, 128, 16, FP, seed=7, magnitude=6.0).check(scale=2.0)
    Case([1, 30], [200, 300], 50, 4, 2, 128, 16, FP, seed=8).check(scale=1e-6)


def test_padding_rows_and_strides():
    """Rows past the last query are not written; q and out are slices of wider tensors."""
    c = Case([1, 5, 40], [33, 50, 40], 70, 8, 2, 128, 16, BF, seed=9)
    want = c.check()
    n = c.q.shape[0]
    wide = torch.randn((n + 6, 12, 128), device="cuda").to(BF)
    wide[:n, 2:10] = c.q
    out = torch.full((n + 6, 10, 128), 7.0, device="cuda", dtype=BF)
    got = c.run(q=wide[:, 2:10], out=out[:, 1:9])
    assert got.data_ptr() == out[:, 1:9].data_ptr()
    assert torch.equal(out[:n, 1:9], want)
    assert bool((out[n:] == 7).all()) and bool((out[:, 0] == 7).all()) and bool((out[:, 9] == 7).all())


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("R,q_len,length,page", [(74, 5, 2200, 128), (90, 9, 700, 16), (160, 5, 390, 64), (40, 70, 1500, 256)])
def test_few_rows_over_many_keys_each(R, q_len, length, page, D, dtype):
    """More blocks than SMs, each with little work a key tile: copies of keys and values land late and out of order."""
    rng = np.random.default_rng(R)
    lens = rng.integers(length // 2, length, R, endpoint=True).tolist()
    c = Case([q_len] * R, lens, 0, 16, 4, D, page, dtype, seed=R)
    first = c.check()
    for _ in range(20):
        assert torch.equal(first, c.run())


def test_same_result_every_time():
    for q_lens, kv in (([1] * 30, [777] * 30), ([100, 300], [200, 300])):
        c = Case(q_lens, kv, 1500, 10, 2, 128, 64, BF, seed=10)
        first = c.run()
        for _ in range(3):
            assert torch.equal(c.run(), first)


def test_loose_bounds_and_other_streams():
    """max_q_len / max_kv_len only bound the lengths; a side stream; a captured graph with new lengths."""
    c = Case([1] * 6, [5, 100, 300, 0, 16, 64], 200, 8, 2, 64, 16, FP, seed=11)
    want = c.run()
    room = c.table.shape[1] * c.page
    got = c.run(max_q_len=2, max_kv_len=room)
    assert bool(((got.double() - want.double()).abs() <= 2.0 ** -9 * (want.double().abs() + 1)).all())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = c.run()
    s.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = c.run(max_kv_len=room)
    g.replay()
    torch.cuda.synchronize()
    first = out.clone()
    c.kv_lens.copy_(torch.tensor([5, 90, 300, 0, 9, 64]))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, c.run(max_kv_len=room)) and not torch.equal(out, first)


@pytest.mark.parametrize("q_lens,kv,prefix", [([1] * 40, [60] * 40, 3000), ([300, 20], [300, 40], 200), ([1] * 3, [9000] * 3, 0)])
def test_captured_graphs(q_lens, kv, prefix):
    c = Case(q_lens, kv, prefix, 10, 2, 128, 64, BF, seed=13)
    want = c.run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = c.run()
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("q_len", [1, 3, 40])
def test_nan_and_infinity_reach_the_rows_that_see_them(q_len):
    """NaN or infinity in a key or a value makes the rows that see it what the formula says and leaves the others."""
    for D, page, seed in ((128, 16, 14), (64, 64, 15)):
        c = Case([q_len] * 3, [200, 130, 90], 60, 4, 2, D, page, BF, seed=seed)
        want, lim = c.reference()
        k0, v0 = c.k.clone(), c.v.clone()
        for r, j in ((0, 3), (0, 127), (0, 163), (0, 199), (1, 95), (1, 129), (2, 70), (2, 89)):
            p, o = int(c.table[r, j // page]), j % page
            first = c.lens[r] - q_len  # place of the request's first query
            sees = torch.zeros(want.shape[:2], dtype=torch.bool, device="cuda")
            sees[r * q_len + max(j - first, 0):(r + 1) * q_len, 2:] = True  # key/value head 1
            for bad in (float("nan"), float("inf"), -float("inf")):
                c.k.copy_(k0)
                c.v.copy_(v0)
                c.v[p, 1, o, 5] = bad
                got = c.run().double()
                ok = (got - want).abs() <= lim
                assert bool(ok[~sees].all()), ("v", r, j, bad)
                assert bool(ok[..., :5][sees].all()) and bool(ok[..., 6:][sees].all()), ("v", r, j, bad)
                assert bool((torch.isnan(got[..., 5][sees]) if bad != bad else got[..., 5][sees] == bad).all()), ("v", r, j, bad)
                c.v.copy_(v0)
                c.k[p, 1, o, 5] = bad
                got = c.run().double()
                assert bool(((got - want).abs() <= lim)[~sees].all()), ("k", r, j, bad)
                x = got[sees]
                if bad != bad:
                    assert bool(torch.isnan(x).all()), ("k", r, j)
                else:  # q * inf: inf, and the row is NaN, or -inf, and the key's weight is 0
                    up = (c.q[..., 5].double() * bad)[sees] > 0
                    assert bool(torch.isnan(x[up]).all()) and bool(torch.isfinite(x[~up]).all()), ("k", r, j, bad)
        c.k.copy_(k0)
        c.v.fill_(float("nan"))
        assert bool(torch.isnan(c.run()).all())


@pytest.mark.parametrize("q_lens,kv,prefix", [([1, 1], [100, 60], 40), ([70, 3], [100, 60], 200)])
def test_offsets_past_32_bits(q_lens, kv, prefix):
    """A pool of over 2^32 bytes and 2^31 elements, the pages in use at its end."""
    c = Case(q_lens, kv, prefix, 4, 2, 128, 64, FP, seed=15)
    want = c.run()
    n, far = c.k.shape[0], 140000
    big = [torch.empty((far, 2, 64, 128), dtype=FP, device="cuda") for _ in range(2)]
    assert big[0].numel() > 2 ** 31
    for b, x in zip(big, (c.k, c.v)):
        b[far - n:] = x
    c.k, c.v = big
    c.table = torch.where(c.table >= 0, c.table + (far - n), -1).to(torch.int32)
    c.prefix_pages = (c.prefix_pages + (far - n)).to(torch.int32)
    assert torch.equal(c.run(), want)


def test_pages_outside_the_pool_read_as_zeros():
    c = Case([1, 40], [60, 60], 40, 4, 2, 64, 16, FP, seed=12)
    bad, good = c.table.clone(), c.table.clone()
    bad[0, 1], bad[1, 2] = -5, 10 ** 9
    zero = next(i for i in range(c.k.shape[0]) if i not in c.table.tolist()[0] + c.table.tolist()[1] + c.prefix_pages.tolist())
    c.k[zero], c.v[zero] = 0, 0
    good[0, 1], good[1, 2] = zero, zero
    c.table = bad
    a = c.run()
    c.table = good
    assert torch.equal(a, c.run())


def test_refusals():
    c = Case([1, 2], [20, 30], 10, 4, 2, 64, 16, FP)
    c.run()
    assert prefix_attention(c.q[:0], c.k, c.v, c.table, c.kv_lens, c.cu, max_q_len=0, max_kv_len=30).shape == (0, 4, 64)
    for bad in (dict(max_kv_len=10 ** 6), dict(max_q_len=-1), dict(prefix_len=17), dict(scale=0.0), dict(scale=-1.0),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(prefix_pages=None),
                dict(workspace=torch.empty(8, dtype=torch.uint8, device="cuda")), dict(out=c.q[:1])):
        with pytest.raises(ValueError):
            c.run(**bad)
    with pytest.raises(ValueError):
        prefix_attention(c.q[:, :3], c.k, c.v, c.table, c.kv_lens, c.cu, max_q_len=2, max_kv_len=30)
    with pytest.raises(ValueError):
        prefix_attention(c.q, c.k.bfloat16(), c.v, c.table, c.kv_lens, c.cu, max_q_len=2, max_kv_len=30)
    with pytest.raises(ValueError):
        prefix_attention(c.q, c.k, c.v, c.table, c.kv_lens, c.cu[:2], max_q_len=2, max_kv_len=30)
    off = torch.empty(c.q.numel() + 8, dtype=FP, device="cuda")[1:1 + c.q.numel()].view(c.q.shape)
    with pytest.raises(ValueError):
        c.run(q=off)
    with pytest.raises(NotImplementedError):
        x = torch.zeros((3, 4, 32), dtype=FP, device="cuda")
        kv = torch.zeros((9, 2, 16, 32), dtype=FP, device="cuda")
        prefix_attention(x, kv, kv, c.table, c.kv_lens, c.cu, max_q_len=2, max_kv_len=30)
    with pytest.raises(NotImplementedError):
        kv = torch.zeros((9, 2, 24, 64), dtype=FP, device="cuda")
        prefix_attention(c.q, kv, kv, c.table, c.kv_lens, c.cu, max_q_len=2, max_kv_len=30)
