"""A step in which some requests get no pages: which they are, and that nothing of the others changes.

Tolerance, before any run: a request alone and in its batch may be split differently; each result is within
u (|o| + A) + 2^-16 A of the exact one (u = 2^-8, A <= max |v|; scores are the same sums), so the two differ by twice that.
"""
import pytest
import torch

from vqlab_b200 import PagedKVCache, paged_tables, prefix_attention, rotary_append, rotary_frequencies

pytestmark = pytest.mark.gpu
H, KH, D, PAGE = 8, 2, 64, 16


def i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("inplace", [False, True])
def test_which_requests_were_refused(inplace):
    # request 1 needs two pages of one, 2 then lacks its page, 3 needs none, 4 has no new tokens, 5 has finished with nothing held
    table = torch.full((6, 4), -1, dtype=torch.int32, device="cuda")
    table[0, 0], table[3, 0], table[4, 0] = 0, 1, 2
    t = paged_tables(i32([10, 0, 0, 4, 16, 0]), i32([3, 20, 1, 2, 0, -1]), table, i32([3, -1, -1, -1]),
                     torch.tensor([0, 1, 0, 0], device="cuda"), page_size=PAGE, max_tokens=30, inplace=inplace)
    assert t.refused_requests().tolist() == [False, True, True, False, False, False]
    assert int(t.state[2]) == 2
    gone = torch.isin(t.requests, i32([1, 2]))
    assert torch.equal(t.slots < 0, gone | (t.requests < 0))
    none = paged_tables(i32([10]), i32([0]), table[:1], i32([3]), torch.tensor([0, 1, 0, 0], device="cuda"), page_size=PAGE, max_tokens=0)
    assert none.refused_requests().tolist() == [False]


@pytest.mark.parametrize("more", [[1, 40, 1], [3, 200, 9]])
def test_attention_around_a_refused_request(more):
    g = torch.Generator(device="cuda").manual_seed(3)
    cache = PagedKVCache(1, 8, PAGE, KH, D, 3, 256)
    freq, amp = rotary_frequencies(D)
    kc, vc = cache.k[0], cache.v[0]

    def step(new):
        t = cache.step(i32(new), sum(new) + 1)
        x = torch.randn((sum(new), H + 2 * KH, D), device="cuda", generator=g).to(torch.bfloat16)
        q = rotary_append(x[:, :H], x[:, H:H + KH], x[:, H + KH:], t.positions, freq, kc, vc, t.slots, amplitude=amp)
        out = prefix_attention(q, kc, vc, t.block_table, t.kv_lens, t.cu_q, max_q_len=max(new), max_kv_len=256)
        return t, q, out

    step([20, 33, 20])  # 2 + 3 + 2 of 8 pages
    row, pages = cache.block_table[1].clone(), cache.block_table[1, :3].long()
    held = (kc[pages].clone(), vc[pages].clone())
    t, q, out = step(more)
    assert t.refused_requests().tolist() == [False, True, False] and cache.refused() == 1
    assert torch.equal(cache.block_table[1], row) and cache.kv_lens.tolist() == [20 + more[0], 33, 20 + more[2]]
    assert torch.equal(kc[pages], held[0]) and torch.equal(vc[pages], held[1])
    cu = t.cu_q.tolist()
    lim = 2 * (2.0 ** -8 * 2 + 2.0 ** -16) * float(vc.float().abs().max())
    for r in (0, 2):
        rows = slice(cu[r], cu[r + 1])
        alone = prefix_attention(q[rows].contiguous(), kc, vc, t.block_table[r:r + 1], t.kv_lens[r:r + 1], i32([0, more[r]]),
                                 max_q_len=more[r], max_kv_len=256)
        assert bool(((out[rows].double() - alone.double()).abs() <= lim).all())
        assert bool((t.slots[rows] >= 0).all())
    assert bool((t.slots[cu[1]:cu[2]] == -1).all())
    cache.step(i32([-1, 0, -1]), 1)  # pages become free, and the request is served
    t, _, out = step([0, 40, 0])
    assert not t.refused_requests().any() and cache.kv_lens.tolist() == [0, 73, 0] and bool(torch.isfinite(out).all())
