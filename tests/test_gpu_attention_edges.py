"""vqb_prefix_attention where few numbers decide: tiny weights beside a large one,
scores and values that are not finite, bounds below the lengths.

Tolerances are those of test_gpu_prefix_attention.py (derived there, before any run).
"""
import ctypes

import pytest
import torch

from test_gpu_prefix_attention import BF, FP, Case
from vqlab_b200 import _lib

pytestmark = pytest.mark.gpu


def sink(c, gap, place):
    """One key `gap` nats above all others, which score 0 alike: its values 0, theirs between 0.5 and 1.5.
    The others' weights are exp(-gap) of its own, and the whole result.  Returns the scale of such a call."""
    c.q.zero_()
    c.q[..., 0] = 4.0
    c.k.copy_(torch.where(torch.isnan(c.k), c.k, 0.0))
    c.v.copy_(torch.where(torch.isnan(c.v), c.v, 0.5 + c.v.float().abs().clamp(max=2.0) / 2).to(c.dtype))
    for r in range(len(c.lens)):
        pages, j = (c.prefix_pages, place) if c.prefix else (c.table[r], place % c.lens[r])
        p, o = int(pages[j // c.page]), j % c.page
        c.k[p, :, o, 0] = gap
        c.v[p, :, o] = 0.0
    return 0.25


# Weights from exp(-17) = 2^-24.5 of the row's largest on take one rounding of u, as the tolerance has it.
@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("gap", [10.0, 13.0, 14.25, 16.0, 17.0])
@pytest.mark.parametrize("R,q_len,length,prefix,H,KH,D,page", [
    (2, 1, 8192, 0, 8, 2, 64, 32), (20, 1, 5000, 0, 8, 8, 128, 16), (20, 3, 3000, 0, 15, 3, 64, 16),
    (70, 5, 700, 0, 15, 3, 128, 16), (1, 300, 8200, 0, 8, 2, 64, 128), (1, 300, 8200, 0, 8, 2, 128, 64),
    (75, 16, 1500, 0, 24, 3, 128, 64), (30, 1, 40, 8192, 10, 2, 128, 64), (30, 1, 40, 8192, 10, 2, 64, 64)])
def test_small_weights_beside_a_large_one(R, q_len, length, prefix, H, KH, D, page, gap, dtype):
    c = Case([q_len] * R, [length] * R, prefix, H, KH, D, page, dtype, seed=R + D)
    c.check(scale=sink(c, gap, 3))


@pytest.mark.parametrize("q_len,prefix", [(3, 60), (3, 0), (40, 0), (40, 130), (300, 60)])
def test_values_that_are_not_finite_leave_the_log_sum_exp(q_len, prefix):
    """Scores alone make the log-sum-exp: no value changes it, seen or not, one of a row's or all of them."""
    for D, page, dtype in ((128, 16, BF), (64, 64, FP)):
        c = Case([q_len] * 3, [q_len + 200, q_len + 60, q_len], prefix, 4, 2, D, page, dtype, seed=16)
        want = c.run(return_lse=True)[1]
        assert torch.isfinite(want).all()
        v0 = c.v.clone()
        for bad in (float("nan"), float("inf"), -float("inf")):
            for r, j in ((0, 0), (0, q_len + 199), (1, q_len + 59), (2, q_len - 1)):
                c.v.copy_(v0)
                c.v[int(c.table[r, j // page]), :, j % page] = bad
                assert torch.equal(c.run(return_lse=True)[1], want), (bad, r, j)
            c.v.fill_(bad)
            assert torch.equal(c.run(return_lse=True)[1], want), bad


@pytest.mark.parametrize("q_lens,lens,prefix,H,KH,D", [
    ([2] * 60, [17] * 60, 0, 16, 8, 64), ([3] * 30, [40] * 30, 700, 15, 3, 128), ([70] * 4, [90] * 4, 0, 4, 2, 128), ([2, 300], [5, 300], 0, 4, 2, 64)])
def test_notes_of_spoiled_rows_in_one_workspace(q_lens, lens, prefix, H, KH, D):
    """Whatever a workspace held, however often a captured call replays: a masked value that is not finite leaves no trace."""
    c = Case(q_lens, lens, prefix, H, KH, D, 16, BF, seed=20)
    want = c.run()
    clean = c.v.clone()
    spoiled = c.v.clone()
    cu = c.cu.tolist()
    seen = torch.ones(want.shape[0], dtype=torch.bool, device="cuda")
    for r, n in enumerate(lens):  # each request's last key: its last query alone sees it
        spoiled[int(c.table[r, (n - 1) // 16]), :, (n - 1) % 16] = float("inf")
        seen[cu[r + 1] - 1] = False
    ws = torch.full((1 << 26,), 255, dtype=torch.uint8, device="cuda")

    def right(got, bad):
        return torch.equal(got[seen], want[seen]) if not bad else bool(torch.isfinite(got[seen]).all()) and bool(
            ((got - want).abs() <= 2.0 ** -6 * (want.abs() + 1))[seen].all()) and not bool(torch.isfinite(got[~seen]).any())
    for fill in (255, 0, 1):
        ws.fill_(fill)
        for bad in (True, False, True, True):
            c.v.copy_(spoiled if bad else clean)
            assert right(c.run(workspace=ws), bad)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = c.run(workspace=ws)
    for bad in (True, False, False, True, True, False):
        c.v.copy_(spoiled if bad else clean)
        g.replay()
        torch.cuda.synchronize()
        assert right(out, bad)
        assert ws[:20].view(torch.int32).tolist()[1:] == [0, 0, 0, 0]  # no status, no count, no note left


def test_rows_that_see_only_scores_of_minus_infinity():
    """exp(-inf) / exp(-inf): such a row is NaN and its log-sum-exp -inf; 0 is for a row that sees no key at all."""
    nan = float("nan")
    for q_lens, lens, prefix, D, page, dtype in (
            ([1, 1, 1], [1, 300, 0], 0, 64, 16, BF), ([1] * 40, [5] * 39 + [0], 0, 128, 16, FP), ([1, 1], [9000, 0], 0, 128, 64, BF),
            ([40, 3], [40, 2], 0, 128, 16, FP), ([300, 2], [300, 0], 0, 64, 64, BF), ([1] * 30, [0] * 15 + [3] * 15, 700, 128, 16, BF),
            ([200, 1], [1000, 0], 0, 128, 128, BF), ([3] * 60, [0] * 30 + [40] * 30, 2000, 64, 16, FP)):
        c = Case(q_lens, lens, prefix, 4, 2, D, page, dtype, seed=17)
        c.q[..., 5] = c.q[..., 5].abs() + 0.5
        c.k[..., 5] = -float("inf")
        got, lse = c.run(return_lse=True)
        assert bool((lse == -float("inf")).all())
        cu = c.cu.tolist()
        for r, length in enumerate(lens):
            for i in range(q_lens[r]):
                sees = prefix + max(length - q_lens[r] + i + 1, 0) > 0
                row = got[cu[r] + i]
                assert bool((torch.isnan(row) if sees else row == 0).all()), (q_lens, lens, prefix, r, i)
    # one such key among others has weight 0, and a row that it masks is untouched
    c = Case([40], [40], 0, 4, 2, 64, 16, BF, seed=18)
    c.q[..., 5] = c.q[..., 5].abs() + 0.5
    want = c.run()
    c.k[int(c.table[0, 0]), :, 0, 5] = -float("inf")
    got = c.run()
    assert bool(torch.isnan(got[0]).all()) and bool(torch.isfinite(got[1:]).all()) and not torch.equal(got[1:], want[1:])


@pytest.mark.parametrize("q_len,H,KH,D,prefix,R", [(5, 6, 2, 64, 0, 3), (5, 6, 2, 128, 300, 3), (40, 8, 2, 64, 50, 3), (40, 8, 2, 128, 0, 3),
                                                   (300, 4, 1, 128, 0, 2), (12, 4, 2, 64, 0, 80), (20, 8, 2, 128, 700, 80)])
def test_bounds_below_the_lengths(q_len, H, KH, D, prefix, R):
    """Keys past max_kv_len are left out, and no other: a query still sees its own place and what lies before it.
    Queries past max_q_len are left out; those before keep their results."""
    c = Case([q_len] * R, [500 + r for r in range(R)], prefix, H, KH, D, 16, BF, seed=19)
    u, G = 2.0 ** -8, H // KH
    for bound, queries in ((520, q_len), (501, q_len), (500 - q_len // 2, q_len), (500 - q_len, q_len), (64, q_len), (0, q_len), (520, q_len // 2 + 1)):
        got = c.run(max_kv_len=bound, max_q_len=queries).double()
        assert torch.equal(got.nan_to_num(7.0), c.run(max_kv_len=bound, max_q_len=queries).double().nan_to_num(7.0)) or queries < q_len
        for r in (0, R - 1):
            length = c.lens[r]
            for h in range(KH):
                pages = c.table[r, :-(-length // 16)]
                k, v = (torch.cat([c.rows(x, c.prefix_pages, prefix, h), c.rows(x, pages, length, h)[:bound]]) for x in (c.k, c.v))
                x = c.q[r * q_len:r * q_len + queries, h * G:(h + 1) * G].double().reshape(-1, D)
                s = x @ k.T * D ** -0.5
                last = prefix + length - q_len + torch.arange(queries, device="cuda").repeat_interleave(G)
                s = s.masked_fill(torch.arange(k.shape[0], device="cuda")[None] > last[:, None], -torch.inf)
                w = torch.softmax(s, -1) if k.shape[0] else s
                o, A = w @ v, w @ v.abs()
                ds = ((x.abs() @ k.abs().T) * D ** 0.5 * 2.0 ** -23 + s.abs().nan_to_num(0, 0, 0) * 2.0 ** -22).amax(-1, keepdim=True) if k.shape[0] else 0.0
                mine = got[r * q_len:r * q_len + queries, h * G:(h + 1) * G].reshape(-1, D)
                assert bool(((mine - o).abs() <= u * o.abs() + (u + 2 * ds + 2.0 ** -16) * A + 1e-38).all()), (bound, queries, r, h)


@pytest.mark.parametrize("q_len", [1, 4, 40])
def test_no_block_table(q_len):
    """A C caller whose requests hold nothing of their own passes no table (max_kv_len 0), whatever its width."""
    c = Case([q_len] * 9, [0] * 9, 333, 10, 2, 128, 16, BF, seed=21)
    want = c.run(max_kv_len=0)
    N = c.q.shape[0]
    k, v = c.k.stride(), c.v.stride()
    for width in (0, 7, 4096):
        d = _lib.AttentionDesc(n_requests=9, n_tokens=N, heads=10, kv_heads=2, head_dim=128, page_size=16, num_pages=c.k.shape[0],
                               table_width=width, max_q_len=q_len, max_kv_len=0, prefix_len=333, causal=1, scale=128 ** -0.5,
                               q_token_stride=1280, q_head_stride=128, out_token_stride=1280, out_head_stride=128,
                               kc_page_stride=k[0], kc_head_stride=k[1], kc_token_stride=k[2], vc_page_stride=v[0],
                               vc_head_stride=v[1], vc_token_stride=v[2])
        L, out = _lib.lib(), torch.zeros_like(c.q)
        ws = torch.empty(L.vqb_prefix_attention_workspace_size(ctypes.byref(d)), dtype=torch.uint8, device="cuda")
        args = [c.q, c.k, c.v, None, c.kv_lens, c.cu, c.prefix_pages, out, None, ws]
        ptr = [ctypes.c_void_p(t.data_ptr() if t is not None else None) for t in args]
        st = L.vqb_prefix_attention(ctypes.byref(d), _lib.VQB_BF16, *ptr, ws.numel(),
                                    ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert st == _lib.VQB_OK
        assert torch.equal(out, want)
