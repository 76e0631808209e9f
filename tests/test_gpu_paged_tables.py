"""vqb_paged_tables against a plain allocator that walks requests and pages one by one."""
import numpy as np
import pytest
import torch

from vqlab_b200 import _lib, paged_tables

pytestmark = pytest.mark.gpu


def plain(context, new, table, ring, state, page, max_tokens, offset):
    """The step, one request and one page at a time (host lists)."""
    R, W = table.shape
    F = len(ring)
    ring, table, kv = ring.copy(), table.copy(), context.copy()
    head, tail, refused = int(state[0]), int(state[1]), 0
    for r in range(R):
        held = -(-context[r] // page)
        if new[r] < 0:
            for j in range(held):
                ring[tail % F] = table[r, j]
                tail += 1
            table[r] = -1
            kv[r] = 0
        else:
            table[r, held:] = -1
    asked, slots, pos, req, cu = 0, [], [], [], [0]
    avail = tail - head
    for r in range(R):
        n = max(int(new[r]), 0)
        if new[r] >= 0:
            held, pages = -(-context[r] // page), -(-(context[r] + n) // page)
            fits = pages <= W
            asked += pages - held if fits else 0
            ok = fits and (pages == held or asked <= avail)
            if ok:
                for j in range(held, pages):
                    table[r, j] = ring[head % F]
                    head += 1
                kv[r] = context[r] + n
            else:
                refused += 1
            for i in range(n):
                at = context[r] + i
                slots.append(table[r, at // page] * page + at % page if ok else -1)
                pos.append(offset + at)
                req.append(r)
        cu.append(len(slots))
    pad = max_tokens - len(slots)
    return dict(block_table=table, kv_lens=kv, cu_q=cu, slots=(slots + [-1] * max(pad, 0))[:max_tokens],
                positions=(pos + [0] * max(pad, 0))[:max_tokens], requests=(req + [-1] * max(pad, 0))[:max_tokens],
                free_pages=ring, state=[head, tail, refused, 0])


def make(R, W, page, ctx, new, free, seed, head=0):
    rng = np.random.default_rng(seed)
    context = np.asarray(ctx, np.int64)
    held = -(-context // page)
    pages = int(held.sum()) + free
    order = rng.permutation(pages)
    table = np.full((R, W), -1, np.int64)
    at = 0
    for r in range(R):
        table[r, :held[r]] = order[at:at + held[r]]
        at += held[r]
    F = max(pages, 1)
    ring = np.full(F, -1, np.int64)
    for i in range(free):
        ring[(head + i) % F] = order[at + i]
    return context, np.asarray(new, np.int64), table, ring, np.array([head, head + free, 0, 0], np.int64)


def check(case, page, max_tokens, offset=0, inplace=False):
    context, new, table, ring, state = case
    dev = [torch.from_numpy(np.ascontiguousarray(a)).to("cuda", torch.int32) for a in (context, new, table, ring)]
    st = torch.from_numpy(state).cuda()
    got = paged_tables(*dev, st, page_size=page, max_tokens=max_tokens, position_offset=offset, inplace=inplace)
    want = plain(context, new, table, ring, state, page, max_tokens, offset)
    for name in got._fields:
        assert np.array_equal(getattr(got, name).cpu().numpy(), np.asarray(want[name])), name
    if not inplace:  # the inputs are as they were
        for a, t in zip((context, new, table, ring), dev):
            assert np.array_equal(a, t.cpu().numpy())
        assert np.array_equal(st.cpu().numpy(), state)
    else:
        assert got.kv_lens.data_ptr() == dev[0].data_ptr() and got.state.data_ptr() == st.data_ptr()
    return got


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("R,page,most,seed", [(1, 1, 5, 0), (1, 16, 100, 1), (7, 16, 100, 2), (33, 3, 40, 3),
                                              (600, 32, 900, 4), (1025, 64, 300, 5)])
def test_random_steps(R, page, most, seed, inplace):
    rng = np.random.default_rng(seed)
    ctx = rng.integers(0, most + 1, R)
    new = np.where(rng.random(R) < 0.2, -1, rng.integers(0, 2 * page + 3, R))
    W = -(-(most + 2 * page + 3) // page)
    free = int((-(-(ctx + np.maximum(new, 0)) // page)).sum())
    case = make(R, W, page, ctx, new, free, seed, head=int(rng.integers(0, 10 ** 12)))
    check(case, page, int(np.maximum(new, 0).sum()) + 3, offset=int(rng.integers(0, 1000)), inplace=inplace)


def test_pages_of_finished_requests_serve_the_same_step():
    """No free page left: the new tokens live on what request 1 gives back, across the ring's end."""
    case = make(4, 8, 16, [16, 40, 0, 31], [1, -1, 20, 1], 0, 6, head=10 ** 9 + 5)
    got = check(case, 16, 22)
    assert got.state.tolist()[2] == 0
    check(case, 16, 22, inplace=True)


@pytest.mark.parametrize("inplace", [False, True])
def test_refused_requests_keep_what_they_hold(inplace):
    # too few pages: request 0 takes the only one, 1 and 2 are refused, 3 needs none
    case = make(4, 8, 16, [16, 32, 0, 10], [1, 1, 60, 2], 1, 7)
    got = check(case, 16, 70, inplace=inplace)
    assert got.state.tolist()[2] == 2
    # too narrow a row does not count against those after it
    case = make(3, 2, 16, [30, 5, 16], [3, 1, 16], 1, 8)
    got = check(case, 16, 25, inplace=inplace)
    assert got.state.tolist()[2] == 1


def test_lengths_of_zero_and_no_tokens():
    check(make(5, 4, 16, [0] * 5, [0] * 5, 3, 9), 16, 0)
    check(make(5, 4, 16, [0, 64, 0, 1, 16], [-1] * 5, 3, 10), 16, 4)
    check(make(2, 4, 16, [0, 0], [64, 0], 4, 11), 16, 64)


@pytest.mark.parametrize("page", [2**30, 2**31 - 1, 715827883])
def test_a_length_past_31_bits_is_refused(page):
    """The pages would fit the rows; the lengths no longer fit their type.  Requests up to 2^31 - 1 tokens are served."""
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    context, new = [2**31 - 10, 2**31 - 10, 5, 2**31 - 1], [100, 9, 1, 0]
    held = [-(-c // page) for c in context]
    table = [[4 * r + j if j < n else -1 for j in range(4)] for r, n in enumerate(held)]
    out = paged_tables(i32(context), i32(new), i32(table), i32([90, 91, 92, 93]), torch.tensor([0, 4, 0, 0], device="cuda"),
                       page_size=page, max_tokens=112)
    assert out.kv_lens.tolist() == [2**31 - 10, 2**31 - 1, 6, 2**31 - 1]
    assert out.state.tolist() == [0, 4, 1, 0]
    assert out.block_table.tolist() == table
    assert out.requests.tolist() == [0] * 100 + [1] * 9 + [2, -1, -1]
    assert out.slots[:100].tolist() == [-1] * 100


def test_more_tokens_than_places_is_safe():
    """Tokens past max_tokens have no place; everything else is as it would be."""
    check(make(3, 8, 16, [3, 0, 20], [30, 10, 7], 9, 12), 16, 20)


def test_steps_in_a_captured_graph():
    """Replays of one captured in-place step keep allocating."""
    page, R, W, pages = 4, 3, 8, 24
    lens = torch.zeros(R, dtype=torch.int32, device="cuda")
    new = torch.tensor([1, 2, 0], dtype=torch.int32, device="cuda")
    table = torch.full((R, W), -1, dtype=torch.int32, device="cuda")
    ring = torch.arange(pages, dtype=torch.int32, device="cuda")
    state = torch.tensor([0, pages, 0, 0], dtype=torch.int64, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = paged_tables(lens, new, table, ring, state, page_size=page, max_tokens=3, inplace=True)
    context = np.zeros(R, np.int64)
    t, f, st = np.full((R, W), -1, np.int64), np.arange(pages), np.array([0, pages, 0, 0])
    for _ in range(9):
        g.replay()
        want = plain(context, np.array([1, 2, 0]), t, f, st, page, 3, 0)
        for name in out._fields:
            assert np.array_equal(getattr(out, name).cpu().numpy(), np.asarray(want[name])), name
        context, t, f, st = want["kv_lens"], want["block_table"], want["free_pages"], np.array(want["state"])


def test_refusals():
    c, n, t, f, st = make(2, 4, 16, [3, 0], [1, 1], 4, 13)
    ok = [torch.from_numpy(a).to("cuda", torch.int32) for a in (c, n, t, f)]
    s = torch.from_numpy(st).cuda()
    with pytest.raises(ValueError):
        paged_tables(ok[0].long(), *ok[1:], s, page_size=16, max_tokens=2)
    with pytest.raises(ValueError):
        paged_tables(ok[0][:1], *ok[1:], s, page_size=16, max_tokens=2)
    with pytest.raises(ValueError):
        paged_tables(*ok, s, page_size=0, max_tokens=2)
    with pytest.raises(ValueError):
        paged_tables(*ok, s.int(), page_size=16, max_tokens=2)
    with pytest.raises(ValueError):
        paged_tables(ok[0], ok[1], ok[2].t(), ok[3], s, page_size=16, max_tokens=2)
    big = torch.zeros(8193, dtype=torch.int32, device="cuda")
    with pytest.raises(NotImplementedError):
        paged_tables(big, big, torch.zeros((8193, 1), dtype=torch.int32, device="cuda"), ok[3], s, page_size=16,
                     max_tokens=2)
    assert _lib.launch_count() >= 0
