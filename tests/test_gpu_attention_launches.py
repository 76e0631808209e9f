"""What the attention calls launch: one kernel for tables and rotary, the planned passes for attention, nothing when refused."""
import pytest
import torch

from test_gpu_prefix_attention import BF, Case
from vqlab_b200 import _lib, paged_tables, prefix_attention, rotary, rotary_frequencies

pytestmark = pytest.mark.gpu


def launches(call):
    before = _lib.launch_count()
    call()
    return _lib.launch_count() - before


def test_launches_of_each_call():
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    args = (i32([3, 0]), i32([1, 5]), torch.full((2, 4), -1, dtype=torch.int32, device="cuda"), i32([1, 2, 3]),
            torch.tensor([0, 3, 0, 0], device="cuda"))
    assert launches(lambda: paged_tables(*args, page_size=16, max_tokens=6)) == 1
    freq, _ = rotary_frequencies(64)
    x = torch.randn((3, 2, 64), device="cuda").bfloat16()
    assert launches(lambda: rotary(x, i32([0, 1, 2]), freq)) == 1
    assert launches(Case([1] * 4, [20, 3, 40, 0], 0, 8, 2, 64, 16, BF).run) == 1          # few rows over few keys: one pass
    assert launches(Case([2] * 4, [20, 3, 40, 2], 0, 8, 2, 64, 16, BF).run) == 2          # a mask: spoiled rows are looked for
    assert launches(Case([1], [40000], 0, 8, 2, 128, 16, BF).run) == 2                    # clusters of blocks and a join
    assert launches(Case([1] * 60, [20] * 60, 5000, 8, 2, 128, 16, BF).run) >= 2          # the prefix, then the requests' own keys


def test_a_refused_call_launches_nothing():
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    c = Case([1, 2], [20, 30], 10, 4, 2, 64, 16, BF)

    def refused(call, error=ValueError):
        with pytest.raises(error):
            call()
    freq, _ = rotary_frequencies(64)
    state = torch.tensor([0, 3, 0, 0], device="cuda")
    table = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    assert launches(lambda: refused(lambda: paged_tables(i32([3, 0]), i32([1, 5]), table, i32([1]), state, page_size=0, max_tokens=6))) == 0
    assert launches(lambda: refused(lambda: rotary(c.q[..., :32], i32([0, 1, 2]), freq))) == 0
    assert launches(lambda: refused(lambda: c.run(scale=0.0))) == 0
    assert launches(lambda: refused(lambda: c.run(max_kv_len=10 ** 6))) == 0
    assert launches(lambda: refused(lambda: c.run(workspace=torch.empty(8, dtype=torch.uint8, device="cuda")))) == 0
    kv = torch.zeros((9, 2, 24, 64), dtype=torch.bfloat16, device="cuda")
    assert launches(lambda: refused(lambda: prefix_attention(c.q, kv, kv, c.table, c.kv_lens, c.cu, max_q_len=2, max_kv_len=30), NotImplementedError)) == 0
