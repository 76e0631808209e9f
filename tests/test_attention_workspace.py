"""A caller's own workspace for the attention calls: its size, and the status that a call leaves in it."""
import pytest
import torch

from vqlab_b200 import _lib, attention_workspace, check_attention


def test_status_of_a_workspace():
    ws = attention_workspace(5, 3, 8, 2, 64, 16, max_q_len=2, max_kv_len=40, prefix_len=7, device="cpu")
    assert ws.dtype == torch.uint8 and ws.numel() >= 16
    ws.zero_()
    check_attention(ws)
    ws[4:8].view(torch.int32)[0] = _lib.VQB_TIMEOUT
    with pytest.raises(_lib.VQBError):
        check_attention(ws)
    for bad in (dict(head_dim=96), dict(page_size=24), dict(heads=7), dict(n_tokens=-1)):
        a = dict(n_tokens=5, requests=3, heads=8, kv_heads=2, head_dim=64, page_size=16, max_q_len=2, max_kv_len=40, device="cpu")
        a.update(bad)
        with pytest.raises(ValueError):
            attention_workspace(**a)


@pytest.mark.gpu
@pytest.mark.parametrize("q_lens,lens,prefix", [([1] * 4, [700, 3, 0, 90], 0), ([1], [30000], 0), ([1] * 60, [50] * 60, 4000),
                                                ([300, 20], [400, 20], 100), ([5] * 70, [300] * 70, 0)])
def test_calls_with_a_workspace_of_that_size(q_lens, lens, prefix):
    from test_gpu_prefix_attention import BF, Case
    for D in (64, 128):
        c = Case(q_lens, lens, prefix, 10, 2, D, 16, BF, seed=22)
        want = c.run()
        ws = attention_workspace(sum(q_lens), len(lens), 10, 2, D, 16, max_q_len=max(q_lens), max_kv_len=max(lens), prefix_len=prefix)
        ws.fill_(_lib.VQB_TIMEOUT)
        assert torch.equal(c.run(workspace=ws), want)
        check_attention(ws)
        with pytest.raises(ValueError):
            c.run(workspace=ws[:-1])
