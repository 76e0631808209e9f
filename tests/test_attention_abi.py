"""Host-side checks of the paged-cache calls: each case is refused before any CUDA call."""
import ctypes

import pytest
import torch

from vqlab_b200 import _lib, paged_tables, prefix_attention, rotary

P = 0x10000  # stands for a device address; never read


def call(fn, d, kinds):
    return getattr(_lib.lib(), fn)(ctypes.byref(d) if d is not None else None, *kinds)


def paged(**kw):
    d = dict(n_requests=4, table_width=8, page_size=16, ring_size=64, max_tokens=8, position_offset=0)
    d.update(kw)
    return _lib.PagedDesc(**d)


@pytest.mark.parametrize("kw,status", [
    (dict(n_requests=-1), _lib.VQB_BAD_SHAPE), (dict(table_width=0), _lib.VQB_BAD_SHAPE),
    (dict(page_size=0), _lib.VQB_BAD_SHAPE), (dict(ring_size=0), _lib.VQB_BAD_SHAPE),
    (dict(max_tokens=-1), _lib.VQB_BAD_SHAPE), (dict(n_requests=8193), _lib.VQB_UNSUPPORTED_GEOMETRY)])
def test_paged_tables_refuses(kw, status):
    assert call("vqb_paged_tables", paged(**kw), [P] * 14) == status


def test_paged_tables_null_pointers():
    assert call("vqb_paged_tables", None, [P] * 14) == _lib.VQB_NULL_POINTER
    for i in range(13):
        args = [P] * 14
        args[i] = None
        assert call("vqb_paged_tables", paged(), args) == _lib.VQB_NULL_POINTER, i


def rot(**kw):
    d = dict(n_tokens=3, heads=4, kv_heads=2, head_dim=64, rotary_dim=64, page_size=16, num_pages=4, amplitude=1.0,
             q_token_stride=256, q_head_stride=64, k_token_stride=128, k_head_stride=64, v_token_stride=128,
             v_head_stride=64, out_token_stride=256, out_head_stride=64, kc_page_stride=2048, kc_head_stride=1024,
             kc_token_stride=64, vc_page_stride=2048, vc_head_stride=1024, vc_token_stride=64)
    d.update(kw)
    return _lib.RotaryDesc(**d)


@pytest.mark.parametrize("kw,status", [
    (dict(rotary_dim=3), _lib.VQB_BAD_SHAPE), (dict(rotary_dim=66), _lib.VQB_BAD_SHAPE),
    (dict(head_dim=63), _lib.VQB_BAD_SHAPE), (dict(n_tokens=-1), _lib.VQB_BAD_SHAPE),
    (dict(page_size=0), _lib.VQB_BAD_SHAPE), (dict(num_pages=0), _lib.VQB_BAD_SHAPE),
    (dict(head_dim=2048), _lib.VQB_UNSUPPORTED_GEOMETRY), (dict(n_tokens=0), _lib.VQB_OK)])
def test_rotary_refuses(kw, status):
    assert call("vqb_rotary_append", rot(**kw), [_lib.VQB_BF16] + [P] * 10) == status


def test_rotary_types_and_null_pointers():
    assert call("vqb_rotary_append", rot(), [_lib.VQB_F32] + [P] * 10) == _lib.VQB_UNSUPPORTED_GEOMETRY
    for i in range(9):
        args = [_lib.VQB_BF16] + [P] * 10
        args[1 + i] = None
        assert call("vqb_rotary_append", rot(), args) == _lib.VQB_NULL_POINTER, i


def attn(**kw):
    d = dict(n_requests=2, n_tokens=3, heads=4, kv_heads=2, head_dim=64, page_size=16, num_pages=9, table_width=4,
             max_q_len=2, max_kv_len=60, prefix_len=5, causal=1, scale=0.125, q_token_stride=256, q_head_stride=64,
             out_token_stride=256, out_head_stride=64, kc_page_stride=2048, kc_head_stride=1024, kc_token_stride=64,
             vc_page_stride=2048, vc_head_stride=1024, vc_token_stride=64)
    d.update(kw)
    return _lib.AttentionDesc(**d)


ARGS = [_lib.VQB_BF16] + [P] * 10 + [1 << 30, None]


@pytest.mark.parametrize("kw,status", [
    (dict(heads=5), _lib.VQB_BAD_SHAPE), (dict(kv_heads=0), _lib.VQB_BAD_SHAPE), (dict(scale=0.0), _lib.VQB_BAD_SHAPE),
    (dict(scale=float("nan")), _lib.VQB_BAD_SHAPE), (dict(scale=float("inf")), _lib.VQB_BAD_SHAPE),
    (dict(max_kv_len=65), _lib.VQB_BAD_SHAPE), (dict(prefix_len=-1), _lib.VQB_BAD_SHAPE),
    (dict(kc_token_stride=-64), _lib.VQB_BAD_SHAPE), (dict(head_dim=96), _lib.VQB_UNSUPPORTED_GEOMETRY),
    (dict(page_size=8), _lib.VQB_UNSUPPORTED_GEOMETRY), (dict(page_size=48), _lib.VQB_UNSUPPORTED_GEOMETRY),
    (dict(q_head_stride=68), _lib.VQB_BAD_ALIGNMENT), (dict(n_tokens=0), _lib.VQB_OK), (dict(n_requests=0), _lib.VQB_OK)])
def test_attention_refuses(kw, status):
    assert call("vqb_prefix_attention", attn(**kw), ARGS) == status
    if status != _lib.VQB_OK:
        assert call("vqb_prefix_attention_workspace_size", attn(**kw), []) == 0


def test_attention_types_pointers_and_workspace():
    assert call("vqb_prefix_attention", attn(), [_lib.VQB_F32] + ARGS[1:]) == _lib.VQB_UNSUPPORTED_GEOMETRY
    for i in (1, 2, 3, 4, 5, 6, 7, 8, 10):
        args = list(ARGS)
        args[i] = None
        assert call("vqb_prefix_attention", attn(), args) == _lib.VQB_NULL_POINTER, i
    for i in (1, 2, 3, 8, 10):
        args = list(ARGS)
        args[i] = P + 8
        assert call("vqb_prefix_attention", attn(), args) == _lib.VQB_BAD_ALIGNMENT, i
    need = call("vqb_prefix_attention_workspace_size", attn(), [])
    assert need >= 16
    assert call("vqb_prefix_attention", attn(), ARGS[:11] + [need - 1, None]) == _lib.VQB_WORKSPACE_TOO_SMALL


def test_cpu_tensors_are_refused():
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        paged_tables(i, i, i.view(2, 1), i, torch.zeros(4, dtype=torch.int64), page_size=16, max_tokens=1)
    x = torch.zeros((2, 4, 64), dtype=torch.float16)
    with pytest.raises(ValueError):
        rotary(x, i, torch.zeros(32, dtype=torch.int64))
    kv = torch.zeros((2, 2, 16, 64), dtype=torch.float16)
    with pytest.raises(ValueError):
        prefix_attention(x, kv, kv, i.view(2, 1), i, torch.zeros(3, dtype=torch.int32), max_q_len=1, max_kv_len=16)
