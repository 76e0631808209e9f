"""The attention part of a served layer: the paged key/value cache, rotary
positions and attention, between the q/k/v projections and the output projection.

Three library calls (include/vqb.h), one launch chain each, all on the current
stream with no host synchronisation (their arguments are checked and their
outputs allocated in csrc/attention_binding.cpp):

  paged_tables      the step's block tables, lengths and slot map, built on the
                    device from the requests' lengths (vqb_paged_tables)
  rotary_append     rotary positions on q and k, k and v into the cache's pages
                    (vqb_rotary_append); `rotary` turns one tensor alone
  prefix_attention  attention over the paged cache, for single tokens up to long
                    prompts, with a prefix that the whole batch shares computed
                    once for all (vqb_prefix_attention)

`PagedKVCache` keeps the pools and the allocator's state over steps, and
`VQAttention` is the layer: four VQLinear projections around the calls.  The
reference's host library supplies this part, so there is no counterpart to
cite; its dense projections are src/vqlab/runtime/vq_dense.py:315-441.
Serving only: no gradients.  CUDA tensors only; fp16 and bf16.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch

from . import _lib
from .vq_dense import VQLinear

_HALF = (torch.float16, torch.bfloat16)


def _need(cond: bool, what: str) -> None:
    if not cond:
        raise ValueError(what)


class PagedTables(NamedTuple):
    """What a step's calls read (vqb_paged_tables)."""
    block_table: torch.Tensor   # int32 [R, W], -1 where no page
    kv_lens: torch.Tensor       # int32 [R], tokens held after the step
    cu_q: torch.Tensor          # int32 [R + 1], where each request's new tokens start
    slots: torch.Tensor         # int32 [max_tokens], -1: not stored
    positions: torch.Tensor     # int32 [max_tokens]
    requests: torch.Tensor      # int32 [max_tokens], -1: padding
    free_pages: torch.Tensor    # int32 [F], the ring of free pages
    state: torch.Tensor         # int64 [4]: start, end, requests refused, 0

    def refused_requests(self) -> torch.Tensor:
        """bool [R], on the device: requests with new tokens that got no place in
        this step.  Their tokens (slots -1) are in no cache, and prefix_attention
        takes their queries for the last of what the request already holds: their
        rows of its result are to be thrown away, and the tokens given again."""
        first, end = self.cu_q[:-1], self.cu_q[1:]
        places = self.slots.numel()
        if places == 0:
            return torch.zeros_like(first, dtype=torch.bool)
        return (end > first) & (first < places) & (self.slots[first.clamp(max=places - 1).long()] < 0)


def paged_tables(context_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor,
                 free_pages: torch.Tensor, state: torch.Tensor, *, page_size: int, max_tokens: int,
                 position_offset: int = 0, inplace: bool = False) -> PagedTables:
    """One step's tables: request r holds context_lens[r] tokens and gets
    new_lens[r] more (-1: it has finished and gives its pages back).

    inplace updates block_table, context_lens (returned as kv_lens), free_pages
    and state; otherwise they are left as they are and new tensors returned
    (state[3] counts the call's blocks meanwhile and is 0 again after it).
    max_tokens must cover the new tokens; further places are padding.  A request
    that gets no pages is refused: it keeps what it holds, and its new tokens,
    which cu_q still counts, have slot -1 (PagedTables.refused_requests)."""
    got = (_lib._native or _lib.native()).paged_tables(context_lens, new_lens, block_table, free_pages, state, page_size,
                                                       max_tokens, position_offset, inplace)
    if type(got) is int:
        _lib.check(got, "vqb_paged_tables")
    return PagedTables._make(got)


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                       original_length: int = 0, low: float = 1.0, high: float = 32.0, device="cuda"):
    """(freq, amplitude) for rotary_append: turns per position of each pair as
    fixed point of 64 fraction bits (int64, taken modulo 2^64), from
    base ** (-2 i / rotary_dim) in 64-bit floating point.

    scaling: None; "linear" (every frequency over `factor`); "base" (the base
    times factor ** (d / (d - 2)), which keeps the fastest pair and slows the
    slowest by `factor`); "ramp" (pairs that turn fewer than `low` times over
    original_length are slowed by `factor`, those over `high` turns kept, a
    linear ramp between in the pair's index; amplitude 0.1 ln(factor) + 1)."""
    _need(rotary_dim >= 2 and rotary_dim % 2 == 0, "rotary_dim must be even")
    _need(scaling in (None, "linear", "base", "ramp"), "scaling must be None, 'linear', 'base' or 'ramp'")
    _need(factor > 0 and base > 1, "factor and base must be positive, base over 1")
    amplitude, d = 1.0, rotary_dim
    if scaling == "base" and d > 2:
        base = base * factor ** (d / (d - 2))
    freq = [base ** (-2.0 * i / d) for i in range(d // 2)]
    if scaling == "linear" or (scaling == "base" and d == 2):
        freq = [f / factor for f in freq]
    elif scaling == "ramp":
        _need(original_length > 0 and 0 < low < high, "'ramp' needs original_length and 0 < low < high")

        def index(turns):  # the (real) pair index that turns this often over original_length
            return d * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))
        first, last = max(math.floor(index(high)), 0), min(math.ceil(index(low)), d - 1)
        for i in range(d // 2):
            slow = min(max((i - first) / max(last - first, 1e-3), 0.0), 1.0)
            freq[i] = freq[i] * (1 - slow) + freq[i] / factor * slow
        amplitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    fixed = [int(f / (2 * math.pi) * 2.0 ** 64) % (1 << 64) for f in freq]
    return torch.tensor([f - (1 << 64) if f >> 63 else f for f in fixed], dtype=torch.int64, device=device), amplitude


def rotary_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, freq: torch.Tensor,
                  k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor, *, interleaved: bool = False,
                  amplitude: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate q [N, heads, D] and k [N, kv_heads, D], store k and v in the caches
    [pages, kv_heads, page_size, D] at `slots` (outside the pool: not stored), and
    return the rotated q (in `out`, which may be q).  positions and slots may be
    longer than N (a step's padding).  The tensors may be slices of one fused
    projection: any strides with contiguous heads."""
    if k is None:
        raise ValueError("k must be a tensor (rotary() rotates one tensor alone)")
    got = (_lib._native or _lib.native()).rotary_append(q, k, v, positions, freq, k_cache, v_cache, slots, interleaved,
                                                        amplitude, out)
    if type(got) is int:
        _lib.check(got, "vqb_rotary_append")
    return got


def rotary(x: torch.Tensor, positions: torch.Tensor, freq: torch.Tensor, *, interleaved: bool = False,
           amplitude: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate x [N, heads, D] alone (vqb_rotary_append without a cache)."""
    got = (_lib._native or _lib.native()).rotary_append(x, None, None, positions, freq, None, None, None, interleaved,
                                                        amplitude, out)
    if type(got) is int:
        _lib.check(got, "vqb_rotary_append")
    return got


def prefix_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                     kv_lens: torch.Tensor, cu_q: torch.Tensor, *, max_q_len: int, max_kv_len: int,
                     prefix_pages: torch.Tensor | None = None, prefix_len: int = 0, scale: float | None = None,
                     causal: bool = True, out: torch.Tensor | None = None, return_lse: bool = False,
                     workspace: torch.Tensor | None = None):
    """Attention of the requests' queries q [N, heads, D] (request r's are rows
    cu_q[r] to cu_q[r + 1], the last of the kv_lens[r] tokens it holds) over the
    caches [pages, kv_heads, page_size, D]: first the prefix that all share
    (prefix_len tokens in prefix_pages), then the request's own tokens in the
    pages of its block table row.  Causal within the request's own tokens; a
    query that sees nothing gives 0.  Scores, softmax and sums are fp32; the
    weights are rounded to the caches' type before they meet the values, and the
    result once.  max_q_len and max_kv_len bound the
    requests' lengths, which stay on the device.  scale defaults to D ** -0.5.
    Returns [N, heads, D], and with return_lse the fp32 log-sum-exp [N, heads]
    of the scaled scores; rows past cu_q[-1] are not written.  out must not
    overlap q or the caches.  workspace: a uint8 tensor that is large enough
    (attention_workspace), whose first 16 bytes become the call's status block
    (check_attention); allocated per call when None, and the status is lost then."""
    got = (_lib._native or _lib.native()).prefix_attention(q, k_cache, v_cache, block_table, kv_lens, cu_q, max_q_len,
                                                           max_kv_len, prefix_pages, prefix_len, scale, causal, out,
                                                           return_lse, workspace)
    if type(got) is int:
        _lib.check(got, "vqb_prefix_attention")
    return got


def attention_workspace(n_tokens: int, requests: int, heads: int, kv_heads: int, head_dim: int, page_size: int, *,
                        max_q_len: int, max_kv_len: int, prefix_len: int = 0, device="cuda") -> torch.Tensor:
    """A workspace for prefix_attention calls of these sizes, for a caller that wants
    to read a call's status (check_attention); without one a call allocates its own."""
    d = _lib.AttentionDesc(n_requests=requests, n_tokens=n_tokens, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                           page_size=page_size, num_pages=1, table_width=-(-max_kv_len // page_size),
                           max_q_len=max_q_len, max_kv_len=max_kv_len, prefix_len=prefix_len, scale=1.0)
    size = int(_lib.lib().vqb_prefix_attention_workspace_size(ctypes.byref(d)))
    _need(size > 0, "prefix_attention does not take these sizes")
    return torch.empty(size, dtype=torch.uint8, device=device)


def check_attention(workspace: torch.Tensor) -> None:
    """Raise VQBError if a bounded wait on the device gave up in the last
    prefix_attention call with this workspace, whose result is then incomplete
    (reads the device).  Every call clears what the one before it left."""
    _lib.check(int(workspace[4:8].view(torch.int32)), "vqb_prefix_attention")


class PagedKVCache:
    """The key and value pools of a model's layers and one batch's tables over
    them.  `step` builds a step's tables in place; `share` turns what a request
    holds into the batch's shared prefix, `unshare` gives its pages back."""

    def __init__(self, layers: int, num_pages: int, page_size: int, kv_heads: int, head_dim: int, max_requests: int,
                 max_context: int, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        _need(dtype in _HALF, "dtype must be float16 or bfloat16")
        shape = (layers, num_pages, kv_heads, page_size, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        self.page_size = int(page_size)
        width = -(-max_context // page_size)
        self.block_table = torch.full((max_requests, width), -1, dtype=torch.int32, device=device)
        self.kv_lens = torch.zeros(max_requests, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(num_pages, dtype=torch.int32, device=device)
        self.state = torch.tensor([0, num_pages, 0, 0], dtype=torch.int64, device=device)
        self.prefix_pages = None
        self.prefix_len = 0

    def step(self, new_lens: torch.Tensor, max_tokens: int) -> PagedTables:
        """The tables of a step in which request r gets new_lens[r] tokens (-1: it has finished)."""
        return paged_tables(self.kv_lens, new_lens, self.block_table, self.free_pages, self.state,
                            page_size=self.page_size, max_tokens=max_tokens, position_offset=self.prefix_len,
                            inplace=True)

    def refused(self) -> int:
        """How many requests the last step could give no pages (reads the device; its
        tables' refused_requests says which)."""
        return int(self.state[2])

    def share(self, request: int) -> None:
        """Make the tokens that `request` holds the prefix of every request (reads
        the device; no other request may hold tokens, and there is one prefix)."""
        _need(self.prefix_len == 0, "the batch has a shared prefix already")
        lens = self.kv_lens.tolist()
        _need(0 <= request < len(lens) and lens[request] > 0, "the request holds nothing")
        _need(sum(n > 0 for n in lens) == 1, "another request holds tokens")
        n = lens[request]
        self.prefix_pages = self.block_table[request, :-(-n // self.page_size)].clone()
        self.prefix_len = n
        self.block_table[request].fill_(-1)
        self.kv_lens[request] = 0

    def unshare(self) -> None:
        """Give the shared prefix's pages back (reads the device; no request may hold
        tokens, whose places follow the prefix's).  Another may then be shared."""
        _need(self.prefix_len > 0, "the batch has no shared prefix")
        _need(not any(self.kv_lens.tolist()), "a request holds tokens behind the prefix")
        n = self.prefix_pages.numel()
        at = (self.state[1] + torch.arange(n, device=self.state.device)) % self.free_pages.numel()
        self.free_pages[at] = self.prefix_pages
        self.state[1] += n
        self.prefix_pages = None
        self.prefix_len = 0


class VQAttention(torch.nn.Module):
    """A layer's attention over the paged cache: q / k / v projections, rotary
    positions and the append, attention, output projection.  The projections
    are VQLinear (or any module of the same shapes): q [heads * D, hidden],
    k and v [kv_heads * D, hidden], o [hidden, heads * D]."""

    def __init__(self, q_proj: VQLinear, k_proj: VQLinear, v_proj: VQLinear, o_proj: VQLinear, heads: int,
                 kv_heads: int, head_dim: int, freq: torch.Tensor, amplitude: float = 1.0, interleaved: bool = False,
                 scale: float | None = None):
        super().__init__()
        self.q_proj, self.k_proj, self.v_proj, self.o_proj = q_proj, k_proj, v_proj, o_proj
        self.heads, self.kv_heads, self.head_dim = int(heads), int(kv_heads), int(head_dim)
        _need(self.heads % self.kv_heads == 0, "heads must be a multiple of kv_heads")
        self.register_buffer("freq", freq, persistent=False)
        self.amplitude, self.interleaved, self.scale = float(amplitude), bool(interleaved), scale

    def forward(self, x: torch.Tensor, cache: PagedKVCache, layer: int, step: PagedTables, max_q_len: int,
                max_kv_len: int, workspace: torch.Tensor | None = None) -> torch.Tensor:
        """x [N, hidden], the step's new tokens in the order of its tables ->
        [N, hidden].  max_q_len / max_kv_len: the largest new_lens and kv_lens.
        Rows of a refused request's tokens (step.slots -1) mean nothing.
        workspace: prefix_attention's."""
        N = x.shape[0]
        q = self.q_proj(x).view(N, self.heads, self.head_dim)
        k = self.k_proj(x).view(N, self.kv_heads, self.head_dim)
        v = self.v_proj(x).view(N, self.kv_heads, self.head_dim)
        kc, vc = cache.k[layer], cache.v[layer]
        q = rotary_append(q, k, v, step.positions, self.freq, kc, vc, step.slots, interleaved=self.interleaved,
                          amplitude=self.amplitude, out=q)
        o = prefix_attention(q, kc, vc, step.block_table, step.kv_lens, step.cu_q, max_q_len=max_q_len,
                             max_kv_len=max_kv_len, prefix_pages=cache.prefix_pages, prefix_len=cache.prefix_len,
                             scale=self.scale, workspace=workspace)
        return self.o_proj(o.view(N, self.heads * self.head_dim))
