"""Maps of a step, from the lengths of its requests.

A step brings ``fresh[i]`` new tokens of request ``i``, behind ``cached[i]`` that are in the paged cache already.  ``step_maps``
makes what the other operators read of that: the padded block tables, the cache slot, position, request and adapter of every token,
and the running sums of the lengths.  The host keeps what it allocates, the pages of each request; it hands them over as one flat
list.  CUDA tensors run ``csrc/batch.cu`` (one launch, no copy to the host, fit for a captured graph); CPU tensors the plain-PyTorch
statement.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import _p, _pdl, _s, native

MAX_REQUESTS = 8192
MAX_ROWS = 1 << 30


@dataclass
class StepMaps:
    """``block_tables [S, width]`` int32 (-1 behind a request's pages); ``slots [T]`` int64; ``positions [3, T]`` int32, alike on the
    three axes; ``token_seq [T]``, ``token_adapter [T]`` int32; ``cu_seqlens_q``, ``cu_seqlens_kv [S + 1]``, ``kv_lens [S]`` int32;
    ``sample_rows [S]`` int64, the row of a request's last new token (-1: it has none).  Rows behind the last request's tokens have
    slot, request and adapter -1 and position 0."""

    block_tables: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    token_seq: torch.Tensor
    cu_seqlens_q: torch.Tensor
    cu_seqlens_kv: torch.Tensor
    kv_lens: torch.Tensor
    sample_rows: torch.Tensor
    token_adapter: Optional[torch.Tensor] = None


def _check_index(name: str, t: torch.Tensor, device: torch.device, shape: Optional[tuple[int, ...]] = None) -> None:
    if t.dtype != torch.int32 or t.device != device or not t.is_contiguous() or t.dim() != 1:
        raise ValueError(f"{name} must be a contiguous one-dimensional int32 tensor on {device}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, not {shape}")


def check_device(t: torch.Tensor) -> None:
    """Kernels go to the current device's current stream."""
    if t.is_cuda and t.device.index != torch.cuda.current_device():
        raise ValueError(f"tensors on {t.device}, but the current device is cuda:{torch.cuda.current_device()}")


def step_maps(pages: torch.Tensor, cached: torch.Tensor, fresh: torch.Tensor, *, page: int, tokens: int, width: int,
              page_offsets: Optional[torch.Tensor] = None, shift: Optional[torch.Tensor] = None,
              adapter: Optional[torch.Tensor] = None) -> StepMaps:
    """``pages``: int32, the ``ceil((cached + fresh) / page)`` pages of every request, one request after another; with
    ``page_offsets [S + 1]`` request ``i`` owns ``pages[page_offsets[i]:page_offsets[i + 1]]``, which may hold more than it needs yet.
    ``tokens``: rows of the per-token maps, at least the sum of ``fresh``; ``width``: entries of a table row, at least the most
    pages that a request needs.  ``shift [S]`` is added to a request's positions; ``adapter [S]`` (-1: none) is spread to its tokens.
    Up to 8192 requests.

    The lengths are read on the device, where nothing can be raised: on a CUDA tensor lengths that contradict the sizes set the
    ``batch`` status word (``native.check_status``).  Negative lengths then count as zero, tokens past ``tokens`` are left out of the
    running sums, tokens without a page have slot -1, pages past ``width`` are left out of the table.  On CPU they raise."""
    S, device = cached.shape[0] if cached.dim() else -1, cached.device
    _check_index("cached", cached, device)
    _check_index("fresh", fresh, device, (S,))
    _check_index("pages", pages, device)
    for name, t, shape in (("page_offsets", page_offsets, (S + 1,)), ("shift", shift, (S,)), ("adapter", adapter, (S,))):
        if t is not None:
            _check_index(name, t, device, shape)
    if page < 1 or tokens < 0 or width < 1:
        raise ValueError(f"page {page} and width {width} must be positive, tokens {tokens} not negative")
    if S > MAX_REQUESTS:
        raise ValueError(f"{S} requests, at most {MAX_REQUESTS} in a step")
    if tokens > MAX_ROWS or width > MAX_ROWS or page >= 2 ** 31 or pages.shape[0] >= 2 ** 31:
        raise ValueError(f"at most {MAX_ROWS} tokens and table entries, pages and their list within 31 bits")
    if not cached.is_cuda:
        return _step_maps_cpu(pages, cached, fresh, page, tokens, width, page_offsets, shift, adapter)
    check_device(cached)
    # one allocation per type
    tables, positions, seq, who, cu_q, cu_kv, kv = torch.split_with_sizes(
        torch.empty(S * width + 5 * tokens + 3 * S + 2, dtype=torch.int32, device=device),
        (S * width, 3 * tokens, tokens, tokens, S + 1, S + 1, S))
    slots, sample = torch.split_with_sizes(torch.empty(tokens + S, dtype=torch.int64, device=device), (tokens, S))
    native.call("prism_step_maps", _p(pages), _p(page_offsets), _p(cached), _p(fresh), _p(shift), _p(adapter), S, tokens, width, page,
                pages.shape[0], _p(tables), _p(slots), _p(positions), _p(seq), _p(who) if adapter is not None else None, _p(cu_q), _p(cu_kv),
                _p(kv), _p(sample), _s(), _pdl())
    return StepMaps(tables.view(S, width), slots, positions.view(3, tokens), seq, cu_q, cu_kv, kv, sample, who if adapter is not None else None)


def _step_maps_cpu(pages, cached, fresh, page, tokens, width, page_offsets, shift, adapter) -> StepMaps:
    S = cached.shape[0]
    c, f = cached.long(), fresh.long()
    if S and int(torch.minimum(c, f).min()) < 0:
        raise ValueError("negative lengths")
    kv = c + f
    zero = torch.zeros(1, dtype=torch.int64)
    cu_q, cu_kv, need = torch.cat([zero, f.cumsum(0)]), torch.cat([zero, kv.cumsum(0)]), (kv + page - 1) // page
    total = int(cu_q[-1])
    if total > tokens or int(cu_kv[-1]) >= 2 ** 31:
        raise ValueError(f"{total} new tokens for {tokens} rows, {int(cu_kv[-1])} tokens in all")
    if S and int(need.max()) > width:
        raise ValueError(f"a request needs {int(need.max())} pages, the tables hold {width}")
    bounds = torch.cat([zero, need.cumsum(0)]) if page_offsets is None else page_offsets.long()
    if S and (int(bounds[1:].max()) > pages.shape[0] or int(bounds[0]) < 0 or bool((bounds[1:] - bounds[:-1] < need).any())):
        raise ValueError("the list holds fewer pages than the lengths need")
    table = torch.full((S, width), -1, dtype=torch.int32)
    slots = torch.full((tokens,), -1, dtype=torch.int64)
    positions = torch.zeros(3, tokens, dtype=torch.int32)
    seq = torch.full((tokens,), -1, dtype=torch.int32)
    who = torch.full((tokens,), -1, dtype=torch.int32) if adapter is not None else None
    for i in range(S):
        mine = pages[int(bounds[i]):int(bounds[i]) + int(need[i])]
        table[i, :len(mine)] = mine
        lo, hi = int(cu_q[i]), int(cu_q[i + 1])
        p = torch.arange(int(c[i]), int(kv[i]))
        ids = mine.long()[p // page]
        slots[lo:hi] = torch.where(ids >= 0, ids * page + p % page, -1)
        positions[:, lo:hi] = (p + (int(shift[i]) if shift is not None else 0)).int()
        seq[lo:hi] = i
        if who is not None:
            who[lo:hi] = adapter[i]
    i32 = torch.int32
    return StepMaps(table, slots, positions, seq, cu_q.to(i32), cu_kv.to(i32), kv.to(i32), torch.where(f > 0, cu_q[1:] - 1, -1), who)
