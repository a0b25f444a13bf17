"""Low-rank adapters of many requests beside a shared projection.

``y_t = W x_t + bias + scale_a B_a (A_a x_t)``, ``a`` the adapter of token ``t``.  ``W`` may stack several matrices by rows (query, key
and value; gate and up): each of these sections has factors of its own.  An ``AdapterPool`` holds the factors of one projection for all
loaded adapters, ``plan`` sorts out once per step which adapters its tokens use, ``linear`` and ``gate_up_glu`` are ``ops.linear`` and
``ops.gate_up_glu`` with them.

CUDA tensors run ``csrc/adapters.cu`` beside the GEMM kernels; CPU tensors the plain-PyTorch statement.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Optional, Sequence, Union

import torch
import torch.nn.functional as F

from . import GLU_ACTS, _p, _pdl, _s, glu_act, native
from .batch import MAX_ROWS, check_device

PANEL = 16             # ranks are padded to multiples of this
TILE_TOKENS = 256      # tokens that share a list of adapters
MAX_SLOTS = 8192
MAX_SECTIONS = 8
MAX_RANK = 256


class AdapterPool:
    """Factors of one projection ``[sum(sections), in_features]`` for up to ``slots`` adapters of rank up to ``rank`` per section, laid
    out as the kernels read them: ``a [slots, sections * panels * 16, in_features]``, ``b [slots, panels, rows, 16]`` with every section's
    features padded to a multiple of 8 rows (in bf16 the ranks of 8 rows as ``[2, 8 rows, 8 ranks]``), ``scale [slots]``,
    ``ranks [slots, sections]``.  A slot that was never loaded adds nothing.  What a slot holds beyond its own ranks is padding: it
    takes no part in the result, but is read and multiplied like the rest."""

    def __init__(self, slots: int, rank: int, in_features: int, sections: Union[int, Sequence[int]], *, device,
                 dtype: torch.dtype = torch.bfloat16):
        sections = (sections,) if isinstance(sections, int) else tuple(int(m) for m in sections)
        if dtype not in (torch.bfloat16, torch.float32):
            raise ValueError(f"adapters are bf16 or fp32, not {dtype}")
        if not 1 <= slots <= MAX_SLOTS or not 1 <= rank <= MAX_RANK:
            raise ValueError(f"{slots} slots of rank {rank}: at most {MAX_SLOTS} of rank {MAX_RANK}")
        if not 1 <= len(sections) <= MAX_SECTIONS or min(sections) < 1 or in_features < 1:
            raise ValueError(f"sections {sections} over {in_features} features: one to {MAX_SECTIONS} sections of at least one feature")
        if dtype == torch.bfloat16 and in_features % 8:
            raise ValueError(f"{in_features} input features: a bf16 row must be whole 16-byte vectors")
        self.slots, self.rank, self.in_features, self.sections, self.dtype = slots, rank, in_features, sections, dtype
        self.features = sum(sections)
        self.panels = -(-rank // PANEL)
        self.low = len(sections) * self.panels * PANEL
        self.rows = sum(-(-m // 8) * 8 for m in sections)
        if slots * self.low >= 2 ** 31 or slots * self.panels * self.rows >= 2 ** 31:
            raise ValueError("the pool's rows must fit 31 bits")
        self.a = torch.zeros(slots, self.low, in_features, dtype=dtype, device=device)
        self.b = torch.zeros(slots, self.panels, self.rows, PANEL, dtype=dtype, device=device)
        self.scale = torch.zeros(slots, dtype=torch.float32, device=device)
        self.ranks = torch.zeros(slots, len(sections), dtype=torch.int32, device=device)
        self.device = self.a.device
        ends = [sum(sections[:i + 1]) for i in range(len(sections))]
        self._ends = (ctypes.c_int * len(ends))(*ends)

    @torch.no_grad()
    def load(self, slot: int, a, b, scale: float = 1.0) -> None:
        """``a``: ``[r, in_features]`` and ``b``: ``[features, r]``, or one of each per section; ranks up to the pool's.  The copies are
        made on the current stream, and the host waits for them: not for the middle of a step, nor for a captured graph.  Factors that
        are not finite are refused: tokens of other adapters meet them as products with zero."""
        a, b = ([f] if isinstance(f, torch.Tensor) else list(f) for f in (a, b))
        if not 0 <= slot < self.slots:
            raise ValueError(f"slot {slot} of {self.slots}")
        if len(a) != len(self.sections) or len(b) != len(self.sections):
            raise ValueError(f"{len(a)} and {len(b)} factors for {len(self.sections)} sections")
        for fa, fb, m in zip(a, b, self.sections):
            if fa.dim() != 2 or fb.dim() != 2 or fa.shape[1] != self.in_features or fb.shape[0] != m or fa.shape[0] != fb.shape[1]:
                raise ValueError(f"factors {tuple(fa.shape)} and {tuple(fb.shape)} for {self.in_features} -> {m}")
            if not 1 <= fa.shape[0] <= self.rank:
                raise ValueError(f"rank {fa.shape[0]}, the pool holds up to {self.rank}")
        pa = torch.zeros(len(a), self.panels * PANEL, self.in_features, dtype=self.dtype, device=self.device)
        pb = torch.zeros(self.rows, self.panels * PANEL, dtype=self.dtype, device=self.device)
        first = 0
        for i, (fa, fb, m) in enumerate(zip(a, b, self.sections)):
            pa[i, :fa.shape[0]] = fa
            pb[first:first + m, :fb.shape[1]] = fb
            first += -(-m // 8) * 8
        if not math.isfinite(ctypes.c_float(float(scale)).value) or not bool(torch.isfinite(pa).all() & torch.isfinite(pb).all()):
            raise ValueError("factors and scale must be finite")
        self.a[slot] = pa.view(self.low, self.in_features)
        self.b[slot] = self._panels(pb.view(self.rows, self.panels, PANEL).transpose(0, 1))
        self.scale[slot] = float(scale)
        for i, fa in enumerate(a):
            self.ranks[slot, i] = fa.shape[0]

    def _panels(self, b: torch.Tensor) -> torch.Tensor:
        """``[panels, rows, 16]`` in the pool's order."""
        return b if self.dtype != torch.bfloat16 else b.reshape(b.shape[0], -1, 8, 2, 8).transpose(2, 3).reshape(b.shape)

    def _features(self, slot: int, section: int) -> torch.Tensor:
        """``[features of the section, panels * 16]`` from the pool's order."""
        first, m = sum(-(-n // 8) * 8 for n in self.sections[:section]), self.sections[section]
        b = self.b[slot, :, first:first + -(-m // 8) * 8]
        if self.dtype == torch.bfloat16:
            b = b.reshape(b.shape[0], -1, 2, 8, 8).transpose(2, 3).reshape(b.shape)
        return b.transpose(0, 1).reshape(b.shape[1], -1)[:m]

    @torch.no_grad()
    def clear(self, slot: int) -> None:
        """The slot adds nothing from here on."""
        if not 0 <= slot < self.slots:
            raise ValueError(f"slot {slot} of {self.slots}")
        self.a[slot] = 0
        self.b[slot] = 0
        self.scale[slot] = 0
        self.ranks[slot] = 0


@dataclass
class AdapterPlan:
    """``adapter [T]``: slot of every token, negative for none; per tile of 256 tokens the slots in use, ascending
    (``lists [tiles, capacity]``, -1 behind), their number (``counts [tiles]``); ``index [T]``: a token's place in its tile's list."""

    adapter: torch.Tensor
    slots: int
    index: torch.Tensor
    lists: torch.Tensor
    counts: torch.Tensor


def plan(adapter: torch.Tensor, slots: int) -> AdapterPlan:
    """Once per step, for every projection whose pool has ``slots`` slots; again when ``adapter`` has changed.  ``adapter``: contiguous int32, one per token.  Slots out of
    range count as none and set the ``adapters`` status word (``native.check_status``); on CPU they raise."""
    if adapter.dtype != torch.int32 or adapter.dim() != 1 or not adapter.is_contiguous():
        raise ValueError("adapter must be a contiguous one-dimensional int32 tensor")
    if not 1 <= slots <= MAX_SLOTS:
        raise ValueError(f"{slots} slots, one to {MAX_SLOTS}")
    T = adapter.shape[0]
    if T > MAX_ROWS:
        raise ValueError(f"{T} tokens")
    tiles, capacity = -(-T // TILE_TOKENS), min(slots, TILE_TOKENS, T)
    if not adapter.is_cuda:
        if T and int(adapter.max()) >= slots:
            raise ValueError(f"adapter {int(adapter.max())} of {slots} slots")
        index, lists, counts = torch.full((T,), -1, dtype=torch.int32), torch.full((tiles, capacity), -1, dtype=torch.int32), torch.zeros(tiles, dtype=torch.int32)
        for i in range(tiles):
            who = adapter[i * TILE_TOKENS:(i + 1) * TILE_TOKENS]
            used = torch.unique(who[who >= 0])
            lists[i, :len(used)] = used
            counts[i] = len(used)
            index[i * TILE_TOKENS:(i + 1) * TILE_TOKENS] = torch.where(who >= 0, torch.searchsorted(used, who).int(), -1)
        return AdapterPlan(adapter, slots, index, lists, counts)
    check_device(adapter)
    index, lists, counts = torch.split_with_sizes(torch.empty(T + tiles * capacity + tiles, dtype=torch.int32, device=adapter.device),
                                                  (T, tiles * capacity, tiles))
    if T:
        native.call("prism_adapter_plan", _p(adapter), T, slots, capacity, _p(index), _p(lists), _p(counts), _s(), _pdl())
    return AdapterPlan(adapter, slots, index, lists.view(tiles, capacity), counts)


def _ld(t: torch.Tensor) -> int:
    """Row stride; a single row may have any."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _check(x: torch.Tensor, w: torch.Tensor, pool: AdapterPool, p: AdapterPlan, bias: Optional[torch.Tensor], out: Optional[torch.Tensor],
           features: int) -> None:
    dtype, device, K = pool.dtype, pool.device, pool.in_features
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != K or w.shape[0] != pool.features or w.shape[1] != K:
        raise ValueError(f"x {tuple(x.shape)} and w {tuple(w.shape)} for a pool of {K} -> {pool.features}")
    if x.dtype != dtype or w.dtype != dtype or x.device != device or w.device != device or p.adapter.device != device:
        raise ValueError(f"tensors must be {dtype} on {device}, as the pool is")
    if p.slots != pool.slots or p.adapter.shape[0] != x.shape[0]:
        raise ValueError(f"a plan of {p.adapter.shape[0]} tokens over {p.slots} slots for {x.shape[0]} tokens and {pool.slots} slots")
    if bias is not None and (bias.dtype != dtype or bias.device != device or bias.shape != (pool.features,) or not bias.is_contiguous()):
        raise ValueError(f"bias must be contiguous {dtype} on {device}, one value for each of {pool.features} features")
    if out is not None and (out.dtype != dtype or out.device != device or out.shape != (x.shape[0], features) or (features > 1 and out.stride(1) != 1)
                            or _ld(out) < features):
        raise ValueError(f"out must be {dtype} on {device} of shape {(x.shape[0], features)}, with contiguous rows that are apart")
    for name, t in (("x", x), ("w", w)):
        ld = _ld(t)
        if (K > 1 and t.stride(1) != 1) or ld < K or (dtype == torch.bfloat16 and (ld % 8 or t.data_ptr() % 16)):
            raise ValueError(f"{name}: rows must be contiguous and apart, in bf16 on 16-byte boundaries")
    check_device(x)


def _adapted_cpu(x, w, pool, p, bias):
    y = F.linear(x.float(), w.float())
    if bias is not None:
        y += bias.float()
    for s in torch.unique(p.adapter[p.adapter >= 0]).tolist():
        rows = (p.adapter == s).nonzero()[:, 0]
        low = F.linear(x[rows].float(), pool.a[s].float()) * pool.scale[s]
        first, r = 0, pool.panels * PANEL
        for i, m in enumerate(pool.sections):
            n = int(pool.ranks[s, i])
            y[rows, first:first + m] += F.linear(low[:, i * r:i * r + n], pool._features(s, i)[:, :n].float())
            first += m
    return y


# bytes of bf16 low-rank rows in one launch, and tokens of either type (tiles of 128 along an axis of the grid); a step that needs more runs in
# runs of tokens
MAX_LOW_BYTES = 256 << 20
MAX_RUN = 65535 * 128


def _tile_rows(tokens: int) -> int:
    """Tokens of a panel: those of a decode step, rounded up to the kernels' sizes, or a tile of a prompt."""
    return TILE_TOKENS if tokens > 128 else 16 if tokens <= 16 else 1 << (tokens - 1).bit_length()


def _run(x, w, pool, p, bias, out, act):
    T = x.shape[0]
    if T == 0:
        return out
    if pool.dtype == torch.float32:
        return _run_f32(x, w, pool, p, bias, out, act)
    tiles, capacity = p.lists.shape
    tile_rows, ldx, ldo = _tile_rows(T), _ld(x), _ld(out)
    per_tile = capacity * pool.low * tile_rows     # values of every panel that a tile's adapters may need
    run = min(tiles, max(1, MAX_LOW_BYTES // (2 * per_tile)), MAX_RUN // TILE_TOKENS)
    h = torch.empty(run * per_tile, dtype=torch.bfloat16, device=x.device)
    x_at, out_at, index_at, lists_at, counts_at = x.data_ptr(), out.data_ptr(), p.index.data_ptr(), p.lists.data_ptr(), p.counts.data_ptr()
    rest = (pool.features, pool.in_features, pool.slots, pool.panels, len(pool.sections), pool._ends, capacity)
    n = min(run * TILE_TOKENS, T)
    while T > 0:
        if n > T:       # the last run of several
            n, tile_rows = T, _tile_rows(T)
        native.call("prism_adapter_linear", x_at, w.data_ptr(), pool.a.data_ptr(), pool.b.data_ptr(), pool.scale.data_ptr(), pool.ranks.data_ptr(), index_at,
                    lists_at, counts_at, _p(bias), out_at, h.data_ptr(), n, *rest, tile_rows, act, ldx, _ld(w), ldo, _s(), _pdl())
        x_at, out_at, index_at = x_at + 2 * n * ldx, out_at + 2 * n * ldo, index_at + 4 * n
        lists_at, counts_at, T = lists_at + 4 * run * capacity, counts_at + 4 * run, T - n
    return out


def _run_f32(x, w, pool, p, bias, out, act):
    T, ldx, ldo = x.shape[0], _ld(x), _ld(out)
    h = torch.empty(min(T, MAX_RUN), pool.low, dtype=torch.float32, device=x.device)
    for first in range(0, T, MAX_RUN):
        native.call("prism_adapter_linear_f32", x.data_ptr() + 4 * first * ldx, _p(w), _p(pool.a), _p(pool.b), _p(pool.scale), _p(pool.ranks),
                    p.adapter.data_ptr() + 4 * first, _p(bias), out.data_ptr() + 4 * first * ldo, _p(h), min(MAX_RUN, T - first), pool.features,
                    pool.in_features, pool.slots, pool.panels, len(pool.sections), pool._ends, act, ldx, _ld(w), ldo, _s(), _pdl())
    return out


def linear(x: torch.Tensor, w: torch.Tensor, pool: AdapterPool, p: AdapterPlan, *, bias: Optional[torch.Tensor] = None,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ w.T + bias`` and every token's adapter; x ``[T, K]``, w ``[M, K]`` -> ``[T, M]``.  Sums and scale in 32 bits; in bf16 the low-rank
    row is rounded once, as an operand of the matrix instructions, and so is the result.  ``out`` shares no memory with the inputs."""
    _check(x, w, pool, p, bias, out, pool.features)
    if not x.is_cuda:
        y = _adapted_cpu(x, w, pool, p, bias).to(x.dtype)
        return y if out is None else out.copy_(y)
    if out is None:
        out = torch.empty(x.shape[0], pool.features, dtype=x.dtype, device=x.device)
    return _run(x, w, pool, p, bias, out, 0)


def gate_up_glu(x: torch.Tensor, w_gate_up: torch.Tensor, pool: AdapterPool, p: AdapterPlan, act: str, *,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(gate) * up`` with ``w_gate_up = [Wg ; Wu]`` and the adapters of both (a pool of two equal sections); ``act`` is ``silu`` or
    ``gelu_tanh``.  Sums, activation and product in 32 bits, rounded as ``linear`` rounds.  In bf16 a row whose low-rank values are
    infinite becomes not a number: the matrix instructions meet a gate's low-rank row with zeros for the up half, and the other way round."""
    if act not in ("silu", "gelu_tanh"):
        raise ValueError(f"act {act!r} is neither silu nor gelu_tanh")
    if len(pool.sections) != 2 or pool.sections[0] != pool.sections[1]:
        raise ValueError(f"a gated unit has two equal sections, the pool {pool.sections}")
    half = pool.sections[0]
    _check(x, w_gate_up, pool, p, None, out, half)
    if not x.is_cuda:
        y = _adapted_cpu(x, w_gate_up, pool, p, None)
        y = (glu_act(y[:, :half], act) * y[:, half:]).to(x.dtype)
        return y if out is None else out.copy_(y)
    if out is None:
        out = torch.empty(x.shape[0], half, dtype=x.dtype, device=x.device)
    return _run(x, w_gate_up, pool, p, None, out, GLU_ACTS[act])
