"""Maps of a step against plain loops.  CPU statement, and the kernel on a B200."""

import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from op_helpers import CPU, GPU32  # noqa: E402

from prism_infer_b200.ops import batch, native  # noqa: E402

BACKENDS = [CPU, GPU32]
FIELDS = ("block_tables", "slots", "positions", "token_seq", "cu_seqlens_q", "cu_seqlens_kv", "kv_lens", "sample_rows", "token_adapter")


def plain(pages, cached, fresh, page, tokens, width, bounds=None, shift=None, adapter=None):
    out = {f: [] for f in FIELDS}
    out["cu_seqlens_q"], out["cu_seqlens_kv"] = [0], [0]
    at, pos = 0, []
    for i, (c, f) in enumerate(zip(cached, fresh)):
        need = -(-(c + f) // page)
        mine = pages[at:at + need] if bounds is None else pages[bounds[i]:bounds[i + 1]][:need]
        at += need
        out["block_tables"].append(mine + [-1] * (width - need))
        for p in range(c, c + f):
            out["slots"].append(mine[p // page] * page + p % page)
            pos.append(p + (shift[i] if shift else 0))
            out["token_seq"].append(i)
            out["token_adapter"].append(adapter[i] if adapter else -1)
        out["cu_seqlens_q"].append(out["cu_seqlens_q"][-1] + f)
        out["cu_seqlens_kv"].append(out["cu_seqlens_kv"][-1] + c + f)
        out["kv_lens"].append(c + f)
        out["sample_rows"].append(out["cu_seqlens_q"][-1] - 1 if f else -1)
    rest = tokens - len(pos)
    for f in ("slots", "token_seq", "token_adapter"):
        out[f] += [-1] * rest
    out["positions"] = [pos + [0] * rest] * 3
    return out


def case(S, most_cached, most_fresh, page, seed):
    g = torch.Generator().manual_seed(seed)
    cached = torch.randint(0, most_cached + 1, (S,), generator=g)
    fresh = torch.randint(0, most_fresh + 1, (S,), generator=g)
    n = int(((cached + fresh + page - 1) // page).sum())
    pages = torch.randperm(n + 5, generator=g)[:n]
    return [t.tolist() for t in (pages, cached, fresh)], g


def call(device, pages, cached, fresh, **kw):
    kw = {k: torch.tensor(v, dtype=torch.int32, device=device) if isinstance(v, list) else v for k, v in kw.items()}
    return batch.step_maps(*(torch.tensor(v, dtype=torch.int32, device=device) for v in (pages, cached, fresh)), **kw)


def same(got, want, S, width, adapter=True):
    for f in FIELDS:
        t = getattr(got, f)
        if f == "token_adapter" and not adapter:
            assert t is None
            continue
        assert t.dtype == (torch.int64 if f in ("slots", "sample_rows") else torch.int32) and t.is_contiguous()
        assert t.tolist() == want[f], f
    assert got.block_tables.shape == (S, width)


@pytest.mark.parametrize("backend", BACKENDS)
@pytest.mark.parametrize("S", [1, 2, 7, 255, 256, 257, 600])
@pytest.mark.parametrize("most_cached,most_fresh,page", [(0, 1, 16), (300, 1, 256), (100, 40, 16), (50, 9, 1), (64, 64, 48), (5000, 0, 7)])
def test_against_loops(backend, S, most_cached, most_fresh, page):
    (pages, cached, fresh), g = case(S, most_cached, most_fresh, page, S + page)
    width = max(1, max(-(-(c + f) // page) for c, f in zip(cached, fresh)) + S % 3)
    tokens = sum(fresh) + S % 4
    shift, adapter = (torch.randint(-9, 9, (S,), generator=g).tolist() for _ in range(2))
    got = call(backend[0], pages, cached, fresh, page=page, tokens=tokens, width=width, shift=shift, adapter=adapter)
    same(got, plain(pages, cached, fresh, page, tokens, width, None, shift, adapter), S, width)
    got = call(backend[0], pages, cached, fresh, page=page, tokens=tokens, width=width)
    same(got, plain(pages, cached, fresh, page, tokens, width), S, width, adapter=False)


@pytest.mark.parametrize("backend", BACKENDS)
def test_reserved_pages(backend):
    """Requests that own more pages than their tokens need, in another order than the requests."""
    pages, cached, fresh, bounds = list(range(100, 120)), [5, 0, 16], [3, 0, 1], [2, 5, 5, 20]
    got = call(backend[0], pages, cached, fresh, page=4, tokens=4, width=6, page_offsets=bounds)
    same(got, plain(pages, cached, fresh, 4, 4, 6, bounds), 3, 6, adapter=False)


@pytest.mark.parametrize("backend", BACKENDS)
def test_empty_steps(backend):
    got = call(backend[0], [], [], [], page=16, tokens=3, width=2)
    same(got, plain([], [], [], 16, 3, 2), 0, 2, adapter=False)
    got = call(backend[0], [], [0, 0], [0, 0], page=16, tokens=0, width=1)
    same(got, plain([], [0, 0], [0, 0], 16, 0, 1), 2, 1, adapter=False)


@pytest.mark.parametrize("backend", BACKENDS)
def test_slots_past_32_bits(backend):
    """Page ids whose slots need 64 bits; a page that was given up (-1) holds no slot."""
    got = call(backend[0], [2 ** 31 - 1, -1], [254], [4], page=256, tokens=4, width=2)
    assert got.slots.tolist() == [(2 ** 31 - 1) * 256 + 254, (2 ** 31 - 1) * 256 + 255, -1, -1]


@pytest.mark.parametrize("backend", BACKENDS)
def test_many_requests(backend):
    S = batch.MAX_REQUESTS
    (pages, cached, fresh), _ = case(S, 30, 3, 16, 1)
    got = call(backend[0], pages, cached, fresh, page=16, tokens=sum(fresh), width=4)
    same(got, plain(pages, cached, fresh, 16, sum(fresh), 4), S, 4, adapter=False)


@pytest.mark.gpu
def test_a_graph_replays_with_new_lengths():
    lengths = [torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, 1, 2, 3, 4, 5, 6, 7], [7, 20, 3], [1, 1, 1])]
    pages, cached, fresh = lengths
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = batch.step_maps(pages, cached, fresh, page=8, tokens=5, width=4)
    for step in ([1, 1, 1], [1, 0, 2], [0, 0, 0], [2, 2, 1]):
        fresh.copy_(torch.tensor(step))
        graph.replay()
        same(got, plain(pages.tolist(), cached.tolist(), step, 8, 5, 4), 3, 4, adapter=False)
        cached.copy_(got.kv_lens)       # the next step's lengths, without the host
    native.check_status()


@pytest.mark.gpu
def test_contradictions_are_reported_and_stay_inside_the_buffers():
    def wrong(*args, **kw):
        native.read_status()
        got = call("cuda:0", *args, **kw)
        assert native.read_status()["batch"][0] == 3
        return got

    got = wrong([4, 5], [3, 0], [2, 3], page=4, tokens=3, width=2)          # five tokens for three rows, three pages of two
    assert got.slots.tolist() == [19, 20, -1] and got.cu_seqlens_q.tolist() == [0, 2, 3] and got.sample_rows.tolist() == [1, -1]
    got = wrong([4, 5], [-1, 3], [2, 1], page=4, tokens=4, width=1)         # a negative length
    assert got.kv_lens.tolist() == [0, 4] and got.slots.tolist() == [19, -1, -1, -1] and got.block_tables.tolist() == [[-1], [4]]
    got = wrong([4, 5], [2 ** 31 - 1], [1], page=4, tokens=1, width=1)      # a length past 31 bits
    assert got.kv_lens.tolist() == [0] and got.slots.tolist() == [-1]
    got = wrong([4, 5], [0], [8], page=4, tokens=8, width=1)                # a table too narrow
    assert got.block_tables.tolist() == [[4]] and got.slots.tolist() == list(range(16, 24))
    for bounds in ([0, 3], [-1, 2], [2, 1]):                                # pages outside the list
        got = wrong([4, 5], [0], [1], page=4, tokens=1, width=1, page_offsets=bounds)
        assert got.block_tables.tolist() == [[-1]] and got.slots.tolist() == [-1]
    got = wrong([4], [2 ** 31 - 2, 2 ** 31 - 2], [0, 0], page=2 ** 30, tokens=1, width=4)
    assert got.cu_seqlens_kv.tolist() == [0, 2 ** 31 - 2, 2 ** 31 - 1]


@pytest.mark.parametrize("backend", BACKENDS)
def test_refusals(backend):
    dev = backend[0]
    ok = dict(page=16, tokens=2, width=1)

    def refused(*args, **kw):
        with pytest.raises(ValueError):
            batch.step_maps(*args, **kw)

    i = lambda v, **k: torch.tensor(v, dtype=torch.int32, device=dev, **k)  # noqa: E731
    refused(i([1]), i([0]), i([1, 1]), **ok)
    refused(i([1]), i([0]).long(), i([1]), **ok)
    refused(i([[1]]), i([0]), i([1]), **ok)
    refused(i([1, 2, 3])[::2], i([0]), i([1]), **ok)
    refused(i([1]), i(0), i(1), **ok)
    for bad in (dict(page=0), dict(width=0), dict(tokens=-1), dict(page=2 ** 31), dict(tokens=2 ** 30 + 1), dict(width=2 ** 30 + 1)):
        refused(i([1]), i([0]), i([1]), **{**ok, **bad})
    for bad in (dict(page_offsets=i([0])), dict(shift=i([0, 0])), dict(adapter=i([0]).long())):
        refused(i([1]), i([0]), i([1]), **ok, **bad)
    S = batch.MAX_REQUESTS + 1
    refused(i([]), i([0] * S), i([0] * S), **ok)
    if dev == "cpu":
        refused(i([1]), i([-1]), i([1]), **ok)
        refused(i([1]), i([0]), i([3]), **ok)
        refused(i([1]), i([16]), i([1]), **ok)
        refused(i([1]), i([16]), i([1]), page=16, tokens=1, width=2)
        refused(i([1]), i([0]), i([1]), **ok, page_offsets=i([0, 2]))
