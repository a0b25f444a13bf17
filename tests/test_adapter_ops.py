"""Projections with low-rank adapters against the plain statement in 64 bits.  CPU statements, and the kernels on a B200."""

import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from op_helpers import CPU, GPU16, GPU32, rand  # noqa: E402

from prism_infer_b200 import ops  # noqa: E402
from prism_infer_b200.ops import adapters, batch, native  # noqa: E402

BACKENDS = [CPU, GPU32, GPU16]
GPU = [GPU32, GPU16]


class Problem:
    """Operands that every type holds exactly, kept on the CPU, and the pool, weights and plan on a backend."""

    def __init__(self, backend, T, K, sections, rank, slots, who, seed=0, bias=False, scale=1.0):
        device, dtype = backend
        self.device, self.dtype, self.sections = device, dtype, sections
        n = len(sections)
        self.x = rand(T, K, seed=seed, scale=scale)
        self.w = rand(sum(sections), K, seed=seed + 1, scale=K ** -0.5)
        self.a = rand(slots, n, rank, K, seed=seed + 2, scale=K ** -0.5)
        self.b = [rand(slots, m, rank, seed=seed + 3 + i, scale=0.5 * rank ** -0.5) for i, m in enumerate(sections)]
        self.scale = [(1.0, 2.0, 0.5)[s % 3] for s in range(slots)]
        self.bias = rand(sum(sections), seed=seed + 20) if bias else None
        self.who = torch.as_tensor(who, dtype=torch.int32)
        self.pool = adapters.AdapterPool(slots, rank, K, sections, device=device, dtype=dtype)
        for s in range(slots):
            self.pool.load(s, list(self.a[s]), [b[s] for b in self.b], self.scale[s])
        self.plan = adapters.plan(self.who.to(device), slots)

    def to(self, t):
        return None if t is None else t.to(self.device, self.dtype)

    def run(self, **kw):
        return adapters.linear(self.to(self.x), self.to(self.w), self.pool, self.plan, bias=self.to(self.bias), **kw)

    def exact(self):
        """(value, bound on the error of sums in 32 bits with the low-rank products rounded to the type), both [T, M] in 64 bits.

        A sum of n products in 32 bits, in any order and truncated at each step, is off by at most n 2^-23 of the sum of their
        magnitudes; a bf16 operand is off by 2^-8 of its value, and so is the result."""
        x, w, u = self.x.double(), self.w.double(), 2.0 ** -8 if self.dtype == torch.bfloat16 else 2.0 ** -23
        K, f = x.shape[1], 2.0 ** -23
        y, err = x @ w.T, (K + 8) * f * (x.abs() @ w.abs().T)
        first = 0
        for i, m in enumerate(self.sections):
            for t, s in enumerate(self.who.tolist()):
                if s < 0:
                    continue
                a, b = self.a[s, i].double(), self.b[i][s].double()
                low, low_abs = self.scale[s] * (a @ x[t]), self.scale[s] * (a.abs() @ x[t].abs())
                y[t, first:first + m] += b @ low
                err[t, first:first + m] += b.abs() @ (u * low.abs() + (K + len(low) + 16) * f * low_abs) * 1.01
            first += m
        if self.bias is not None:
            y += self.bias.double()
        err += 8 * f * y.abs()
        return y, err

    def check(self, got, y=None, err=None):
        if y is None:
            y, err = self.exact()
        last = 2.0 ** -8 if self.dtype == torch.bfloat16 else 2.0 ** -24
        assert got.dtype == self.dtype and got.shape == y.shape
        off = (got.double().cpu() - y).abs() - (err * 1.01 + last * (y.abs() + err) + 1e-30)
        assert float(off.max()) <= 0, (float(off.max()), (off > 0).nonzero()[:5].tolist())


def mixed(T, slots, seed=1, bare=0.2):
    g = torch.Generator().manual_seed(seed)
    who = torch.randint(0, slots, (T,), generator=g, dtype=torch.int32)
    return torch.where(torch.rand(T, generator=g) < bare, -1, who)


@pytest.mark.parametrize("backend", BACKENDS)
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 33, 64, 65, 127, 128, 129, 200, 256, 257, 300, 513])
@pytest.mark.parametrize("K,sections,rank,slots", [(64, (128,), 16, 4), (200, (96, 40, 24), 5, 9), (8, (1,), 1, 1), (1000, (272, 16), 33, 3)])
def test_tokens_with_adapters_in_any_order(backend, T, K, sections, rank, slots):
    p = Problem(backend, T, K, sections, rank, slots, mixed(T, slots), bias=T % 2 == 0)
    p.check(p.run())


@pytest.mark.parametrize("backend", BACKENDS)
@pytest.mark.parametrize("T,K,sections,rank,slots", [
    (128, 320, (256,), 16, 128),            # every token an adapter of its own
    (256, 128, (144,), 16, 256),            # and a whole tile of them
    (400, 264, (64, 64), 64, 300),          # more slots than a tile has tokens
    (130, 4096, (512,), 64, 2),             # a long sum
    (40, 2048, (1024, 256, 256), 24, 20),
])
def test_many_adapters(backend, T, K, sections, rank, slots):
    order = torch.randperm(slots, generator=torch.Generator().manual_seed(3)).int()
    p = Problem(backend, T, K, sections, rank, slots, order.repeat(-(-T // slots))[:T])
    p.check(p.run())


@pytest.mark.parametrize("backend", BACKENDS)
@pytest.mark.parametrize("T", [1, 40, 300])
def test_steps_without_adapters(backend, T):
    """Nobody has one; loaded and empty slots beside each other; slots cleared again."""
    p = Problem(backend, T, 96, (48, 32), 8, 5, [-1] * T, bias=True)
    plain = p.run()
    p.check(plain)
    p.pool.clear(3)
    p.plan = adapters.plan(torch.full((T,), 3, dtype=torch.int32, device=p.device), 5)
    assert torch.equal(p.run(), plain)


@pytest.mark.parametrize("backend", BACKENDS)
def test_ranks_and_reloading(backend):
    """A slot loaded with a smaller rank than before keeps nothing of the one before."""
    p = Problem(backend, 20, 64, (32, 32), 20, 2, mixed(20, 2))
    p.run()
    p.a, p.b = p.a[:, :, :3], [b[:, :, :3] for b in p.b]
    for s in range(2):
        p.pool.load(s, list(p.a[s]), [b[s] for b in p.b], p.scale[s])
    p.check(p.run())


@pytest.mark.parametrize("backend", BACKENDS)
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("T,K,half,rank,slots", [(1, 64, 64, 16, 2), (7, 200, 40, 5, 3), (128, 136, 96, 16, 128), (130, 64, 80, 40, 7), (300, 512, 256, 16, 5),
                                                 (33, 72, 13, 4, 2), (300, 72, 13, 4, 2)])
def test_gated_unit(backend, act, T, K, half, rank, slots):
    p = Problem(backend, T, K, (half, half), rank, slots, mixed(T, slots))
    got = adapters.gate_up_glu(p.to(p.x), p.to(p.w), p.pool, p.plan, act)
    y, err = p.exact()
    g, u, eg, eu = y[:, :half], y[:, half:], err[:, :half], err[:, half:]
    unit = torch.nn.functional.silu(g) if act == "silu" else torch.nn.functional.gelu(g, approximate="tanh")
    # both activations have slopes of at most 1.13; in bf16 their exponentials and hyperbolic tangent are approximate: 2^-10 of the unit's scale
    fast = 2.0 ** -10 if p.dtype == torch.bfloat16 else 2.0 ** -10 if act == "gelu_tanh" and p.device != "cpu" else 2.0 ** -20
    bound = 1.13 * eg * (u.abs() + eu) + (unit.abs() + 1.13 * eg) * eu + fast * (g.abs() + eg) * (u.abs() + eu)
    p.check(got, unit * u, bound)


@pytest.mark.parametrize("backend", GPU)
def test_strided_operands_and_output(backend):
    """Rows of a wider buffer; columns beside the output stay as they were."""
    for T in (9, 200):
        p = Problem(backend, T, 64, (48,), 8, 3, mixed(T, 3), bias=True)
        x = torch.full((T, 96), 7.0, dtype=p.dtype, device=p.device)
        x[:, 16:80] = p.to(p.x)
        w = torch.full((48, 128), 7.0, dtype=p.dtype, device=p.device)
        w[:, 64:] = p.to(p.w)
        for left, width in ((8, 64), (3, 53)):
            out = torch.full((T + 2, width), 5.0, dtype=p.dtype, device=p.device)
            got = adapters.linear(x[:, 16:80], w[:, 64:], p.pool, p.plan, bias=p.to(p.bias), out=out[1:T + 1, left:left + 48])
            p.check(got)
            out[1:T + 1, left:left + 48] = 5.0
            assert bool((out == 5.0).all())


@pytest.mark.parametrize("backend", GPU)
@pytest.mark.parametrize("T", [6, 300])
def test_rows_do_not_meet(backend, T):
    """A row that is infinite or not a number leaves the other rows as they are."""
    p = Problem(backend, T, 128, (64,), 16, 4, mixed(T, 4, bare=0.3))
    clean = p.run().clone()
    bad = torch.tensor([1, T // 2])
    p.x[bad[0], 3], p.x[bad[1]] = float("inf"), float("nan")
    got = p.run()
    keep = torch.ones(T, dtype=torch.bool)
    keep[bad] = False
    assert torch.equal(got[keep.to(got.device)], clean[keep.to(got.device)])
    assert not bool(torch.isfinite(got[bad.to(got.device)]).any())


@pytest.mark.parametrize("backend", GPU)
@pytest.mark.parametrize("T", [5, 128, 300])
def test_repeated_calls_and_graph_replays_agree(backend, T):
    """Bit for bit, on another stream too; a replay reads new activations, adapters and plans."""
    p = Problem(backend, T, 256, (96, 32), 16, 6, mixed(T, 6))
    want = p.run().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = p.run()
    side.synchronize()
    assert torch.equal(again, want)
    x, w, who = p.to(p.x), p.to(p.w), p.who.to(p.device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = adapters.plan(who, 6)
        y = adapters.linear(x, w, p.pool, plan)
    graph.replay()
    assert torch.equal(y, want)
    q = Problem(backend, T, 256, (96, 32), 16, 6, mixed(T, 6, seed=5), seed=40)
    x.copy_(q.to(q.x)), w.copy_(q.to(q.w)), who.copy_(q.who)
    for s in range(6):
        p.pool.load(s, list(q.a[s]), [b[s] for b in q.b], q.scale[s])
    graph.replay()
    q.check(y)
    native.check_status()


@pytest.mark.parametrize("backend", GPU)
def test_calls_on_two_streams_at_once(backend):
    a, b = (Problem(backend, T, 512, (256,), 16, 8, mixed(T, 8), seed=T) for T in (64, 300))
    want = a.run().clone(), b.run().clone()
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    got = [], []
    for _ in range(10):
        for i, p in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(p.run())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


@pytest.mark.parametrize("backend", GPU)
@pytest.mark.parametrize("T", [40, 300])
def test_one_pool_on_two_streams_at_once(backend, T):
    p, q = (Problem(backend, T, 512, (256,), 16, 8, mixed(T, 8), seed=3, scale=s) for s in (1.0, 2.0))
    q.pool = p.pool
    want = p.run().clone(), q.run().clone()
    torch.cuda.synchronize()
    streams, got = (torch.cuda.Stream(), torch.cuda.Stream()), ([], [])
    for _ in range(10):
        for i, r in enumerate((p, q)):
            with torch.cuda.stream(streams[i]):
                got[i].append(r.run())
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


@pytest.mark.parametrize("backend", GPU)
@pytest.mark.parametrize("T", [12, 128, 300])
def test_overlapped_launches_agree(backend, T):
    """Programmatic launches of every kernel: the plan, two projections that read one another's results, bit for bit."""
    p = Problem(backend, T, 256, (256,), 16, 6, mixed(T, 6))
    x, w, who = p.to(p.x), p.to(p.w), p.who.to(p.device)

    def chain():
        y = x
        for _ in range(6):
            y = adapters.linear(y, w, p.pool, adapters.plan(who, 6)) * 0.5
            y = adapters.linear(y, w, p.pool, adapters.plan(who, 6))
        return y

    want = chain().clone()
    ops.set_pdl(True)
    try:
        got = [chain() for _ in range(5)]
    finally:
        ops.set_pdl(False)
    assert all(torch.equal(g, want) for g in got)
    native.check_status()


@pytest.mark.parametrize("backend", BACKENDS)
@pytest.mark.parametrize("T", [3, 40, 200])
def test_large_ranks_and_all_sections(backend, T):
    p = Problem(backend, T, 192, (24, 8, 40, 16, 32, 8, 64, 16), 40, 3, mixed(T, 3))
    p.check(p.run())
    p = Problem(backend, T, 64, (48, 48), 250, 3, mixed(T, 3), scale=0.25)
    p.check(p.run())


@pytest.mark.parametrize("backend", GPU)
@pytest.mark.parametrize("T", [257, 300, 640, 1000])
def test_steps_that_run_in_pieces(backend, T, monkeypatch):
    """Low-rank rows that would pass their limit: a tile at a time, with bits as in one launch where the pieces' kernels are the same."""
    p = Problem(backend, T, 128, (96, 32), 16, 40, mixed(T, 40), bias=True)
    monkeypatch.setattr(adapters, "MAX_LOW_BYTES", 1)
    out = torch.full((T, 160), 3.0, dtype=p.dtype, device=p.device)
    p.check(p.run(out=out[:, 16:144]))
    assert bool((out[:, :16] == 3.0).all()) and bool((out[:, 144:] == 3.0).all())


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
def test_odd_rows_in_32_bits(device):
    """Widths and strides that no vector load fits."""
    for T in (5, 70):
        p = Problem((device, torch.float32), T, 37, (13, 6), 3, 4, mixed(T, 4), bias=True)
        wide = torch.full((T, 39), 7.0, device=device)
        wide[:, 1:38] = p.to(p.x)
        p.check(adapters.linear(wide[:, 1:38], p.to(p.w), p.pool, p.plan, bias=p.to(p.bias)))


@pytest.mark.parametrize("backend", BACKENDS)
def test_factors_that_require_gradients_are_copied(backend):
    p = Problem(backend, 4, 64, (32,), 8, 2, [0, 1, -1, 0])
    a, b = torch.randn(8, 64, requires_grad=True), torch.randn(32, 8, requires_grad=True)
    p.pool.load(1, a, b)
    assert not p.pool.a.requires_grad and not p.run().requires_grad


def plan_of(who, slots):
    index, lists, counts = [], [], []
    for lo in range(0, len(who), 256):
        here = sorted({w for w in who[lo:lo + 256] if w >= 0})
        index += [here.index(w) if w >= 0 else -1 for w in who[lo:lo + 256]]
        lists.append(here + [-1] * (min(slots, 256, len(who)) - len(here)))
        counts.append(len(here))
    return index, lists, counts


@pytest.mark.parametrize("backend", [CPU, GPU32])
@pytest.mark.parametrize("T", [1, 31, 256, 257, 1000])
@pytest.mark.parametrize("slots", [1, 2, 32, 33, 300, 8192])
def test_plan(backend, T, slots):
    for bare in (0.0, 0.3, 1.0):
        who = mixed(T, slots, seed=T + slots, bare=bare)
        p = adapters.plan(who.to(backend[0]), slots)
        assert (p.index.tolist(), p.lists.tolist(), p.counts.tolist()) == plan_of(who.tolist(), slots)


@pytest.mark.parametrize("backend", BACKENDS)
def test_no_tokens(backend):
    p = Problem(backend, 0, 64, (32, 32), 8, 2, [])
    assert p.run().shape == (0, 64)
    assert adapters.gate_up_glu(p.to(p.x), p.to(p.w), p.pool, p.plan, "silu").shape == (0, 32)


@pytest.mark.gpu
def test_slots_out_of_range_count_as_none_and_are_reported():
    p = Problem(("cuda:0", torch.bfloat16), 10, 64, (32,), 8, 2, [0, 1] * 5)
    native.read_status()
    plan = adapters.plan(torch.tensor([0, 1, 2, -7, 2 ** 31 - 1, 1, 0, 1, 0, 1], dtype=torch.int32, device="cuda"), 2)
    assert plan.index.tolist() == [0, 1, -1, -1, -1, 1, 0, 1, 0, 1]
    assert native.read_status()["adapters"][0] == 3
    p.plan, p.who[2:5] = plan, -1
    p.check(p.run())


@pytest.mark.gpu
def test_tensors_of_another_device_than_the_current_one_are_refused(monkeypatch):
    p = Problem(("cuda:0", torch.bfloat16), 4, 64, (32,), 8, 2, [0, 1, -1, 0])
    lengths = torch.ones(1, dtype=torch.int32, device="cuda:0")
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    for call in (p.run, lambda: adapters.plan(p.plan.adapter, 2), lambda: batch.step_maps(lengths, lengths, lengths, page=16, tokens=1, width=1)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("backend", BACKENDS)
def test_refusals(backend):
    device, dtype = backend
    p = Problem(backend, 4, 64, (32, 32), 8, 2, [0, 1, -1, 0])
    x, w = p.to(p.x), p.to(p.w)

    def refused(call, *args, **kw):
        with pytest.raises(ValueError):
            call(*args, **kw)

    refused(adapters.linear, x[:, :32], w, p.pool, p.plan)
    refused(adapters.linear, x[:3], w, p.pool, p.plan)
    refused(adapters.linear, x, w[:32], p.pool, p.plan)
    refused(adapters.linear, x.double(), w, p.pool, p.plan)
    refused(adapters.linear, x.t().contiguous().t(), w, p.pool, p.plan)
    refused(adapters.linear, x, w, p.pool, p.plan, bias=w[0, :32])
    refused(adapters.linear, x, w, p.pool, p.plan, out=torch.empty(4, 63, dtype=dtype, device=device))
    refused(adapters.linear, x, w, p.pool, adapters.plan(p.who.to(device), 3))
    refused(adapters.linear, x[:1].expand(4, 64), w, p.pool, p.plan)
    if dtype == torch.bfloat16:
        refused(adapters.linear, torch.zeros(4 * 64 + 8, dtype=dtype, device=device)[1:257].view(4, 64), w, p.pool, p.plan)
        refused(adapters.AdapterPool, 2, 8, 60, 32, device=device)
    refused(adapters.gate_up_glu, x, w, p.pool, p.plan, "relu")
    refused(adapters.gate_up_glu, x, w, adapters.AdapterPool(2, 8, 64, (16, 48), device=device, dtype=dtype), p.plan, "silu")
    refused(adapters.plan, p.who.long().to(device), 2)
    refused(adapters.plan, p.who.to(device), 0)
    refused(adapters.plan, p.who.to(device), 8193)
    refused(adapters.AdapterPool, 0, 8, 64, 32, device=device)
    refused(adapters.AdapterPool, 2, 257, 64, 32, device=device)
    refused(adapters.AdapterPool, 2, 8, 64, (), device=device)
    refused(adapters.AdapterPool, 2, 8, 64, 32, device=device, dtype=torch.float16)
    pool = adapters.AdapterPool(2, 8, 64, 32, device=device, dtype=dtype)
    a, b = torch.ones(8, 64), torch.ones(32, 8)
    refused(pool.load, 2, a, b)
    refused(pool.load, 0, a, b[:, :7])
    refused(pool.load, 0, a, b[:31])
    refused(pool.load, 0, [a, a], [b, b])
    refused(pool.load, 0, torch.ones(9, 64), torch.ones(32, 9))
    refused(pool.load, 0, a, b, float("nan"))
    refused(pool.load, 0, a, b * float("inf"))
    refused(pool.load, 0, a * 1e39, b)
    refused(pool.load, 0, a, b, 1e39)
    refused(pool.clear, -1)
    if device == "cpu":
        refused(adapters.plan, torch.tensor([2], dtype=torch.int32), 2)


@pytest.mark.parametrize("backend", BACKENDS)
@pytest.mark.parametrize("T", [3, 40, 200, 300])
def test_infinite_rows_meet_the_ranks_of_their_own_adapter_only(backend, T):
    """Slots are padded to the pool's rank.  Padding times infinity is no number, and takes no part: a row with an infinite value gets what
    its adapter's own ranks make of it, and an empty slot adds nothing to it."""
    ranks = [(20, 20), (3, 17), (16, 1)]                 # of three slots, by section; the fourth stays empty
    p = Problem(backend, T, 64, (40, 24), 20, 4, torch.arange(T, dtype=torch.int32) % 5 - 1)
    p.pool.clear(3)
    p.a, p.w = p.a.abs() + 2.0 ** -6, p.w.abs() + 2.0 ** -6
    p.b = [b.abs() + 2.0 ** -6 for b in p.b]
    p.a, p.w, p.b = p.a.bfloat16().float(), p.w.bfloat16().float(), [b.bfloat16().float() for b in p.b]
    for s in range(4):
        for i in range(2):
            own = ranks[s][i] if s < 3 else 0
            p.a[s, i, own:], p.b[i][s, :, own:] = 0, 0
        if s < 3:
            p.pool.load(s, [p.a[s, i, :r] for i, r in enumerate(ranks[s])], [p.b[i][s, :, :r] for i, r in enumerate(ranks[s])], p.scale[s])
    bad = torch.arange(T) % 7 < 5 if T > 3 else torch.tensor([True, False, True])
    clean = p.run().clone()
    p.check(clean)
    p.x[bad, 9] = float("inf")                           # every weight and factor that it meets is positive
    got = p.run()
    assert torch.equal(got[~bad.to(got.device)], clean[~bad.to(got.device)])
    assert bool((got[bad.to(got.device)] == float("inf")).all())


@pytest.mark.parametrize("backend", BACKENDS)
@pytest.mark.parametrize("T", [3, 200, 300])
def test_infinite_rows_of_empty_slots_in_a_gated_unit(backend, T):
    p = Problem(backend, T, 64, (32, 32), 8, 2, torch.arange(T, dtype=torch.int32) % 3 - 1)
    p.pool.clear(1)
    p.x[::2, 5] = float("inf")
    p.x[1::4, 6] = float("nan")
    got = adapters.gate_up_glu(p.to(p.x), p.to(p.w), p.pool, p.plan, "silu")
    none = adapters.plan(torch.full((T,), -1, dtype=torch.int32, device=p.device), 2)
    want = adapters.gate_up_glu(p.to(p.x), p.to(p.w), p.pool, none, "silu")
    empty = (p.who != 0).to(got.device)
    assert torch.equal(got[empty].isnan(), want[empty].isnan())
    assert torch.equal(got[empty].nan_to_num(nan=0.5), want[empty].nan_to_num(nan=0.5))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,features", [(torch.bfloat16, 1), (torch.bfloat16, 16), (torch.float32, 1)])
def test_more_tokens_than_a_grid_has_rows_of_tiles(dtype, features):
    """65535 blocks of 128 tokens and one token more.  Whole numbers small enough that every sum and product is exact."""
    T = 65535 * 128 + 1
    g = torch.Generator("cuda").manual_seed(5)

    def whole(*shape, most):
        return torch.randint(-most, most + 1, shape, generator=g, device="cuda", dtype=torch.int8).to(dtype)

    x, w, a, b = whole(T, 8, most=2), whole(features, 8, most=2), whole(3, 8, most=1), whole(features, 3, most=1)
    pool = adapters.AdapterPool(1, 3, 8, features, device="cuda", dtype=dtype)
    pool.load(0, a, b)
    who = torch.randint(-1, 1, (T,), generator=g, device="cuda", dtype=torch.int32)
    got = adapters.linear(x, w, pool, adapters.plan(who, 1))
    low = x.float() @ a.float().T * (who >= 0)[:, None]
    assert torch.equal(got.float(), x.float() @ w.float().T + low @ b.float().T)
    native.check_status()


@pytest.mark.parametrize("backend", [CPU, GPU32])
def test_a_single_input_feature_has_any_stride(backend):
    """Strides of an axis of one element mean nothing."""
    p = Problem(backend, 5, 1, (6,), 2, 2, [0, 1, -1, 0, 1])
    x, w = p.to(p.x).reshape(1, 5).t(), p.to(p.w).reshape(1, 6).t()
    assert x.stride() == (1, 5) and x.is_contiguous() and w.stride() == (1, 6)
    p.check(adapters.linear(x, w, p.pool, p.plan))


@pytest.mark.parametrize("backend", [CPU, GPU32])
@pytest.mark.parametrize("T,K,half,rank,slots", [(1, 64, 64, 16, 2), (7, 200, 40, 5, 3), (128, 136, 96, 16, 128), (300, 512, 256, 16, 5), (33, 72, 13, 4, 2)])
def test_gelu_of_a_gated_unit_in_32_bits(backend, T, K, half, rank, slots):
    """tanhf, not its approximation: 2^-20 of the unit's scale is sixteen roundings, the approximation is off by 2^-11."""
    p = Problem(backend, T, K, (half, half), rank, slots, mixed(T, slots))
    got = adapters.gate_up_glu(p.to(p.x), p.to(p.w), p.pool, p.plan, "gelu_tanh")
    y, err = p.exact()
    g, u, eg, eu = y[:, :half], y[:, half:], err[:, :half], err[:, half:]
    unit = torch.nn.functional.gelu(g, approximate="tanh")
    p.check(got, unit * u, 1.13 * eg * (u.abs() + eu) + (unit.abs() + 1.13 * eg) * eu + 2.0 ** -20 * (g.abs() + eg) * (u.abs() + eu))


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
def test_pieces_of_two_tiles_have_the_bits_of_one_launch(gated, monkeypatch):
    """Runs of two tiles of 256 tokens and a shorter one, all of them prompts on pairs of SMs, against the call in one piece; tokens and
    outputs are columns of wider buffers."""
    T, sections = 1200, (128, 128)
    p = Problem(("cuda:0", torch.bfloat16), T, 128, sections, 16, 8, mixed(T, 8), bias=not gated)
    x = torch.full((T, 160), 7.0, dtype=p.dtype, device=p.device)
    x[:, 16:144] = p.to(p.x)
    M = 128 if gated else 256

    def call():
        out = torch.full((T, M + 32), 3.0, dtype=p.dtype, device=p.device)
        if gated:
            adapters.gate_up_glu(x[:, 16:144], p.to(p.w), p.pool, p.plan, "silu", out=out[:, 16:16 + M])
        else:
            adapters.linear(x[:, 16:144], p.to(p.w), p.pool, p.plan, bias=p.to(p.bias), out=out[:, 16:16 + M])
        assert bool((out[:, :16] == 3.0).all()) and bool((out[:, 16 + M:] == 3.0).all())
        return out[:, 16:16 + M]

    want, calls, launch = call(), [], native.call
    if not gated:
        p.check(want)
    per_tile = 2 * p.plan.lists.shape[1] * p.pool.low * adapters.TILE_TOKENS
    monkeypatch.setattr(adapters, "MAX_LOW_BYTES", 2 * per_tile + 5)
    monkeypatch.setattr(native, "call", lambda name, *args: (calls.append(name), launch(name, *args))[1])
    assert torch.equal(call(), want)
    assert calls == ["prism_adapter_linear"] * 3


@pytest.mark.parametrize("backend", GPU)
@pytest.mark.parametrize("T", [6, 150, 256, 300])
def test_rows_of_a_gated_unit_do_not_meet(backend, T):
    """A row that is infinite or not a number leaves the other rows as they are: decode tiles, two of them, pairs of SMs."""
    p = Problem(backend, T, 128, (64, 64), 16, 24, mixed(T, 24, bare=0.3))

    def run():
        return adapters.gate_up_glu(p.to(p.x), p.to(p.w), p.pool, p.plan, "gelu_tanh"), p.run()

    clean = run()
    bad = torch.tensor([1, T // 2, T - 1])
    p.x[1, 3], p.x[T // 2], p.x[T - 1, 7] = float("inf"), float("nan"), float("-inf")
    keep = torch.ones(T, dtype=torch.bool)
    keep[bad] = False
    for got, want in zip(run(), clean):
        assert torch.equal(got[keep.to(got.device)], want[keep.to(got.device)])
    assert bool(got[T // 2].isnan().all())
