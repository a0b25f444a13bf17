"""Timed cases of the step maps and of the projections with low-rank adapters.

A case is one call as a server makes it: the maps of a step (block tables, cache slots, positions, adapters) from the lengths of its
requests, or one stacked projection (or gated unit) of a step whose requests bring adapters of their own.  ``tokens`` counts the new
tokens of all ``requests``; a decode step has one token per request, a prompt step runs of different lengths, no two alike, unless it
has one request.  Request ``i`` uses adapter ``i % adapters`` of the ``slots`` loaded ones, every eighth request uses none
(``bare``).  ``out`` names the features of the stacked matrices, each with low-rank factors of its own.
"""

import math

import torch

own = False
DEV = "cuda"
PHI = 0.6180339887


def listed():
    def maps(name, requests, fresh, history, page, adapters=8):
        return dict(name=name, op="maps", requests=requests, fresh=fresh, history=history, page=page, slots=64, adapters=adapters, bare=True)

    def linear(name, requests, tokens, width, out, rank, *, op="linear", slots=64, adapters=16, bare=True, bias=False, dtype="bf16"):
        return dict(name=name, op=op, requests=requests, tokens=tokens, width=width, out=out, rank=rank, slots=slots, adapters=adapters,
                    bare=bare, bias=bias, dtype=dtype)

    return [
        # the smallest call: one user's decode step over a short conversation; a launch and its latency
        maps("maps decode 1", 1, 1, 332, 256, adapters=1),
        # a full decode batch over long conversations, the cache's default pages
        maps("maps decode 128", 128, 1, 16384, 256),
        # a throughput server's step: many requests in small pages, wide tables, a few new tokens for each
        maps("maps mixed 1024, pages of 16", 1024, 31, 8192, 16),
        # the attention output of a small model for one user with one adapter
        linear("linear 1, width 2048", 1, 1, 2048, "2048", 16, adapters=1, bare=False),
        # query, key and value projections of a server under load
        linear("linear 32, qkv", 32, 32, 4096, "4096+1024+1024", 16),
        # the down projection of a full batch, every request with a large adapter of its own
        linear("linear 128, down", 128, 128, 12288, "4096", 64, adapters=128, slots=128, bare=False),
        # the headline request's prompt (1616 tokens) under one adapter
        linear("linear prompt 1616", 1, 1616, 4096, "4096", 16, adapters=1, bare=False),
        # a packed prompt step: requests of many tenants
        linear("linear prompts 24 of 8192, qkv", 24, 8192, 4096, "4096+1024+1024", 32, bias=True),
        # the 32-bit mode of the text families
        linear("linear 100 in 32 bits", 100, 100, 2048, "2048", 16, dtype="fp32"),
        # the feed-forward's gated unit in a decode step
        linear("gated 32", 32, 32, 4096, "12288+12288", 16, op="gated"),
        # and of a packed prompt step
        linear("gated prompts 5 of 2048", 5, 2048, 4096, "12288+12288", 16, op="gated"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["maps", "linear", "linear", "linear", "gated"])
    slots = log(1, 128)
    if op == "maps":
        requests = log(1, 1024)
        return dict(op=op, requests=requests, fresh=rng.choice([1, 1, log(2, 2048)]) if requests < 64 else rng.choice([1, log(2, 32)]),
                    history=log(1, 16384), page=rng.choice([1, 16, 48, 64, 256]) if requests < 64 else rng.choice([16, 24, 256]), slots=slots,
                    adapters=rng.randint(1, slots), bare=bool(rng.randint(0, 1)))
    width = 8 * log(32, 1536)
    grain = rng.choice([64, 64, 16, 16, 8, 1])
    parts = 2 if op == "gated" else rng.choice([1, 1, 2, 3])
    most = min(12288 // parts if op == "linear" else 12288, 4096 * 24576 // (width * parts))
    out = [max(grain, log(64, most) // grain * grain) for _ in range(parts)]
    if op == "gated":
        out = out[:1] * 2
    if rng.random() < 0.5:
        tokens = requests = log(1, 128)
    else:
        tokens = log(129, max(130, min(8192, 8192 * 4096 * 6144 // (width * sum(out)))))
        requests = log(1, min(64, tokens // 4))
    dtype = "fp32" if rng.random() < 0.15 else "bf16"
    if dtype == "fp32":
        tokens, requests = min(tokens, 700), min(tokens, requests)
    return dict(op=op, requests=requests, tokens=tokens, width=width, out="+".join(map(str, out)), rank=log(1, 64), slots=slots,
                adapters=rng.randint(1, slots), bare=bool(rng.randint(0, 1)), bias=bool(rng.randint(0, 1)) and op == "linear", dtype=dtype)


# ------------------------------------------------------------------------------------------------ inputs
def _lens(case):
    """(tokens in the cache, new tokens) of every request."""
    if case["op"] == "maps":
        share = [0.25 + 0.75 * ((i + 1) * PHI % 1.0) for i in range(case["requests"])]
        return [(int(case["history"] * s), max(1, round(case["fresh"] * s))) for s in share]
    n, total = case["requests"], case["tokens"]
    if n == total:
        return [(0, 1)] * n
    share = [0.25 + 0.75 * ((i + 1) * PHI % 1.0) for i in range(n)]
    ends = [round(total * sum(share[:i + 1]) / sum(share)) for i in range(n)]
    return [(0, b - a) for a, b in zip([0] + ends, ends)]


def _numbers(case):
    """The adapter of every request, counted from zero; -1: none."""
    return [-1 if case["bare"] and i % 8 == 7 else i % case["adapters"] for i in range(case["requests"])]


def _parts(case):
    return [int(p) for p in case["out"].split("+")]


def _dtype(case):
    return torch.float32 if case["dtype"] == "fp32" else torch.bfloat16


def _inputs(case, seed):
    g = torch.Generator(DEV).manual_seed(seed * 7919 + 11)
    i32 = dict(dtype=torch.int32, device=DEV)
    lens = _lens(case)
    order = torch.randperm(case["slots"], generator=g, device=DEV).tolist()     # where each adapter was loaded
    used = [-1 if n < 0 else order[n] for n in _numbers(case)]
    x = dict(case=case, lens=lens, used=used, adapter=torch.tensor(used, **i32))
    if case["op"] == "maps":
        page = case["page"]
        counts = [-(-(a + b) // page) for a, b in lens]
        x["pages"] = torch.randperm(sum(counts), generator=g, device=DEV).to(torch.int32)
        x["cached"], x["fresh"] = torch.tensor([a for a, _ in lens], **i32), torch.tensor([b for _, b in lens], **i32)
        # a third of the requests are conversations about images, whose positions run behind their tokens
        x["shift"] = -torch.randint(0, 200, (len(lens),), generator=g, **i32) * (torch.arange(len(lens), device=DEV) % 3 == 2).int()
        x["tokens"], x["width"] = sum(b for _, b in lens), max(counts)
        return x
    width, parts, rank, slots, dt = case["width"], _parts(case), case["rank"], case["slots"], _dtype(case)

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device=DEV).mul_(scale).to(dt)

    x["x"] = normal(case["tokens"], width)          # rows behind a norm
    x["x"][:, ::97] *= 6                            # and its few loud channels
    x["w"] = normal(sum(parts), width, scale=width ** -0.5)
    x["bias"] = normal(sum(parts), scale=0.3) if case["bias"] else None
    x["a"] = normal(slots, len(parts), rank, width, scale=width ** -0.5)
    x["b"] = [normal(slots, m, rank, scale=0.25 * rank ** -0.5) for m in parts]
    x["scale"] = [(1.0, 2.0, 0.5)[s % 3] for s in range(slots)]
    return x


def prepare(case, seed):
    st = _inputs(case, seed)
    if case["op"] != "maps":
        # what a step's maps hand on: the adapter of every token
        st["token_adapter"] = torch.repeat_interleave(st["adapter"], torch.tensor([n for _, n in st["lens"]], device=DEV))
        if own:
            from prism_infer_b200.ops import adapters
            pool = adapters.AdapterPool(case["slots"], case["rank"], case["width"], _parts(case), device=DEV, dtype=_dtype(case))
            for s in range(case["slots"]):
                pool.load(s, list(st["a"][s]), [b[s] for b in st["b"]], st["scale"][s])
            st["pool"], st["plan"] = pool, adapters.plan(st["token_adapter"], case["slots"])
        else:
            st["scales"] = torch.tensor(st["scale"], device=DEV)
    return st


# ------------------------------------------------------------------------------------------------ one pass
def run(st):
    case = st["case"]
    if own:
        from prism_infer_b200.ops import adapters, batch
        if case["op"] == "maps":
            m = batch.step_maps(st["pages"], st["cached"], st["fresh"], page=case["page"], tokens=st["tokens"], width=st["width"],
                                shift=st["shift"], adapter=st["adapter"])
            p = adapters.plan(m.token_adapter, case["slots"])
            return (m.block_tables, m.slots, m.positions, m.token_seq, m.token_adapter, m.cu_seqlens_q, m.cu_seqlens_kv, m.kv_lens,
                    m.sample_rows, p.index, p.lists, p.counts)
        if case["op"] == "gated":
            return adapters.gate_up_glu(st["x"], st["w"], st["pool"], st["plan"], "silu")
        return adapters.linear(st["x"], st["w"], st["pool"], st["plan"], bias=st["bias"])
    return _plain_maps(st) if case["op"] == "maps" else _plain_projection(st)


def _plain_maps(st):
    case = st["case"]
    page, tokens = case["page"], st["tokens"]
    pages, cached, fresh = st["pages"], st["cached"].long(), st["fresh"].long()
    kv = cached + fresh
    zero = kv.new_zeros(1)
    cu_q, cu_kv = torch.cat([zero, fresh.cumsum(0)]), torch.cat([zero, kv.cumsum(0)])
    counts = (kv + page - 1) // page
    start = counts.cumsum(0) - counts
    j = torch.arange(st["width"], device=DEV)
    table = torch.where(j < counts[:, None], pages[(start[:, None] + j).clamp_max(len(pages) - 1)].long(), -1)
    t = torch.arange(tokens, device=DEV)
    seq = torch.searchsorted(cu_q[1:], t, right=True)
    at = cached[seq] + t - cu_q[seq]
    slots = pages[start[seq] + at // page].long() * page + at % page
    positions = (at + st["shift"].long()[seq]).expand(3, -1)
    token_adapter = st["adapter"][seq]
    sample = torch.where(fresh > 0, cu_q[1:] - 1, -1)
    # adapters of every 256 tokens, ascending, and each token's place among them
    tiles, n = -(-tokens // 256), case["slots"]
    padded = torch.full((tiles * 256,), -1, device=DEV)
    padded[:tokens] = token_adapter.long()
    present = (padded.view(tiles, 256, 1) == torch.arange(n, device=DEV)).any(1)
    rank = present.long().cumsum(1) - 1
    capacity = min(n, 256, tokens)
    order = torch.where(present, torch.arange(n, device=DEV), n).sort(1).values[:, :capacity]
    lists = torch.where(order < n, order, -1)
    index = torch.where(padded >= 0, rank.gather(1, padded.view(tiles, 256).clamp_min(0)).view(-1), -1)[:tokens]
    i32 = torch.int32
    return (table.to(i32), slots, positions.to(i32).contiguous(), seq.to(i32), token_adapter, cu_q.to(i32), cu_kv.to(i32), kv.to(i32), sample,
            index.to(i32), lists.to(i32), present.sum(1).to(i32))


def _plain_projection(st):
    case = st["case"]
    parts, x = _parts(case), st["x"].float()
    y = x @ st["w"].float().T
    if st["bias"] is not None:
        y += st["bias"].float()
    first = 0
    for i, m in enumerate(parts):
        out = y[:, first:first + m]
        if case["tokens"] <= 128:       # every token with the factors of its own adapter
            who = st["token_adapter"].long()
            low = torch.bmm(st["a"][who.clamp_min(0), i].float(), x[:, :, None])
            low = torch.where(who[:, None, None] >= 0, low * st["scales"][who.clamp_min(0), None, None], 0.0)
            out += torch.bmm(st["b"][i][who.clamp_min(0)].float(), low)[:, :, 0]
        else:                           # request by request
            row = 0
            for (_, n), s in zip(st["lens"], st["used"]):
                if s >= 0:
                    out[row:row + n] += (x[row:row + n] @ st["a"][s, i].float().T * st["scales"][s]) @ st["b"][i][s].float().T
                row += n
        first += m
    if case["op"] == "gated":
        gate, up = y[:, :parts[0]], y[:, parts[0]:]
        y = gate / (1 + torch.exp(-gate)) * up
    return y.to(_dtype(case))


# ------------------------------------------------------------------------------------------------ definition in 64 bits
def exact(case, seed):
    x = _inputs(case, seed)
    return _exact_maps(x) if case["op"] == "maps" else _exact_projection(x)


def _exact_maps(x):
    case, page = x["case"], x["case"]["page"]
    pages, shift = x["pages"].tolist(), x["shift"].tolist()
    table, slots, positions, seq, who, cu_q, cu_kv, kv, sample, at = [], [], [], [], [], [0], [0], [], [], 0
    for i, (cached, fresh) in enumerate(x["lens"]):
        mine = pages[at:at - (-(cached + fresh) // page)]
        at += len(mine)
        table.append(mine + [-1] * (x["width"] - len(mine)))
        for p in range(cached, cached + fresh):
            slots.append(mine[p // page] * page + p % page)
            positions.append(p + shift[i])
            seq.append(i)
            who.append(x["used"][i])
        cu_q.append(cu_q[-1] + fresh)
        cu_kv.append(cu_kv[-1] + cached + fresh)
        kv.append(cached + fresh)
        sample.append(cu_q[-1] - 1 if fresh else -1)
    index, lists, counts = [], [], []
    for lo in range(0, len(who), 256):
        here = sorted(set(who[lo:lo + 256]) - {-1})
        index += [here.index(w) if w >= 0 else -1 for w in who[lo:lo + 256]]
        lists.append(here + [-1] * (min(case["slots"], 256, len(who)) - len(here)))
        counts.append(len(here))
    i32, i64 = dict(dtype=torch.int32, device=DEV), dict(dtype=torch.int64, device=DEV)
    return (torch.tensor(table, **i32), torch.tensor(slots, **i64), torch.tensor([positions] * 3, **i32), torch.tensor(seq, **i32),
            torch.tensor(who, **i32), torch.tensor(cu_q, **i32), torch.tensor(cu_kv, **i32), torch.tensor(kv, **i32), torch.tensor(sample, **i64),
            torch.tensor(index, **i32), torch.tensor(lists, **i32), torch.tensor(counts, **i32))


def _exact_projection(x):
    """Every adapter folded into the weights: y = x (W + scale B A)^T + bias, the tokens of one adapter at a time."""
    case, parts = x["case"], _parts(x["case"])
    rows = {}
    row = 0
    for (_, n), s in zip(x["lens"], x["used"]):
        rows.setdefault(s, []).extend(range(row, row + n))
        row += n
    w = x["w"].double()
    y = torch.empty(case["tokens"], sum(parts), dtype=torch.float64, device=DEV)
    for s, mine in rows.items():
        mine = torch.tensor(mine, device=DEV)
        full = w if s < 0 else w + x["scale"][s] * torch.cat([b[s].double() @ x["a"][s, i].double() for i, b in enumerate(x["b"])])
        y[mine] = x["x"][mine].double() @ full.T
    if x["bias"] is not None:
        y += x["bias"].double()
    if case["op"] == "gated":
        y = y[:, :parts[0]] * torch.sigmoid(y[:, :parts[0]]) * y[:, parts[0]:]
    return y


# ------------------------------------------------------------------------------------------------ floors
def work(case):
    lens = _lens(case)
    if case["op"] == "maps":
        counts = [-(-(a + b) // case["page"]) for a, b in lens]
        tokens, n = sum(b for _, b in lens), len(lens)
        tiles = -(-tokens // 256)
        return {"bytes": 4 * (sum(counts) + n * max(counts)) + 16 * n + 28 * tokens + 20 * n + 8 + 4 * tokens
                + 4 * tiles * (1 + min(case["slots"], 256, tokens)), "flops": 0}
    size = 4 if case["dtype"] == "fp32" else 2
    features, tokens, width, rank = sum(_parts(case)), case["tokens"], case["width"], case["rank"]
    numbers = _numbers(case)
    used, low = len(set(numbers) - {-1}), len(_parts(case)) * rank
    with_adapter = sum(n for (_, n), k in zip(lens, numbers) if k >= 0)
    out = features // 2 if case["op"] == "gated" else features
    return {"bytes": size * (features * width + tokens * (width + out) + used * (low * width + rank * features) + (features if case["bias"] else 0))
            + 4 * tokens,
            "flops": 2 * tokens * features * width + 2 * with_adapter * (low * width + rank * features)}
