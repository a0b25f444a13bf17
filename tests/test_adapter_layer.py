"""A decoder layer whose requests bring adapters of their own: step maps, plan, adapted projections, paged cache and attention as a server
runs them, prompts first, then decode steps whose lengths stay on the device.  Against one request at a time in 64 bits with its adapter
folded into the weights."""

import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from op_helpers import CPU, GPU16, rand  # noqa: E402

from prism_infer_b200 import ops  # noqa: E402
from prism_infer_b200.models.position import mrope_cos_sin, rotate_half  # noqa: E402
from prism_infer_b200.ops import adapters, batch, native  # noqa: E402

H, HEADS, KV, D, FF, SLOTS, RANK, PAGE, EPS, THETA, SECTION = 256, 4, 2, 128, 320, 5, 12, 16, 1e-6, 1e4, (24, 20, 20)
QKV = (HEADS * D, KV * D, KV * D)
SHAPES = {"qkv": (H, QKV), "o": (HEADS * D, (H,)), "gate_up": (H, (FF, FF)), "down": (FF, (H,))}


class Layer:
    def __init__(self, device, dtype):
        self.w, self.a, self.b, self.pools = {}, {}, {}, {}
        self.norms = {n: 1.0 + rand(size, seed=70 + i, scale=0.1) for i, (n, size) in enumerate((("in", H), ("post", H), ("q", D), ("k", D)))}
        for i, (name, (k, sections)) in enumerate(SHAPES.items()):
            self.w[name] = rand(sum(sections), k, seed=10 * i, scale=k ** -0.5)
            self.a[name] = rand(SLOTS, len(sections), RANK, k, seed=10 * i + 1, scale=k ** -0.5)
            self.b[name] = [rand(SLOTS, m, RANK, seed=10 * i + 2 + j, scale=0.5 * RANK ** -0.5) for j, m in enumerate(sections)]
            pool = self.pools[name] = adapters.AdapterPool(SLOTS, RANK, k, sections, device=device, dtype=dtype)
            for s in range(SLOTS):
                pool.load(s, list(self.a[name][s]), [b[s] for b in self.b[name]], 2.0 - 0.25 * s)
        self.dev_w = {n: w.to(device, dtype) for n, w in self.w.items()}
        self.dev_norms = {n: w.to(device, dtype) for n, w in self.norms.items()}

    def run(self, x, maps, plan, cache, decode, max_q=0):
        w, norm = self.dev_w, self.dev_norms
        h = ops.rmsnorm(x, norm["in"], EPS)
        qkv = adapters.linear(h, w["qkv"], self.pools["qkv"], plan)
        q = ops.qk_norm_rope_store(qkv=qkv, partials=None, positions=maps.positions, q_weight=norm["q"], k_weight=norm["k"], num_heads=HEADS, num_kv_heads=KV,
                                   head_dim=D, theta=THETA, section=SECTION, eps=EPS, slots=maps.slots, cache=cache, layer=0)
        if decode:
            o = ops.paged_decode_attention(q, cache, 0, maps.block_tables, maps.kv_lens)
        else:
            o = ops.paged_prefill_attention(q, cache, 0, maps.cu_seqlens_q, maps.kv_lens, maps.block_tables, max_q, cu_seqlens_kv=maps.cu_seqlens_kv,
                                            total_kv=int(maps.cu_seqlens_kv[-1]), max_kv_len=int(maps.kv_lens.max()))
        y = adapters.linear(o.reshape(len(x), -1), w["o"], self.pools["o"], plan)
        h, x = ops.add_rmsnorm(norm["post"], EPS, x=y, residual=x.clone())
        h = adapters.gate_up_glu(h, w["gate_up"], self.pools["gate_up"], plan, "silu")
        return x + adapters.linear(h, w["down"], self.pools["down"], plan)

    def folded(self, slot):
        out = {n: w.double() for n, w in self.w.items()}
        if slot >= 0:
            for n in out:
                out[n] = out[n] + (2.0 - 0.25 * slot) * torch.cat([b[slot].double() @ a.double() for a, b in zip(self.a[n][slot], self.b[n])])
        return out

    def plain(self, x, slot, first, keys):
        """One request's new rows ``x`` behind ``first`` earlier ones, whose keys and values are in ``keys``."""
        w, x, norm = self.folded(slot), x.double(), {n: v.double() for n, v in self.norms.items()}

        def rms(z, g):
            return z / (z.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * g

        q, k, v = (rms(x, norm["in"]) @ w["qkv"].T).split(QKV, 1)
        q, k, v = q.view(-1, HEADS, D), k.view(-1, KV, D), v.view(-1, KV, D)
        cos, sin = mrope_cos_sin(torch.arange(first, first + len(x)).expand(3, -1), D, THETA, SECTION)
        q, k = (z * cos[:, None].double() + rotate_half(z) * sin[:, None].double() for z in (rms(q, norm["q"]), rms(k, norm["k"])))
        keys.append((k, v))
        k, v = (torch.cat([p[i] for p in keys]).repeat_interleave(HEADS // KV, 1) for i in (0, 1))
        s = torch.einsum("qhd,khd->hqk", q, k) * D ** -0.5
        s = s.masked_fill(torch.arange(len(k))[None] > torch.arange(first, first + len(x))[:, None], float("-inf"))
        x = x + torch.einsum("hqk,khd->qhd", s.softmax(-1), v).reshape(len(x), -1) @ w["o"].T
        gate, up = (rms(x, norm["post"]) @ w["gate_up"].T).split(FF, 1)
        return x + (torch.nn.functional.silu(gate) * up) @ w["down"].T


@pytest.mark.parametrize("backend", [CPU, GPU16])
@pytest.mark.parametrize("lengths", [(1, 2, 3), (5, 17, 40, 1, 16), (150, 33, 300, 90)])
def test_prompts_then_decode_steps(backend, lengths):
    device, dtype = backend
    S, steps = len(lengths), 6
    slots = [s % (SLOTS + 1) - 1 for s in range(S)]
    layer = Layer(device, dtype)
    per = [-(-(n + steps) // PAGE) for n in lengths]
    order = torch.randperm(sum(per) + 3, generator=torch.Generator().manual_seed(1))[:sum(per)].int()
    i32 = dict(dtype=torch.int32, device=device)
    cache = ops.KVCache(1, sum(per) + 3, KV, PAGE, D, ops.KV_BF16, device, dtype=dtype)
    args = dict(page=PAGE, width=max(per), page_offsets=torch.tensor([sum(per[:i]) for i in range(S + 1)], **i32), adapter=torch.tensor(slots, **i32))
    pages, zero = order.to(device), torch.zeros(S, **i32)
    x = rand(sum(lengths), H, seed=90)
    state = [[] for _ in range(S)]
    # From the input to the output a value is rounded about ten times (projections, norms, rotation, weights of the attention, gated unit,
    # sums), each time by at most 2^-8 of the largest value of its tensor in bf16; errors of that size add up with either sign.
    tol = 10 * 2.0 ** -8 if dtype == torch.bfloat16 else 1e-4

    def same(got, rows, at):
        first = 0
        for s in range(S):
            want = layer.plain(rows[first:first + at[s][1]], slots[s], at[s][0], state[s])
            err = (got[first:first + at[s][1]].double().cpu() - want).abs().max() / want.abs().max()
            assert float(err) < tol, (s, float(err))
            first += at[s][1]

    # padding rows behind the last request take no part
    T = sum(lengths) + 3
    maps = batch.step_maps(pages, zero, torch.tensor(lengths, **i32), tokens=T, **args)
    padded = torch.cat([x, torch.full((3, H), 9.0)]).to(device, dtype)
    got = layer.run(padded, maps, adapters.plan(maps.token_adapter, SLOTS), cache, False, max(lengths))
    same(got[:sum(lengths)], x, [(0, n) for n in lengths])

    cached, one, xin = maps.kv_lens.clone(), torch.ones(S, **i32), torch.empty(S, H, dtype=dtype, device=device)

    def step():
        m = batch.step_maps(pages, cached, one, tokens=S, **args)
        y = layer.run(xin, m, adapters.plan(m.token_adapter, SLOTS), cache, True)
        cached.copy_(m.kv_lens)
        return y

    graph, out = None, None
    for n in range(steps):
        x = rand(S, H, seed=100 + n)
        xin.copy_(x.to(device, dtype))
        if device == "cpu" or n < 2:
            out = step()
        else:
            if graph is None:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                keep = cached.clone()
                with torch.cuda.graph(graph):
                    out = step()
                cached.copy_(keep)
            graph.replay()
        same(out, x, [(length + n, 1) for length in lengths])
    if device != "cpu":
        native.check_status()
