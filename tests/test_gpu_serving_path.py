"""The batched serving operators as one layer's step uses them: the step's batch from
the requests' lengths, q/k norm with rotation of a projection's output, the append to a
16-bit or a 4-bit cache, and attention over it.  Eager over several steps, a mix of
prompts and single tokens, and as one captured graph replayed step after step."""
from __future__ import annotations

import pytest
import torch

import braidinfer_amd
from braidinfer_amd.kernels import Fp4KVCache, append_paged_kv_batch, append_paged_kv_fp4, build_paged_kv_batch
from braidinfer_amd.layers import linear, paged_attention, qk_norm_rope
from oracle import torch_ref as R
from tests.helpers import gen, randn
from tests.paged_reference import attention64, attention_allowance, from_fp4, make_batch, to_fp4

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, HQ, HKV, D, PS, WINDOW, SINKS = 512, 8, 2, 64, 16, 50, 3
B, WIDTH = 5, 12


class Layer:
    def __init__(self, seed, kind):
        g = gen(seed)
        self.kind = kind
        self.w = randn(g, (HQ + 2 * HKV) * D, H, std=0.04).to(DEV)
        self.qn, self.kn = randn(g, D, mean=1.0, std=0.2).to(DEV), randn(g, D, std=0.3).exp().to(DEV)
        self.table = R.cos_sin_cache(D, 512, 1e4).to(DEV)
        pages = B * WIDTH
        self.page_tables = torch.randperm(pages, generator=g).to(torch.int32).reshape(B, WIDTH).to(DEV)
        if kind == "fp4":
            self.cache = Fp4KVCache.empty(pages, HKV, PS, D)
            self.cache.codes.fill_(0x77), self.cache.scales.fill_(255)  # what no token wrote reads as NaN
        else:
            self.cache = torch.full((pages, 2, HKV, PS, D), float("nan"), dtype=torch.bfloat16, device=DEV)

    def step(self, x, seq, query):
        """(attention output, q, k, v, batch) of the step's rows x."""
        batch = build_paged_kv_batch(self.page_tables, seq, query, PS, x.shape[0])
        q, k, v = linear(x, self.w).split([HQ * D, HKV * D, HKV * D], -1)
        q, k = qk_norm_rope(q, k, self.qn, self.kn, batch.positions, self.table, 1e-6)
        q, k, v = q.view(-1, HQ, D), k.view(-1, HKV, D), v.unflatten(1, (HKV, D))
        if self.kind == "fp4":
            append_paged_kv_fp4(k, v, self.cache, batch.kv_indices, batch.kv_indptr, batch.batch_indices, batch.positions)
        else:
            append_paged_kv_batch(k, v, self.cache, batch.kv_indices, batch.kv_indptr, batch.batch_indices, batch.positions, PS)
        out = paged_attention(q, self.cache, batch.kv_indices, batch.kv_indptr, batch.kv_last_page_len, batch.qo_indptr,
                              window=WINDOW, num_sinks=SINKS)
        return out, q, k, v, batch

    def values(self):
        if self.kind == "fp4":
            return from_fp4(self.cache.codes, self.cache.scales).to(DEV)
        return self.cache.double()


class Expected:
    """Every request's own keys and values, kept on the side, token by token."""

    def __init__(self, kind):
        self.kind, self.rows = kind, [[torch.empty(0, HKV, D, dtype=torch.float64), torch.empty(0, HKV, D, dtype=torch.float64)]
                                      for _ in range(B)]

    def check(self, layer, seq, query, out, q, k, v, batch, what):
        live = sum(query)
        at = 0
        ref = make_batch(0, seq, query, PS)
        ref.kv_indices = batch.kv_indices.cpu()[: int(batch.kv_indptr[-1])]
        assert ref.kv_indptr.tolist() == batch.kv_indptr.tolist() and ref.qo_indptr.tolist() == batch.qo_indptr.tolist()
        values = layer.values()
        for b in range(B):
            for i, x in enumerate((k, v)):
                new = x[at: at + query[b]].cpu()
                new = from_fp4(*to_fp4(new)) if self.kind == "fp4" else new.double()
                self.rows[b][i] = torch.cat((self.rows[b][i], new))
                ids = ref.kv_indices[int(ref.kv_indptr[b]): int(ref.kv_indptr[b + 1])].long().to(DEV)
                held = values[ids, i].transpose(1, 2).flatten(0, 1)[: seq[b]]
                assert torch.equal(held.cpu(), self.rows[b][i]), f"{what}: the cache of request {b}"
            at += query[b]
        want, parts = attention64(q[:live], values, ref, D ** -0.5, WINDOW, SINKS)
        allow = attention_allowance(want, parts, torch.bfloat16, WIDTH * PS // 32)
        off = (out[:live].double().reshape(want.shape) - want).abs()
        assert bool((off <= allow).all()), f"{what}: {float((off / allow).max()):.2f} of the allowance"


STEPS = [[60, 1, 17, 33, 0], [1, 1, 1, 1, 40], [1, 30, 1, 1, 1], [1, 1, 1, 1, 1], [5, 1, 3, 1, 20]]


@pytest.mark.parametrize("kind", ["16", "fp4"])
def test_steps_of_prompts_and_single_tokens(kind):
    layer, expected, seq = Layer(1, kind), Expected(kind), [0] * B
    g = gen(2)
    for n, query in enumerate(STEPS):
        seq = [a + b for a, b in zip(seq, query)]
        x = randn(g, sum(query), H).to(DEV)
        got = layer.step(x, torch.tensor(seq, device=DEV), torch.tensor(query, device=DEV))
        expected.check(layer, seq, query, *got, f"step {n}")
        braidinfer_amd.check_device_status()


@pytest.mark.parametrize("kind", ["16", "fp4"])
def test_one_graph_for_every_step(kind):
    """Single tokens of every request, the lengths advanced on the device between the
    replays; an eager call of another layer runs in between."""
    layer, other, expected = Layer(3, kind), Layer(4, kind), Expected(kind)
    g = gen(5)
    seq, query = [20, 1, 16, 47, 100], [20, 1, 16, 47, 100]
    first = randn(g, sum(query), H).to(DEV)
    lens, ones = torch.tensor(seq, device=DEV), torch.ones(B, dtype=torch.int64, device=DEV)
    got = layer.step(first, lens, torch.tensor(query, device=DEV))
    expected.check(layer, seq, query, *got, "prompts")
    other.step(first, lens, torch.tensor(query, device=DEV))
    x = torch.empty(B, H, dtype=torch.bfloat16, device=DEV)
    x.copy_(randn(g, B, H))
    lens.add_(1)
    layer.step(x, lens, ones)  # warm, and the first step's tokens, which the first replay writes again
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer.step(x, lens, ones)
    for n in range(40):
        if n:
            x.copy_(randn(g, B, H))
            lens.add_(1)
        seq = [v + 1 for v in seq]
        graph.replay()
        other.step(x, lens, ones)
        torch.cuda.synchronize()
        expected.check(layer, seq, [1] * B, *got, f"replay {n}")
    braidinfer_amd.check_device_status()
