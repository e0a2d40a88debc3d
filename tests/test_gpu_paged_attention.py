"""Paged attention of ragged batches against 64-bit softmax attention over the same
cached values, within the allowance that tests/paged_reference.py derives."""
from __future__ import annotations

import math
import threading

import pytest
import torch

import braidinfer_amd
from braidinfer_amd import _lib
from braidinfer_amd.kernels import Fp4KVCache
from braidinfer_amd.layers import paged_attention
from tests.helpers import gen
from tests.paged_reference import attention64, attention_allowance, from_fp4, make_batch, request_rows, to_fp4

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16 = torch.bfloat16, torch.float16


def make_cache(seed, batch, hkv, d, kind, dtype, layout="HND", fill=None):
    """(what the call takes, the float64 values of it in HND order, on the GPU).  Slots
    that hold no token are NaN (in 4 bits: a scale of 255) unless `fill` is given."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(batch.num_pages, 2, hkv, batch.page_size, d, generator=g, device=DEV)
    x[..., 3] *= 4
    unused = torch.ones(batch.num_pages, batch.page_size, dtype=torch.bool, device=DEV)
    for s, n in enumerate(batch.seq):
        ids = batch.kv_indices[int(batch.kv_indptr[s]): int(batch.kv_indptr[s + 1])].long().to(DEV)
        for i, page in enumerate(ids.tolist()):
            unused[page, : max(0, min(batch.page_size, n - i * batch.page_size))] = False
    hole = unused[:, None, None, :, None].expand_as(x)
    x = torch.where(hole, torch.full_like(x, math.nan if fill is None else fill), x)
    if kind == "fp4":
        codes, scales = to_fp4(torch.nan_to_num(x).cpu().float())
        scales = torch.where(torch.isnan(x).cpu().unflatten(-1, (-1, 32)).any(-1), torch.tensor(255, dtype=torch.uint8), scales)
        return Fp4KVCache(codes.to(DEV), scales.to(DEV)), from_fp4(codes, scales).to(DEV)
    x = x.to(dtype)
    return (x if layout == "HND" else x.transpose(2, 3).contiguous()), x.double()


def attention_without(q, values, batch, s, gone):
    """64-bit attention of request s's rows without the keys `gone`."""
    n, m, at = batch.seq[s], batch.query[s], int(batch.qo_indptr[s])
    group = q.shape[1] // values.shape[2]
    k, v = (x.repeat_interleave(group, 1).permute(1, 0, 2).contiguous() for x in request_rows(values, batch, s))
    z = torch.matmul(q[at: at + m].double().permute(1, 0, 2).contiguous(), k.transpose(1, 2).contiguous()) * q.shape[2] ** -0.5
    hidden = torch.arange(n, device=DEV)[None] > torch.arange(n - m, n, device=DEV)[:, None]
    hidden[:, list(gone)] = True
    return torch.matmul(torch.softmax(z.masked_fill(hidden, -math.inf), -1), v).permute(1, 0, 2)


def lists(batch):
    return [t.to(DEV) for t in (batch.kv_indices, batch.kv_indptr, batch.last, batch.qo_indptr)]


def check(got, q, values, batch, scale, window, sinks, what=""):
    want, parts = attention64(q, values, batch, scale, window, sinks)
    allow = attention_allowance(want, parts, q.dtype, -(-max(batch.seq + [1]) // 32))
    got = got[: batch.tokens].double().reshape(want[: batch.tokens].shape)
    want, allow = want[: batch.tokens], allow[: batch.tokens]
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: other values are NaN"
    off = torch.nan_to_num((got - want).abs() / allow.clamp(min=1e-30))
    assert bool((off <= 1).all()), f"{what}: {float(off.max()):.2f} of the allowance"


def run(seed, seq, query, hq, hkv, d, *, dtype=BF16, kind="16", ps=16, window=None, sinks=0, layout="HND", scale=None, std=1.5):
    batch = make_batch(seed, seq, query, ps)
    cache, values = make_cache(seed, batch, hkv, d, kind, dtype, layout)
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    q = torch.randn(batch.tokens, hq, d, generator=g, device=DEV).mul_(std).to(dtype)
    got = paged_attention(q, cache, *lists(batch), scale=scale, window=window, num_sinks=sinks, kv_layout=layout)
    again = paged_attention(q, cache, *lists(batch), scale=scale, window=window, num_sinks=sinks, kv_layout=layout)
    torch.cuda.synchronize()
    assert got.shape == (batch.tokens, hq * d) and got.dtype == dtype
    assert torch.equal(got.view(torch.int16), again.view(torch.int16)), "two calls differ"
    check(got, q, values, batch, d ** -0.5 if scale is None else scale, window, sinks)
    braidinfer_amd.check_device_status()
    return got


KINDS = [(BF16, "16"), (F16, "16"), (BF16, "fp4"), (F16, "fp4")]
# query heads, kv heads, head_dim: every group from a head of its own to more than a block's 16 rows
HEADS = [(32, 4, 64), (32, 8, 128), (16, 8, 128), (4, 4, 64), (15, 3, 128), (71, 1, 64), (20, 4, 128)]


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_single_tokens(dtype, kind, hq, hkv, d):
    """Lengths around the tile and page borders, one key among them, and one long."""
    run(hq + d, [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 700], [1] * 14, hq, hkv, d, dtype=dtype, kind=kind)


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_windows_and_sinks_over_single_tokens(dtype, kind, hq, hkv, d):
    for window, sinks in ((1, 0), (33, 4), (100, 70), (64, 0), (5000, 3)):
        run(hq + window, [1, 40, 64, 300, 901], [1] * 5, hq, hkv, d, dtype=dtype, kind=kind, window=window, sinks=sinks)


# rows of a block and workgroups of the key split: the planner's own choice, and every
# form, whole and split, at sizes where it would not pick it
FORMS = [(None, None), (16, 200), (64, 0), (64, 200), (128, 0), (128, 200)]


@pytest.mark.parametrize("rows,wgs", FORMS)
@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_prompts(tuning, dtype, kind, hq, hkv, d, rows, wgs):
    """Whole prompts and pieces over a cached context, of odd lengths, in one batch."""
    tuning("PAGED_ROWS", rows), tuning("PAGED_WG", wgs)
    run(hq, [77, 1, 300, 130, 1100], [77, 1, 60, 129, 40], hq, hkv, d, dtype=dtype, kind=kind)


@pytest.mark.parametrize("rows,wgs", [(None, None), (64, 0), (128, 0), (128, 300)])
@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("hq,hkv,d", [(32, 4, 64), (16, 8, 128), (15, 3, 128)])
def test_prompts_with_windows(tuning, dtype, kind, hq, hkv, d, rows, wgs):
    tuning("PAGED_ROWS", rows), tuning("PAGED_WG", wgs)
    for window, sinks in ((1, 0), (17, 1), (64, 64), (65, 4), (200, 130)):
        run(window, [210, 333, 64], [210, 100, 64], hq, hkv, d, dtype=dtype, kind=kind, window=window, sinks=sinks)


@pytest.mark.parametrize("rows", [None, 64, 128])
@pytest.mark.parametrize("ps", [1, 3, 16, 64, 100])
@pytest.mark.parametrize("kind", ["16", "fp4"])
def test_page_sizes(tuning, ps, kind, rows):
    tuning("PAGED_ROWS", rows)
    run(ps, [1, 99, 100, 101, 260], [1] * 5, 8, 2, 64, ps=ps, kind=kind, window=90, sinks=2)
    run(ps, [150, 260], [150, 100], 8, 2, 128, ps=ps, kind=kind)


@pytest.mark.parametrize("rows", [None, 128])
@pytest.mark.parametrize("layout", ["HND", "NHD"])
def test_layouts(tuning, layout, rows):
    tuning("PAGED_ROWS", rows)
    run(1, [5, 200, 64], [1, 1, 1], 16, 4, 128, layout=layout)
    run(2, [5, 200, 64], [5, 150, 3], 16, 4, 128, layout=layout, window=70, sinks=4)


def test_few_rows_of_each_request():
    """Drafts: 2 to 9 rows a request, which mix blocks of one and two tokens' heads."""
    run(3, [40, 9, 500, 77], [9, 9, 5, 2], 8, 4, 128)
    run(4, [40, 9, 500, 77], [3, 4, 5, 2], 32, 4, 64, window=50, sinks=5)
    run(5, [40, 9, 500], [2, 0, 3], 8, 4, 64, kind="fp4")


@pytest.mark.parametrize("kind", ["16", "fp4"])
def test_one_long_request_among_short_ones(kind):
    run(6, [20000, 3, 40, 1], [1, 1, 1, 1], 8, 2, 128, kind=kind)
    run(7, [9000, 3, 40], [130, 3, 40], 8, 2, 64, kind=kind)


def test_many_requests():
    """More requests than a wave has lanes."""
    g = gen(8)
    seq = torch.randint(1, 90, (150,), generator=g).tolist()
    run(8, seq, [1] * 150, 8, 2, 64)
    run(9, seq, [min(n, 1 + i % 3) for i, n in enumerate(seq)], 8, 2, 128, kind="fp4", window=40, sinks=1)
    run(10, seq, [min(n, 1 + 31 * (i % 5 == 0)) for i, n in enumerate(seq)], 16, 2, 64)


@pytest.mark.parametrize("rows", [16, 64, 128])
@pytest.mark.parametrize("scale", [1.0, -0.3, 0.0, 1e-3])
def test_scales(tuning, scale, rows):
    tuning("PAGED_ROWS", rows)
    run(11, [70, 300], [20, 1], 8, 2, 64, scale=scale)


@pytest.mark.parametrize("rows", [16, 64, 128])
@pytest.mark.parametrize("std", [300.0, 1e6])
def test_scores_that_leave_one_key(tuning, std, rows):
    """Scores in the thousands and in the millions (where the product with the scale is
    rounded before the difference), so that a row is all but one key's value."""
    tuning("PAGED_ROWS", rows)
    run(12, [70, 300, 5], [20, 1, 5], 8, 2, 128, std=std)


def test_rows_that_see_nothing():
    """Requests without pages, rows in front of the first cached token, a last page
    without tokens: zeros."""
    batch = make_batch(13, [40, 0, 3, 32], [2, 3, 5, 1], 16)
    batch.kv_indptr = torch.tensor([0, 3, 3, 4, 6], dtype=torch.int32)
    cache, values = make_cache(13, batch, 2, 64, "16", BF16)
    q = torch.randn(11, 4, 64, device=DEV).to(BF16)
    got = paged_attention(q, cache, *lists(batch))
    want, parts = attention64(q, values, batch, 0.125)
    assert not got[2:5].any() and not got[5:7].any() and got[7:].any()
    check(got, q, values, batch, 0.125, None, 0)
    batch.last[3] = 0  # the last request: one full page, then an empty one
    batch.seq[3] = 16
    got = paged_attention(q, cache, *lists(batch))
    check(got, q, values, batch, 0.125, None, 0)
    nothing = torch.zeros(0, dtype=torch.int32, device=DEV)
    zero = torch.zeros(2, dtype=torch.int32, device=DEV)
    got = paged_attention(q, cache, nothing, zero, zero[:1], torch.tensor([0, 11], dtype=torch.int32, device=DEV))
    assert not got.any()
    braidinfer_amd.check_device_status()


def test_rows_behind_the_last_request_stay():
    batch = make_batch(14, [40, 70], [1, 1], 16)
    cache, values = make_cache(14, batch, 2, 64, "16", BF16)
    for more in (1, 300):
        q = torch.randn(2 + more, 4, 64, device=DEV).to(BF16)
        buf = torch.full((2 + more, 4 * 64 + 8), 7.0, dtype=BF16, device=DEV)
        out = buf[:, : 4 * 64]
        assert paged_attention(q, cache, *lists(batch), out=out) is out
        assert bool((buf[2:] == 7).all()) and bool((buf[:, 256:] == 7).all())
        check(out, q, values, batch, 0.125, None, 0)


@pytest.mark.parametrize("rows,ps", [(16, 16), (64, 16), (128, 16), (128, 5)])
@pytest.mark.parametrize("kind", ["16", "fp4"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_key_reaches_only_the_rows_that_see_it(tuning, kind, bad, rows, ps):
    """A token whose key and value are not finite, in the middle of a prompt and of a few
    drafted tokens: rows before it, and rows whose window has passed it, are as without."""
    for seq, query, window in (([150], [150], None), ([300], [150], 40), ([300], [4], None), ([300], [4], 2)):
        tuning("PAGED_ROWS", rows)
        batch = make_batch(15, seq, query, ps)
        cache, values = make_cache(15, batch, 2, 64, kind, BF16)
        at = seq[0] - query[0] // 2 - 1
        page, slot = int(batch.kv_indices[at // ps]), at % ps
        if kind == "fp4":
            cache.scales[page, 1, :, slot, 1] = 255
            values[page, 1, :, slot, 32:] = math.nan
        else:
            cache[page, 1, :, slot, 5] = bad
            values[page, 1, :, slot, 5] = bad
        q = torch.randn(query[0], 4, 64, device=DEV).to(BF16)
        got = paged_attention(q, cache, *lists(batch), window=window)
        pos = torch.arange(query[0]) + seq[0] - query[0]
        clean = (pos < at) | (pos - at >= (window or 10 ** 9))
        assert bool(clean.any()) and torch.isfinite(got[clean]).all()
        assert not torch.isfinite(got[~clean]).all(-1).any()
        want, parts = attention64(q, values, batch, 0.125, window)
        allow = attention_allowance(want, parts, BF16, 10)
        off = (got.double().reshape(want.shape) - want).abs()
        assert bool((off <= allow)[clean].all())
        # a key that is not finite: its score is, too, for the rows that see it alone
        if kind == "16":
            cache[page, 1, :, slot, 5] = 0.5
            cache[page, 0, :, slot, 7] = math.nan
            got = paged_attention(q, cache, *lists(batch), window=window)
            assert torch.isfinite(got[clean]).all() and not torch.isfinite(got[~clean]).any()


@pytest.mark.parametrize("rows", [16, 64, 128])
def test_pages_and_offsets_that_do_not_exist(tuning, rows):
    """Each is told, and what is there is attended all the same."""
    tuning("PAGED_ROWS", rows)
    batch = make_batch(16, [40, 70, 33], [1, 30, 1], 16)
    cache, values = make_cache(16, batch, 2, 64, "16", BF16)
    q = torch.randn(32, 4, 64, device=DEV).to(BF16)
    good = paged_attention(q, cache, *lists(batch))
    braidinfer_amd.check_device_status()
    wrapped = batch.kv_indices - batch.num_pages  # ids from the end
    idx, ptr, last, qo = lists(batch)
    assert torch.equal(paged_attention(q, cache, wrapped.to(DEV), ptr, last, qo), good)
    braidinfer_amd.check_device_status()

    def told(idx=idx, ptr=ptr, last=last, qo=qo):
        got = paged_attention(q, cache, idx, ptr, last, qo)
        with pytest.raises(IndexError):
            braidinfer_amd.check_device_status()
        return got

    for page in (batch.num_pages, -batch.num_pages - 1, 2 ** 31 - 1, -2 ** 31):
        bad = idx.clone()
        bad[4] = page  # keys 16 .. 31 of the second request
        got = told(idx=bad)
        assert torch.equal(got[0], good[0]) and torch.equal(got[31], good[31])
        # (half a step of the weights and of the result, and as much for scores of up to 128)
        want = attention_without(q, values, batch, 1, range(16, 32))
        off = (got[1:31].double().reshape(30, 4, 64) - want).abs()
        assert float(off.max()) < 3 * 2.0 ** -8 * float(torch.nan_to_num(values).abs().max())
    # (s: as it was, 0: left out, -: more pages than the request has, whose unused slots are NaN)
    for t, kinds in (([0, 3, 8, 99], "ss0"), ([-1, 3, 8, 11], "0ss"), ([0, 9, 8, 11], "-0s"), ([0, 3, 2 ** 31 - 1, 11], "s00")):
        got = told(ptr=torch.tensor(t, dtype=torch.int32, device=DEV))
        for kind, a, b in zip(kinds, (0, 1, 31), (1, 31, 32)):
            assert kind == "-" or torch.equal(got[a:b], good[a:b] if kind == "s" else torch.zeros_like(good[a:b])), (t, a)
    for t in ([8, 17, 1], [8, -1, 1], [-2 ** 31, 2 ** 31 - 1, 1]):
        got = told(last=torch.tensor(t, dtype=torch.int32, device=DEV))
        assert torch.equal(got[31], good[31])
    for t in ([0, 1, 31, 33], [-1, 1, 31, 32], [0, 40, 31, 32], [0, 32, 0, 32], [0, 2 ** 31 - 1, -2 ** 31, 32]):
        told(qo=torch.tensor(t, dtype=torch.int32, device=DEV))
    many = torch.tensor([0, 32] * 100 + [0], dtype=torch.int32, device=DEV)  # every other request holds all rows
    told(qo=many, ptr=torch.zeros(201, dtype=torch.int32, device=DEV), last=torch.zeros(200, dtype=torch.int32, device=DEV))


def test_strided_queries():
    batch = make_batch(17, [40, 70], [1, 30], 16)
    cache, values = make_cache(17, batch, 2, 64, "16", BF16)
    qkv = torch.randn(31, 12, 64, device=DEV).to(BF16)
    q = qkv[:, 2:6]
    check(paged_attention(q, cache, *lists(batch)), q, values, batch, 0.125, None, 0)
    odd = torch.randn(31, 4, 65, device=DEV).to(BF16)[..., 1:]  # copied: unaligned
    check(paged_attention(odd, cache, *lists(batch)), odd, values, batch, 0.125, None, 0)
    big = torch.zeros(batch.num_pages, 2, 4, 16, 64, dtype=BF16, device=DEV)  # a slice of a cache of more heads
    big[:, :, 1:3] = cache
    check(paged_attention(q, big[:, :, 1:3], *lists(batch)), q, values, batch, 0.125, None, 0)


@pytest.mark.parametrize("kind", ["16", "fp4"])
def test_a_captured_graph_follows_the_lengths(kind):
    """One graph of a padded batch, replayed over other lengths with eager calls between."""
    batch = make_batch(18, [900, 900, 900], [1, 1, 1], 16)
    cache, values = make_cache(18, batch, 2, 64, kind, BF16, fill=0.25)
    idx, ptr, last, qo = lists(batch)
    q = torch.randn(5, 8, 64, device=DEV).to(BF16)
    paged_attention(q, cache, idx, ptr, last, qo, window=300, num_sinks=3)
    torch.cuda.synchronize()
    graphs = []
    for window in (None, 300):  # two graphs, each with scratch memory of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = paged_attention(q, cache, idx, ptr, last, qo, window=window, num_sinks=3)
        graphs.append((graph, out, window))
    for seq, query in (([900, 900, 900], [1, 1, 1]), ([1, 880, 33], [1, 1, 1]), ([17, 400, 64], [1, 3, 1]), ([900, 5, 500], [0, 1, 2])):
        b = make_batch(18, seq, query, 16)
        pages = [-(-n // 16) for n in seq]
        b.kv_indices = torch.cat([batch.kv_indices[57 * i: 57 * i + p] for i, p in enumerate(pages)])
        idx[: b.kv_indices.numel()].copy_(b.kv_indices)
        ptr.copy_(b.kv_indptr), last.copy_(b.last), qo.copy_(b.qo_indptr)
        for graph, out, window in graphs:
            out.fill_(3.0)
            graph.replay()
            eager = paged_attention(q, cache, idx, ptr, last, qo, window=window, num_sinks=3)
            torch.cuda.synchronize()
            assert torch.equal(out[: b.tokens], eager[: b.tokens]) and bool((out[b.tokens:] == 3).all())
            check(out, q[: b.tokens], values, b, 0.125, window, 3)
    braidinfer_amd.check_device_status()


def test_streams_and_threads():
    """Calls at once from four threads on one stream, and on streams of their own."""
    jobs = []
    for i in range(4):
        batch = make_batch(20 + i, [900 + 50 * i, 40], [1 + 3 * i, 1], 16)
        cache, _ = make_cache(20 + i, batch, 2, 64, "fp4" if i % 2 else "16", BF16)
        q = torch.randn(batch.tokens, 8, 64, device=DEV).to(BF16)
        jobs.append(lambda q=q, cache=cache, batch=lists(batch): paged_attention(q, cache, *batch))
    alone = [j() for j in jobs]
    torch.cuda.synchronize()
    for own_stream in (False, True):
        start, wrong = threading.Barrier(4), []

        def work(i):
            stream = torch.cuda.Stream() if own_stream else torch.cuda.default_stream()
            start.wait()
            with torch.cuda.stream(stream):
                outs = [jobs[i]() for _ in range(20)]
                stream.synchronize()
                wrong.extend(i for o in outs if not torch.equal(o, alone[i]))

        threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join(60)
        assert not any(t.is_alive() for t in threads) and not wrong


def test_a_cache_past_four_gigabytes():
    """Byte offsets past 32 bits (in 16-byte units they are not)."""
    pages, hkv, ps, d = 70000, 8, 16, 128  # 4.6 GB in bf16
    cache = torch.empty(pages, 2, hkv, ps, d, dtype=BF16, device=DEV)
    batch = make_batch(30, [50, 33], [1, 20], ps)
    ids = torch.tensor([69999, 3, 69998, 40000, 69000, 1, 65536], dtype=torch.int32)
    batch.kv_indices = ids
    g = torch.Generator(device=DEV).manual_seed(30)
    small = torch.randn(7, 2, hkv, ps, d, generator=g, device=DEV).to(BF16)
    cache[ids.long().to(DEV)] = small
    q = torch.randn(21, 16, d, device=DEV).to(BF16)
    got = paged_attention(q, cache, *lists(batch))
    batch.kv_indices = torch.arange(7, dtype=torch.int32)
    check(got, q, small.double(), batch, d ** -0.5, None, 0)


@pytest.mark.parametrize("kind", ["16", "fp4"])
@pytest.mark.parametrize("rows,wgs", [(16, 0), (16, 300), (64, 0), (64, 300), (128, 300)])
def test_shared_pages_and_an_output_over_the_queries(tuning, rows, wgs, kind):
    """Requests that share a prefix list the same pages, one request one page twice; the
    output may be the queries' own memory, which a block reads before its rows are written."""
    tuning("PAGED_ROWS", rows), tuning("PAGED_WG", wgs)
    batch = make_batch(21, [900, 700, 900, 64], [70, 1, 130, 40], 16)
    at = batch.kv_indptr.tolist()
    batch.kv_indices[at[1]: at[1] + 40] = batch.kv_indices[:40]
    batch.kv_indices[at[2]: at[2] + 40] = batch.kv_indices[:40]
    batch.kv_indices[at[3] + 1] = batch.kv_indices[at[3]]
    cache, values = make_cache(21, batch, 2, 64, kind, BF16)
    q = torch.randn(batch.tokens, 8, 64, device=DEV, generator=torch.Generator(device=DEV).manual_seed(22)).to(BF16)
    both = q.clone()
    out = both.view(batch.tokens, 512)
    assert paged_attention(both, cache, *lists(batch), window=500, num_sinks=3, out=out) is out
    check(out, q, values, batch, 0.125, 500, 3)
    braidinfer_amd.check_device_status()
