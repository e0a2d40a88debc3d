"""A step's batch built on the GPU against a walk over Python lists: whole numbers, all
of them equal, what is behind the last request among them."""
from __future__ import annotations

import pytest
import torch

import braidinfer_amd
from braidinfer_amd.kernels import build_paged_kv_batch
from tests.helpers import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32, I64 = torch.int32, torch.int64


def expected(tables, seq, query, ps, num_tokens):
    rows, width = tables.tolist(), tables.shape[1]
    qo, kv, indices, last, owner, pos, slot = [0], [0], [], [], [], [], []
    for b, (n, m) in enumerate(zip(seq, query)):
        n, m = max(n, 0), max(m, 0)
        held = min(n, width * ps)
        used = -(-held // ps)
        indices += rows[b][:used]
        kv.append(len(indices))
        last.append(held - (used - 1) * ps if used else 0)
        for p in range(n - m, n):
            owner.append(b)
            pos.append(p)
            slot.append(rows[b][p // ps] * ps + p % ps if 0 <= p < held else -1)
        qo.append(len(owner))
    pad = lambda v, n: (v + [-1] * (n - len(v)))[:n]  # noqa: E731
    return ([min(v, num_tokens) for v in qo], kv, pad(indices, tables.numel()), last, pad(owner, num_tokens),
            pad(pos, num_tokens), pad(slot, num_tokens))


def check(tables, seq, query, ps, num_tokens, dtypes=(I32, I32), what="", tables_dev=None, out=None):
    got = build_paged_kv_batch(tables.to(DEV) if tables_dev is None else tables_dev, torch.tensor(seq, dtype=dtypes[0], device=DEV),
                               torch.tensor(query, dtype=dtypes[1], device=DEV), ps, num_tokens, out)
    for name, g, e in zip(got._fields, got, expected(tables, seq, query, ps, num_tokens)):
        assert g.tolist() == e, f"{what} {name}"
    return got


def make_tables(seed, b, width, dtype=I32):
    return torch.randperm(max(b * width, 1), generator=gen(seed))[: b * width].reshape(b, width).to(dtype)


@pytest.mark.parametrize("b,width,ps,dtype,lens", [
    (1, 1, 16, I32, (I32, I32)), (1, 700, 16, I64, (I64, I32)), (3, 5, 1, I32, (I32, I64)), (64, 40, 16, I32, (I64, I64)),
    (257, 9, 7, I64, (I32, I32)), (1000, 6, 128, I32, (I32, I32)), (2, 3000, 3, I32, (I32, I32))])
def test_batches(b, width, ps, dtype, lens):
    g = gen(b + width)
    seq = torch.randint(0, width * ps + 1, (b,), generator=g).tolist()
    seq[0] = width * ps  # a full table
    if b > 2:
        seq[1], seq[2] = 0, ps * (width // 2)  # an empty request, and a last page that is full
    query = [int(torch.randint(0, min(n, 40) + 1, (1,), generator=g)) for n in seq]
    for pad in (0, 19):
        check(make_tables(b, b, width, dtype), seq, query, ps, sum(query) + pad, lens, f"pad {pad}")
    braidinfer_amd.check_device_status()


def test_decode_batch_and_whole_prompts():
    tables = make_tables(5, 6, 70)
    check(tables, [1, 16, 17, 1000, 33, 1120], [1] * 6, 16, 6)
    check(tables, [1, 16, 17, 1000, 33, 1120], [1, 16, 17, 1000, 33, 1120], 16, 2187)
    braidinfer_amd.check_device_status()


def test_no_requests_and_no_tokens():
    check(torch.empty(0, 4, dtype=I32), [], [], 16, 3)
    check(torch.empty(2, 0, dtype=I32), [0, 0], [0, 0], 16, 2)
    check(make_tables(1, 2, 3), [5, 0], [0, 0], 16, 0)
    braidinfer_amd.check_device_status()


def test_strided_table_and_written_again():
    whole = make_tables(2, 8, 20).to(DEV)
    part = whole[:, 3:11]
    out = check(part.cpu(), [100, 3, 0, 128, 64, 1, 17, 90], [4, 3, 0, 1, 64, 1, 2, 5], 16, 90, tables_dev=part)
    again = check(part.cpu(), [3, 100, 128, 0, 1, 64, 90, 17], [1, 1, 1, 0, 1, 1, 1, 1], 16, 90, tables_dev=part, out=out)
    assert again is out
    rows = whole[::2]
    check(rows.cpu(), [7, 300, 20, 33], [7, 1, 20, 2], 16, 30, tables_dev=rows)
    braidinfer_amd.check_device_status()


@pytest.mark.parametrize("seq,query,tokens", [([-3, 20], [1, 2], 3), ([20, 65], [1, 1], 2), ([3, 20], [5, 2], 7),
                                              ([20, 20], [-1, 2], 2), ([64, 2 ** 31 - 1], [1, 3], 4), ([20, 20], [3, 4], 5)])
def test_lengths_that_do_not_fit_are_told(seq, query, tokens):
    check(make_tables(3, 2, 4), seq, query, 16, tokens)
    with pytest.raises(IndexError):
        braidinfer_amd.check_device_status()


def test_a_captured_graph_follows_the_lengths():
    tables = make_tables(4, 5, 12).to(DEV)
    seq, query = torch.zeros(5, dtype=I32, device=DEV), torch.zeros(5, dtype=I32, device=DEV)
    build_paged_kv_batch(tables, seq, query, 16, 30)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = build_paged_kv_batch(tables, seq, query, 16, 30)
    for lens in ([1, 2, 3, 4, 5], [192, 0, 64, 65, 63], [17] * 5):
        q = [min(n, 6) for n in lens]
        seq.copy_(torch.tensor(lens)), query.copy_(torch.tensor(q))
        graph.replay()
        torch.cuda.synchronize()
        for name, g, e in zip(got._fields, got, expected(tables.cpu(), lens, q, 16, 30)):
            assert g.tolist() == e, name
        check(tables.cpu(), lens, q, 16, 30)  # eager work between the replays
    braidinfer_amd.check_device_status()
