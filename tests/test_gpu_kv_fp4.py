"""The 4-bit cache: codes and scales bit by bit against the definition (every step but
the rounding to a code is exact), the values read back, and the addressing of tokens."""
from __future__ import annotations

import math
import warnings

import pytest
import torch

import braidinfer_amd
from braidinfer_amd.kernels import Fp4KVCache, append_paged_kv_batch, append_paged_kv_fp4, gather_paged_kv_fp4
from tests.helpers import gen, randn
from tests.paged_reference import from_fp4, make_batch, to_fp4

pytestmark = pytest.mark.gpu
DEV = "cuda"


def new_cache(pages, heads, ps, d, fill=0x5A):
    c = Fp4KVCache.empty(pages, heads, ps, d)
    c.codes.fill_(fill), c.scales.fill_(fill)
    return c


def tokens_of(batch):
    owner = torch.repeat_interleave(torch.arange(len(batch.seq)), torch.tensor(batch.query))
    pos = torch.cat([torch.arange(n - m, n) for n, m in zip(batch.seq, batch.query)] or [torch.empty(0, dtype=torch.long)])
    return owner, pos


def same_values(a, b):
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,d,ps", [(4, 64, 16), (8, 128, 16), (1, 32, 1), (3, 96, 7), (2, 256, 64)])
def test_append_and_gather(dtype, heads, d, ps):
    g = gen(heads + d)
    batch = make_batch(d, [50, 1, 0, 130], [50, 1, 0, 9], ps)
    owner, pos = tokens_of(batch)
    t = batch.tokens
    k, v = (randn(g, t, heads, d, dtype=torch.float32) * torch.exp(3 * randn(g, t, heads, 1, dtype=torch.float32)) for _ in range(2))
    k, v = k.to(dtype), v.to(dtype)
    cache = new_cache(batch.num_pages, heads, ps, d)
    args = (batch.kv_indices.to(DEV), batch.kv_indptr.to(DEV), owner.to(DEV), pos.to(DEV))
    append_paged_kv_fp4(k.to(DEV), v.to(DEV), cache, *args)
    want_c, want_s = torch.full_like(cache.codes.cpu(), 0x5A), torch.full_like(cache.scales.cpu(), 0x5A)
    page = batch.kv_indices[batch.kv_indptr[owner] + pos // ps].long()
    for i, x in enumerate((k, v)):
        c, s = to_fp4(x)
        want_c[page, i, :, pos % ps], want_s[page, i, :, pos % ps] = c, s
    got_c, got_s = cache.codes.cpu(), cache.scales.cpu()
    assert torch.equal(got_s, want_s)  # (slots that no token has keep their bytes)
    zero = lambda c: torch.where(c % 16 == 8, c - 8, c) - torch.where(c // 16 == 8, 128, 0)  # noqa: E731  (-0 as 0)
    assert torch.equal(zero(got_c.int()), zero(want_c.int()))
    for out in (torch.bfloat16, torch.float32):
        ko, vo = gather_paged_kv_fp4(cache, *args, out)
        for got, x in ((ko, k), (vo, v)):
            assert got.dtype == out and same_values(got.double().cpu(), from_fp4(*to_fp4(x)))  # (a block with an fp16 inf is NaN)
    braidinfer_amd.check_device_status()


def test_values_at_the_edges_of_the_format():
    """Ties, the steps of the scale, zeros, tiny and subnormal values, the largest, and
    blocks with an infinity or a NaN, whose neighbours are not touched."""
    rows = [torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4), torch.tensor([-0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 6.0] * 4),
            torch.tensor([6.0] + [6.0 * 2.0 ** -k for k in range(31)]), torch.tensor([6.0625] + [0.5] * 31),
            torch.tensor([3.0] + [0.1] * 31), torch.tensor([3.015625] + [0.25] * 31), torch.zeros(32),
            torch.tensor([2.0 ** -126, 2.0 ** -127, 2.0 ** -128, -2.0 ** -127] * 8), torch.tensor([3.0 * 2.0 ** 126] + [2.0 ** 126] * 31),
            torch.tensor([torch.finfo(torch.bfloat16).max] + [2.0 ** 127] * 31), torch.tensor([math.inf] + [1.0] * 31),
            torch.tensor([1.0] * 31 + [math.nan]), torch.tensor([-math.inf, math.nan] + [0.0] * 30), torch.tensor([-0.0] * 32)]
    x = torch.stack(rows).reshape(1, 1, -1)
    x = torch.cat((x, torch.ones(1, 1, 64)), -1)  # an even number of blocks, the last ones ordinary
    for dtype in (torch.float32, torch.bfloat16):
        xd = x.to(dtype)
        cache = new_cache(1, 1, 4, xd.shape[-1])
        idx, pos = torch.zeros(1, dtype=torch.int32, device=DEV), torch.tensor([2], device=DEV)
        append_paged_kv_fp4(xd.to(DEV), xd.neg().to(DEV), cache, idx, None, None, pos)
        for i, y in enumerate((xd, xd.neg())):
            c, s = to_fp4(y)
            assert torch.equal(cache.scales[0, i, 0, 2].cpu(), s[0, 0]), dtype
            assert same_values(from_fp4(cache.codes[0, i, 0, 2], cache.scales[0, i, 0, 2]), from_fp4(c, s)[0, 0]), dtype
        k, _ = gather_paged_kv_fp4(cache, idx, None, None, pos, torch.float32)
        # (the largest bf16 rounds to 4 x 2^126, which is past fp32)
        assert same_values(k.double().cpu(), from_fp4(*to_fp4(xd)).float().double())


def test_strided_heads_unaligned_rows_and_a_slice_of_the_cache():
    g = gen(3)
    t, heads, d = 21, 2, 64
    buf = randn(g, t, 3 * heads, d + 1).to(DEV)
    k, v = buf[:, :heads, 1:], buf[:, heads: 2 * heads, :d]  # unaligned; an odd token stride
    big = new_cache(5, 2 * heads, 16, d)
    cache = Fp4KVCache(big.codes[:, :, 1::2], big.scales[:, :, 1::2])
    idx, pos = torch.tensor([3, -1], device=DEV), torch.arange(5, 5 + t, device=DEV, dtype=torch.int32)
    append_paged_kv_fp4(k, v, cache, idx, None, None, pos)
    ko, vo = gather_paged_kv_fp4(cache, idx, None, None, pos, torch.float32)
    assert torch.equal(ko.double().cpu(), from_fp4(*to_fp4(k.cpu()))) and torch.equal(vo.double().cpu(), from_fp4(*to_fp4(v.cpu())))
    assert bool((big.codes[:, :, 0::2] == 0x5A).all()) and bool((big.scales[:, :, 0::2] == 0x5A).all())
    braidinfer_amd.check_device_status()


def test_the_same_slots_as_the_16_bit_append():
    """Random page tables, negative ids and positions included: the tokens land where
    append_paged_kv_batch puts them."""
    g = gen(4)
    heads, d, ps, pages = 2, 64, 8, 40
    idx = torch.randperm(pages, generator=g)[:30]
    idx = torch.where(torch.arange(30) % 3 == 0, idx - pages, idx).to(torch.int32).to(DEV)
    indptr = torch.tensor([0, 10, 10, 30], dtype=torch.int32, device=DEV)
    owner = torch.cat((torch.zeros(30, dtype=torch.long), torch.full((50,), 2))).to(DEV)
    pos = torch.cat((torch.randperm(80, generator=g)[:30], torch.randperm(160, generator=g)[:50])).to(DEV)
    k, v = randn(g, 80, heads, d).to(DEV), randn(g, 80, heads, d).to(DEV)
    wide = torch.zeros(pages, 2, heads, ps, d, dtype=torch.bfloat16, device=DEV)
    append_paged_kv_batch(k, v, wide, idx, indptr, owner, pos, ps)
    cache = Fp4KVCache(torch.zeros(pages, 2, heads, ps, d // 2, dtype=torch.uint8, device=DEV),
                       torch.full((pages, 2, heads, ps, d // 32), 127, dtype=torch.uint8, device=DEV))
    append_paged_kv_fp4(k, v, cache, idx, indptr, owner, pos)
    assert torch.equal(from_fp4(cache.codes, cache.scales), from_fp4(*to_fp4(wide.cpu())))
    braidinfer_amd.check_device_status()


def test_tokens_without_a_place():
    """Padding is skipped without a word, a token past its pages with a warning, and
    broken requests and pages raise; none of them writes."""
    g = gen(5)
    k = randn(g, 1, 1, 32).to(DEV)
    idx, indptr = torch.tensor([1, 7], dtype=torch.int32, device=DEV), torch.tensor([0, 2], dtype=torch.int32, device=DEV)

    def put(owner, pos, indptr=indptr):
        cache = new_cache(3, 1, 4, 32)
        args = (idx, indptr, torch.tensor([owner], device=DEV), torch.tensor([pos], device=DEV))
        append_paged_kv_fp4(k, k, cache, *args)
        ko, vo = gather_paged_kv_fp4(cache, *args)
        wrote = not bool((cache.codes == 0x5A).all() and (cache.scales == 0x5A).all())
        assert wrote == bool(ko.any()) == bool(vo.any())
        return wrote

    assert put(0, 3)
    assert not put(-1, 0)
    braidinfer_amd.check_device_status()
    assert not put(0, 8)
    with warnings.catch_warnings(record=True) as seen:
        warnings.simplefilter("always")
        braidinfer_amd.check_device_status()
    assert len(seen) == 1
    for owner, pos, ptr in ((0, 4, indptr), (1, 0, indptr), (-2, 0, indptr), (0, -9, indptr),
                            (0, 0, torch.tensor([5, 6], dtype=torch.int32, device=DEV)),
                            (0, 0, torch.tensor([-2, 6], dtype=torch.int32, device=DEV))):
        assert not put(owner, pos, ptr)
        with pytest.raises(IndexError):
            braidinfer_amd.check_device_status()


def test_no_tokens():
    cache = new_cache(2, 1, 4, 64)
    empty = torch.empty(0, dtype=torch.int64, device=DEV)
    append_paged_kv_fp4(torch.empty(0, 1, 64, device=DEV), torch.empty(0, 1, 64, device=DEV), cache, empty, None, None, empty)
    k, v = gather_paged_kv_fp4(cache, empty, None, None, empty)
    assert k.shape == v.shape == (0, 1, 64)
