"""The batched serving operators' checks of their arguments, which need no GPU: they
raise before anything is launched, and a call of no tokens ends there."""
from __future__ import annotations

import ctypes

import pytest
import torch

from braidinfer_amd import _lib
from braidinfer_amd.kernels import (Fp4KVCache, append_paged_kv_fp4, build_paged_kv_batch, gather_paged_kv_fp4)
from braidinfer_amd.layers import paged_attention, qk_norm_rope

I32 = torch.int32
BF16 = torch.bfloat16


def attention_args(**change):
    a = dict(query=torch.zeros(3, 8, 64, dtype=BF16), kv_cache=torch.zeros(4, 2, 2, 16, 64, dtype=BF16),
             kv_indices=torch.zeros(2, dtype=I32), kv_indptr=torch.zeros(3, dtype=I32),
             kv_last_page_len=torch.zeros(2, dtype=I32), qo_indptr=torch.zeros(3, dtype=I32))
    a.update(change)
    return a


@pytest.mark.parametrize("change,error,match", [
    (dict(query=torch.zeros(3, 512, dtype=BF16)), ValueError, "tokens, heads"),
    (dict(query=torch.zeros(3, 8, 64)), TypeError, "bf16 or fp16"),
    (dict(query=torch.zeros(3, 8, 64, dtype=torch.float16)), TypeError, "share a dtype"),
    (dict(query=torch.zeros(3, 7, 64, dtype=BF16)), ValueError, "evenly"),
    (dict(query=torch.zeros(3, 8, 128, dtype=BF16)), ValueError, "64 elements"),
    (dict(query=torch.zeros(3, 8, 96, dtype=BF16), kv_cache=torch.zeros(4, 2, 2, 16, 96, dtype=BF16)), ValueError, "head_dim 96"),
    (dict(kv_cache=torch.zeros(4, 3, 2, 16, 64, dtype=BF16)), ValueError, "one layer"),
    (dict(kv_cache=torch.zeros(4, 2, 2, 0, 64, dtype=BF16)), ValueError, "no slots"),
    (dict(kv_cache=torch.zeros(4, 2, 2, 16, 68, dtype=BF16)[..., :64]), ValueError, "multiples of 16 bytes"),
    (dict(kv_layout="DHN"), ValueError, "kv_layout"),
    (dict(kv_cache=Fp4KVCache.empty(4, 2, 16, 64, device="cpu"), kv_layout="NHD"), ValueError, "HND"),
    (dict(window=0), ValueError, "window"),
    (dict(num_sinks=-1), ValueError, "num_sinks"),
    (dict(kv_indices=torch.zeros(2, dtype=torch.int64)), TypeError, "kv_indices"),
    (dict(kv_indptr=torch.zeros(2, dtype=I32)), ValueError, "kv_indptr"),
    (dict(qo_indptr=torch.zeros(4, dtype=I32)), ValueError, "qo_indptr"),
    (dict(kv_last_page_len=torch.zeros(2, 1, dtype=I32)), (TypeError, ValueError), "kv_"),
    (dict(), RuntimeError, "ROCm"),
])
def test_attention_refuses(change, error, match):
    with pytest.raises(error, match=match):
        paged_attention(**attention_args(**change))


def test_attention_out_is_checked(monkeypatch):
    monkeypatch.setattr(_lib, "require_device", lambda *t: torch.device("cpu"))
    for out in (torch.zeros(3, 512), torch.zeros(2, 512, dtype=BF16), torch.zeros(3, 516, dtype=BF16)[:, :512]):
        with pytest.raises(ValueError, match="out must be"):
            paged_attention(**attention_args(out=out))
    assert paged_attention(**attention_args(query=torch.zeros(0, 8, 64, dtype=BF16))).shape == (0, 512)


def rc(name, *args):
    code = getattr(_lib.load(), name)(*args)
    return code, _lib.load().bfa_last_error().decode()


def entry_args(**change):
    """bfa_paged_attention's arguments; the pointers are never read on these paths."""
    base = (ctypes.c_char * 64)()
    p = (ctypes.addressof(base) + 15) // 16 * 16
    a = dict(query=p, dtype=_lib.BF16, tokens=3, hq=8, q_st=512, q_sh=64, cache=p, cache_dtype=_lib.BF16, pages=4, hkv=2,
             ps=16, d=64, sp=4096, skv=2048, sh=1024, ss=64, scales=None, ssp=0, sskv=0, ssh=0, sss=0, indices=p,
             num_indices=8, indptr=p, last=p, qo=p, seqs=2, scale=0.125, window=0, sinks=0, out=p, out_st=512, ws=None,
             ws_bytes=0, status=None, stream=None)
    a.update(change)
    return tuple(a.values())


@pytest.mark.parametrize("change,code,match", [
    (dict(dtype=_lib.F32), -1, "bf16 or fp16"), (dict(cache_dtype=_lib.F16), -1, "queries' dtype"),
    (dict(d=80), -2, "head_dim"), (dict(hq=7), -1, "evenly"), (dict(tokens=-1), -1, "geometry"),
    (dict(hkv=0), -1, "geometry"), (dict(ps=0), -1, "geometry"), (dict(pages=-1), -1, "negative"),
    (dict(window=-1), -1, "negative"), (dict(sinks=-1), -1, "negative"), (dict(ss=-64), -1, "negative cache strides"),
    (dict(q_st=4), -1, "aligned"), (dict(sh=12), -1, "aligned"), (dict(query=8), -1, "aligned"),
    (dict(num_indices=1 << 28), -1, "cached tokens"), (dict(tokens=1 << 28), -1, "query rows"),
    (dict(query=None), -1, "null pointer"), (dict(indices=None), -1, "null cache"), (dict(cache=None), -1, "null cache"),
    (dict(pages=0), -1, "null cache"), (dict(sp=1 << 40, pages=2), -1, "64 GiB"), (dict(pages=1 << 30), -1, "64 GiB"),
    (dict(cache_dtype=_lib.FP4, sp=2048, skv=1024, sh=512, ss=32), -1, "null cache"),
    (dict(cache_dtype=_lib.FP4, sp=2048, skv=1024, sh=512, ss=24), -1, "aligned"),
    (dict(num_indices=4096), -1, "workspace"),
])
def test_attention_entry_refuses(change, code, match):
    got, text = rc("bfa_paged_attention", *entry_args(**change))
    assert got == code and match in text, text


def test_attention_entry_of_no_rows():
    assert rc("bfa_paged_attention", *entry_args(tokens=0, query=None, out=None))[0] == 0
    assert rc("bfa_paged_attention", *entry_args(seqs=0))[0] == 0


def test_workspace_follows_the_work():
    size = lambda *a: _lib.workspace_size("bfa_paged_attention_workspace_size", *a)  # noqa: E731
    assert size(64, 64, 32, 8, 128, 16000, 16, 0, 0, _lib.BF16) > 0
    assert size(1, 1, 32, 8, 128, 2, 16, 0, 0, _lib.BF16) == 0     # a few keys: one workgroup a head
    assert size(8192, 1, 32, 8, 128, 512, 16, 0, 0, _lib.BF16) == 0  # enough blocks without splits
    assert size(0, 1, 32, 8, 128, 512, 16, 0, 0, _lib.BF16) == 0
    assert size(1, 1, 32, 8, 96, 512, 16, 0, 0, _lib.BF16) == 0    # refused by the call itself


def test_cache_shapes():
    c = Fp4KVCache.empty(3, 2, 16, 96, device="cpu")
    assert c.codes.shape == (3, 2, 2, 16, 48) and c.scales.shape == (3, 2, 2, 16, 3)
    assert (c.num_pages, c.num_kv_heads, c.page_size, c.head_dim) == (3, 2, 16, 96)
    with pytest.raises(ValueError, match="multiple of 32"):
        Fp4KVCache.empty(3, 2, 16, 80, device="cpu")
    with pytest.raises(TypeError, match="uint8"):
        Fp4KVCache(c.codes.int(), c.scales)
    for codes, scales in ((c.codes[:2], c.scales), (c.codes[..., :32], c.scales), (c.codes[:, :1], c.scales[:, :1])):
        with pytest.raises(ValueError, match="must be"):
            Fp4KVCache(codes, scales)
    with pytest.raises(ValueError, match="unit stride"):
        Fp4KVCache(torch.empty(3, 2, 2, 16, 96, dtype=torch.uint8)[..., ::2], c.scales)


def cache_args(**change):
    a = dict(k=torch.zeros(5, 2, 64, dtype=BF16), v=torch.zeros(5, 2, 64, dtype=BF16),
             cache=Fp4KVCache.empty(4, 2, 16, 64, device="cpu"), kv_indices=torch.zeros(4, dtype=I32),
             kv_indptr=torch.zeros(2, dtype=I32), batch_indices=torch.zeros(5, dtype=I32), positions=torch.zeros(5, dtype=I32))
    a.update(change)
    return a


@pytest.mark.parametrize("change,error,match", [
    (dict(k=torch.zeros(5, 2, 32, dtype=BF16)), ValueError, "k of shape"),
    (dict(v=torch.zeros(4, 2, 64, dtype=BF16)), ValueError, "v of shape"),
    (dict(v=torch.zeros(5, 2, 64)), TypeError, "share a dtype"),
    (dict(k=torch.zeros(5, 2, 64, dtype=I32), v=torch.zeros(5, 2, 64, dtype=I32)), TypeError, "bf16, fp16 or fp32"),
    (dict(positions=torch.zeros(4, dtype=I32)), IndexError, "positions"),
    (dict(positions=torch.zeros(5)), TypeError, "positions"),
    (dict(batch_indices=torch.zeros(6, dtype=I32)), IndexError, "batch indices"),
    (dict(batch_indices=None), ValueError, "together"), (dict(kv_indptr=None), ValueError, "together"),
    (dict(kv_indptr=torch.zeros(2, dtype=torch.int64)), TypeError, "kv_indptr"),
    (dict(kv_indices=torch.zeros(2, 2, dtype=I32)), ValueError, "one-dimensional"),
    (dict(cache=Fp4KVCache.empty(4, 2, 0, 64, device="cpu")), ValueError, "no slots"),
    (dict(), RuntimeError, "ROCm"),
])
def test_append_and_gather_refuse(change, error, match):
    a = cache_args(**change)
    with pytest.raises(error, match=match):
        append_paged_kv_fp4(**a)
    if not {"k", "v"} & set(change):
        if "positions" in change and change["positions"].shape[0] == 4:
            a["batch_indices"] = torch.zeros(7, dtype=I32)  # (the gather takes its count from positions)
            match = "batch indices"
        a.pop("k"), a.pop("v")
        with pytest.raises(error, match=match):
            gather_paged_kv_fp4(**a)
    with pytest.raises(TypeError):
        gather_paged_kv_fp4(a["cache"], a["kv_indices"], None, None, a["positions"], torch.int32)


def test_a_cache_keeps_its_tensors():
    """Calls take the sizes and strides from the time it was made."""
    cache = Fp4KVCache(torch.zeros(2, 2, 1, 16, 32, dtype=torch.uint8), torch.zeros(2, 2, 1, 16, 2, dtype=torch.uint8))
    assert (cache.num_pages, cache.num_kv_heads, cache.page_size, cache.head_dim) == (2, 1, 16, 64)
    with pytest.raises(AttributeError, match="make another"):
        cache.codes = torch.zeros(1, 2, 1, 16, 32, dtype=torch.uint8)


def test_calls_past_a_launch_are_refused():
    """2^24 workgroups of 256 threads are the 2^32 threads that one launch has at most."""
    got, text = rc("bfa_paged_attention", *entry_args(tokens=1 << 23, seqs=1 << 23))
    assert got == -1 and "too many query rows" in text
    a = dict(q=16, qh=1, qt=64, qs=64, qo=16, k=16, kh=0, kt=0, ks=0, ko=16, dt=_lib.BF16, tokens=1 << 26, d=62, qw=None,
             kw=None, wdt=0, eps=1e-6, pos=16, pdt=_lib.I64, table=16, most=8, status=None, stream=None)
    got, text = rc("bfa_qk_norm_rope", *a.values())
    assert got == -1 and "too many rows" in text
    got, text = rc("bfa_build_paged_kv_batch", 16, _lib.I32, 1 << 24, 1, 1, 16, _lib.I32, 16, _lib.I32, 16, 1, 1, 16, 16, 16,
                   16, 16, 16, 16, None, None)
    assert got == -1 and "2^24 requests" in text


def test_fp4_entry_refuses():
    base = (ctypes.c_char * 64)()
    p = (ctypes.addressof(base) + 15) // 16 * 16

    def append(**change):
        a = dict(k=p, v=p, dt=_lib.BF16, tokens=1, heads=2, d=64, kt=128, kh=64, vt=128, vh=64, codes=p, scales=p, pages=4,
                 ps=16, sp=2048, skv=1024, sh=512, ss=32, ssp=128, sskv=64, ssh=32, sss=2, idx=p, idx_dt=_lib.I32, n=4,
                 indptr=None, batch=None, batch_dt=0, seqs=0, pos=p, pos_dt=_lib.I32, status=None, stream=None)
        a.update(change)
        return rc("bfa_append_paged_kv_fp4", *a.values())

    for change, match in ((dict(dt=_lib.I32), "bad dtype"), (dict(d=48), "multiple of 32"), (dict(ss=30), "multiples of 4"),
                          (dict(codes=p + 2), "4-byte"), (dict(ps=0), "page_size"), (dict(k=None), "null pointer"),
                          (dict(scales=None), "null pointer"), (dict(idx=None), "null kv_indices"), (dict(pos=None), "null pointer"),
                          (dict(idx_dt=_lib.F32), "kv_indices"), (dict(pos_dt=_lib.F32), "positions"),
                          (dict(indptr=p), "batch_indices"), (dict(tokens=1 << 28), "too many"), (dict(tokens=-1), "geometry")):
        code, text = append(**change)
        assert code == -1 and match in text, (change, text)
    assert append(tokens=0, k=None)[0] == 0


@pytest.mark.parametrize("change,error,match", [
    (dict(page_tables=torch.zeros(6, dtype=I32)), ValueError, "max_pages"),
    (dict(seq_lens=torch.zeros(3, dtype=I32)), ValueError, "seq_lens"),
    (dict(query_lens=torch.zeros(2)), TypeError, "query_lens"),
    (dict(page_size=0), ValueError, "page_size"), (dict(num_tokens=-1), ValueError, "num_tokens"),
    (dict(), RuntimeError, "ROCm"),
])
def test_batch_refuses(change, error, match):
    a = dict(page_tables=torch.zeros(2, 3, dtype=I32), seq_lens=torch.zeros(2, dtype=I32),
             query_lens=torch.zeros(2, dtype=I32), page_size=16, num_tokens=2)
    a.update(change)
    with pytest.raises(error, match=match):
        build_paged_kv_batch(**a)


def test_batch_entry_refuses():
    def batch(**change):
        a = dict(tables=16, tdt=_lib.I32, seqs=2, width=3, stride=3, seq=16, sdt=_lib.I32, query=16, qdt=_lib.I32, ps=16,
                 tokens=4, indices=6, qo=16, kv=16, idx=16, last=16, batch=16, pos=16, slots=16, status=None, stream=None)
        a.update(change)
        return rc("bfa_build_paged_kv_batch", *a.values())

    for change, match in ((dict(tdt=_lib.F32), "int32/int64"), (dict(seqs=-1), "geometry"), (dict(ps=0), "page_size"),
                          (dict(tokens=1 << 30), "2^30 requests"), (dict(seq=None), "null pointer"),
                          (dict(kv=None), "null pointer"), (dict(slots=None), "null output"), (dict(idx=None), "null output")):
        code, text = batch(**change)
        assert code == -1 and match in text, (change, text)


@pytest.mark.parametrize("change,error,match", [
    (dict(query=torch.zeros(3, 130, dtype=BF16)), ValueError, "query of shape"),
    (dict(key=torch.zeros(2, 64, dtype=BF16)), ValueError, "key of shape"),
    (dict(key=torch.zeros(3, 64)), TypeError, "share a dtype"),
    (dict(query=torch.zeros(3, 128, dtype=I32), key=torch.zeros(3, 64, dtype=I32)), TypeError, "bf16, fp16 or fp32"),
    (dict(q_norm_weight=torch.ones(32)), ValueError, "head_dim = 64"),
    (dict(q_norm_weight=torch.ones(64), k_norm_weight=torch.ones(64, dtype=BF16)), TypeError, "share a dtype"),
    (dict(positions=torch.zeros(3)), ValueError, "positions"), (dict(positions=torch.zeros(1, 3, dtype=I32)), ValueError, "positions"),
    (dict(cos_sin_cache=torch.zeros(8, 64, dtype=BF16)), ValueError, "cos_sin_cache"),
    (dict(cos_sin_cache=torch.zeros(8, 63)), ValueError, "even"),
    (dict(), RuntimeError, "ROCm"),
])
def test_qk_norm_rope_refuses(change, error, match):
    a = dict(query=torch.zeros(3, 128, dtype=BF16), key=torch.zeros(3, 64, dtype=BF16), q_norm_weight=None,
             k_norm_weight=None, positions=torch.zeros(3, dtype=I32), cos_sin_cache=torch.zeros(8, 64))
    a.update(change)
    with pytest.raises(error, match=match):
        qk_norm_rope(**a)


def test_qk_norm_rope_entry_refuses():
    def call(**change):
        a = dict(q=16, qh=2, qt=128, qs=64, qo=16, k=16, kh=1, kt=64, ks=64, ko=16, dt=_lib.BF16, tokens=3, d=64, qw=None,
                 kw=None, wdt=0, eps=1e-6, pos=16, pdt=_lib.I64, table=16, most=8, status=None, stream=None)
        a.update(change)
        return rc("bfa_qk_norm_rope", *a.values())

    for change, match in ((dict(dt=_lib.I32), "bad dtype"), (dict(qw=16, wdt=_lib.I32), "weight dtype"), (dict(d=63), "even"),
                          (dict(pdt=_lib.F32), "positions"), (dict(tokens=1 << 30), "2^31 rows"), (dict(q=None), "null pointer"),
                          (dict(table=None), "null pointer"), (dict(most=0), "empty rotary table"), (dict(tokens=-1), "geometry")):
        code, text = call(**change)
        assert code == -1 and match in text, (change, text)
    assert call(tokens=0, q=None)[0] == 0
