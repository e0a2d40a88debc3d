"""RMSNorm of query and key heads with their rotation against the formula in 64 bits.

Allowance, u = half a step of the type: the mean of D squares in fp32 is off by at most
D 2^-24 of itself, its root by half that, and root, division and the two products of the
norm by 2^-24 each and 2 for the root's and the division's own error: r = (D / 2 + 8) 2^-24
of x'; the two products and the sum of the rotation add 2 x 2^-24 each of their terms.
With t = |x1' cos| + |x2' sin| the result is off by (r + 4 x 2^-24) t and u |y| for its own
rounding, and by 2^-24 where it is below the type's normal range (fp16)."""
from __future__ import annotations

import pytest
import torch

import braidinfer_amd
from braidinfer_amd.layers import RMSNorm, RotaryEmbedding, qk_norm_rope
from oracle import torch_ref as R
from tests.helpers import assert_close, gen, randn
from tests.paged_reference import half_step

pytestmark = pytest.mark.gpu
DEV = "cuda"


def reference(x, w, pos, table, eps, heads):
    d = table.shape[1]
    x = x.double().reshape(x.shape[0], heads, d)
    if w is not None:
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w.double()
    p = torch.where(pos < 0, pos + table.shape[0], pos)
    ok = (p >= 0) & (p < table.shape[0])
    c, s = table.double()[p.clamp(0, table.shape[0] - 1)][:, None].chunk(2, -1)
    a, b = x.chunk(2, -1)
    y = torch.cat((a * c - b * s, b * c + a * s), -1) * ok[:, None, None]
    t = torch.cat(((a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()), -1)
    return y, t


def check(got, x, w, pos, table, eps, heads, what):
    y, t = reference(x.cpu(), w.cpu() if w is not None else None, pos.cpu().long(), table.cpu(), eps, heads)
    d = table.shape[1]
    allow = (d / 2 + 12) * 2.0 ** -24 * t + half_step(x.dtype) * y.abs() + 2.0 ** -24
    off = (got.detach().cpu().double().reshape(y.shape) - y).abs()
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    assert bool((off <= allow).all()), f"{what}: {float((off / allow).max()):.2f} of the allowance"


DIMS = [(64, 32, 4), (128, 16, 8), (128, 1, 1), (256, 3, 1), (96, 5, 2), (80, 4, 4), (32, 6, 2), (16, 2, 1), (6, 3, 2), (1040, 1, 1)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,hq,hkv", DIMS)
def test_against_the_formula(dtype, d, hq, hkv):
    table = R.cos_sin_cache(d, 512, 1e4).to(DEV)
    for t in (1, 37):
        g = gen(d + hq + t)
        qkv = randn(g, t, (hq + 2 * hkv) * d, dtype=dtype).to(DEV)
        q, k, _ = qkv.split([hq * d, hkv * d, hkv * d], -1)
        qw, kw = randn(g, d, mean=1.0, std=0.2, dtype=dtype).to(DEV), randn(g, d, dtype=dtype).exp().to(DEV)
        pos = torch.randint(-512, 512, (t,), generator=g).to(DEV)
        qo, ko = qk_norm_rope(q, k, qw, kw, pos, table, 1e-6)
        check(qo, q, qw, pos, table, 1e-6, hq, "q")
        check(ko, k, kw, pos, table, 1e-6, hkv, "k")
    braidinfer_amd.check_device_status()


@pytest.mark.parametrize("off", [0, 1])
def test_views_weights_and_positions_of_other_kinds(off):
    """Three-dimensional strided views (an unaligned one among them), fp32 weights over
    bf16 heads, one norm or none, int32 positions; the inputs stay as they were."""
    g = gen(8)
    t, hq, hkv, d = 19, 4, 2, 64
    table = R.cos_sin_cache(d, 300, 1e6).to(DEV)
    buf = randn(g, t, hq + hkv, d + 9).to(DEV)
    q, k = buf[:, :hq, off: off + d], buf[:, hq:, off: off + d]
    before = buf.clone()
    w = randn(g, d, mean=1.0, dtype=torch.float32).to(DEV)
    pos = torch.randint(0, 300, (t,), generator=g, dtype=torch.int32).to(DEV)
    for qw, kw in ((w, w), (w, None), (None, w), (None, None)):
        qo, ko = qk_norm_rope(q, k, qw, kw, pos, table, 1e-5)
        check(qo, q, qw, pos, table, 1e-5, hq, "q")
        check(ko, k, kw, pos, table, 1e-5, hkv, "k")
    assert torch.equal(buf, before)
    wide = randn(g, d, 2, dtype=torch.float32).to(DEV)[:, 1]  # a strided weight
    qo, _ = qk_norm_rope(q, k, wide, wide, pos, table)
    check(qo, q, wide, pos, table, 1e-6, hq, "strided weight")
    braidinfer_amd.check_device_status()


def test_positions_past_the_table():
    g = gen(9)
    table = R.cos_sin_cache(64, 100, 1e4).to(DEV)
    q, k = randn(g, 4, 128).to(DEV), randn(g, 4, 64).to(DEV)
    pos = torch.tensor([100, 99, -100, -101], device=DEV)
    qo, ko = qk_norm_rope(q, k, None, None, pos, table)
    check(qo, q, None, pos, table, 1e-6, 2, "q")
    assert not qo[0].any() and not qo[3].any() and not ko[0].any() and qo[1].any()
    with pytest.raises(IndexError):
        braidinfer_amd.check_device_status()


def test_beside_the_three_calls():
    """What q_norm, k_norm and rotary_emb give, up to their rounding in between."""
    g = gen(10)
    t, hq, hkv, d = 50, 16, 8, 128
    rope = RotaryEmbedding(d, d, 2048, 1e6).to(DEV)
    qn, kn = RMSNorm(d).to(DEV, torch.bfloat16), RMSNorm(d).to(DEV, torch.bfloat16)
    with torch.no_grad():
        kn.weight.copy_(randn(g, d).exp())
    q, k = randn(g, t, hq, d).to(DEV), randn(g, t, hkv, d).to(DEV)
    pos = torch.randint(0, 2048, (t,), generator=g).to(DEV)
    eq, ek = rope(pos, qn(q.clone()), kn(k.clone()))
    gq, gk = qk_norm_rope(q, k, qn.weight, kn.weight, pos, rope.cos_sin_cache, qn.eps)
    # (two more roundings of each of a pair: three half steps of both at most)
    top = max(float(eq.abs().max()), float(ek.abs().max()))
    assert_close(gq, eq, atol=6 * 2.0 ** -8 * top, rtol=0, what="q")
    assert_close(gk, ek, atol=6 * 2.0 ** -8 * top, rtol=0, what="k")


def test_no_tokens_and_a_large_call():
    table = R.cos_sin_cache(64, 100, 1e4).to(DEV)
    q, k = qk_norm_rope(torch.empty(0, 128, device=DEV), torch.empty(0, 1, 64, device=DEV), None, None,
                        torch.empty(0, dtype=torch.int64, device=DEV), table)
    assert q.shape == (0, 128) and k.shape == (0, 1, 64)
    g = gen(11)
    t = 6001
    x = randn(g, t, 12 * 64).to(DEV)
    w = randn(g, 64, mean=1.0).to(DEV)
    pos = torch.randint(0, 100, (t,), generator=g).to(DEV)
    qo, ko = qk_norm_rope(x[:, :640], x[:, 640:], w, w, pos, table)
    check(qo, x[:, :640], w, pos, table, 1e-6, 10, "q")
    check(ko, x[:, 640:], w, pos, table, 1e-6, 2, "k")
