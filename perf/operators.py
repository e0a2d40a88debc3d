"""Performance cases of the batched serving path: what an engine calls between a layer's QKV projection
and its output projection when many requests share one paged cache.

Five operators, each case one pass through one of them:

* ``batch``   page lists, token positions and cache slots of a step from the requests' lengths
* ``qk_rope`` RMSNorm of every query and key head and the rotation by position, in one pass
* ``window``  attention of a ragged batch over a 16-bit paged cache, where a token sees the last ``window``
  tokens and the first ``sinks``
* ``append4`` new keys and values written to a cache held in 4 bits, and read back as the values stored
* ``attn4``   attention of a ragged batch over that cache

The 4-bit cache holds E2M1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), two to a byte with the even element
low, and for each 32 elements of a head's row the exponent of their power-of-two scale, plus 127, in a byte: the
smallest scale that keeps the largest magnitude within 6.
"""
from __future__ import annotations

import functools
import math
import random
from types import SimpleNamespace

import torch

own = False

PAGE = 16
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
# q heads, kv heads, head_dim, rope theta, table length, eps
MODELS = {
    "tinyllama": SimpleNamespace(hq=32, hkv=4, d=64, theta=1e4, maxpos=4096, eps=1e-5),
    "qwen3": SimpleNamespace(hq=16, hkv=8, d=128, theta=1e6, maxpos=40960, eps=1e-6),
    "llama3": SimpleNamespace(hq=32, hkv=8, d=128, theta=5e5, maxpos=8192, eps=1e-5),
}


def listed():
    return [
        # the plan of one decode step: 64 running requests, one new token each
        dict(name="batch_decode_b64", op="batch", batch=64, context=4000, new=1),
        # the plan of a full engine's step: a thousand requests, some decoding, some with a piece of prompt
        dict(name="batch_mixed_b1000", op="batch", batch=1000, context=8000, new=24),
        # a few interactive users, fp16: latency of one call
        dict(name="qk_rope_tinyllama_t5_fp16", op="qk_rope", model="tinyllama", dtype="fp16", tokens=5),
        # a long prefill
        dict(name="qk_rope_qwen3_t8192", op="qk_rope", model="qwen3", dtype="bf16", tokens=8192),
        # a few interactive users decoding with a short window, fp16, tokens before heads in the cache
        dict(name="window_tinyllama_b5_fp16", op="window", model="tinyllama", dtype="fp16", layout="NHD", batch=5,
             context=2000, new=1, window=500, sinks=4),
        # a full decode batch whose longer requests have outgrown the window
        dict(name="window_llama3_b64", op="window", model="llama3", dtype="bf16", layout="HND", batch=64,
             context=16000, new=1, window=4000, sinks=4),
        # three prompts of odd lengths that arrived together
        dict(name="window_qwen3_prompts", op="window", model="qwen3", dtype="bf16", layout="HND", batch=3,
             context=300, new=300, window=130, sinks=16),
        # a long prompt in one piece
        dict(name="window_llama3_t8192", op="window", model="llama3", dtype="bf16", layout="HND", batch=1,
             context=8192, new=8192, window=4096, sinks=4),
        # the new tokens of a full decode batch
        dict(name="append4_llama3_b64", op="append4", model="llama3", dtype="bf16", batch=64, context=2000, new=1),
        # a long prompt
        dict(name="append4_qwen3_t6000", op="append4", model="qwen3", dtype="bf16", batch=1, context=6000, new=6000),
        # a full decode batch over the 4-bit cache
        dict(name="attn4_llama3_b64", op="attn4", model="llama3", dtype="bf16", batch=64, context=8000, new=1),
        # a piece of a prompt over a long cached context
        dict(name="attn4_qwen3_t1000", op="attn4", model="qwen3", dtype="bf16", batch=1, context=9000, new=1000),
    ]


def _spread(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["batch", "qk_rope", "window", "window", "append4", "attn4", "attn4"])
    case = dict(op=op)
    if op == "batch":
        case.update(batch=_spread(rng, 1, 1000), context=_spread(rng, 50, 8000), new=_spread(rng, 1, 24))
        return case
    case.update(model=rng.choice(sorted(MODELS)), dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if op == "qk_rope":
        case.update(tokens=_spread(rng, 1, 8192))
    elif op == "append4":
        batch = _spread(rng, 1, 64)
        new = _spread(rng, 1, 6000 // batch)
        case.update(batch=batch, context=_spread(rng, new, max(new, 2000)), new=new)
    else:
        kind = rng.choice(["decode", "decode", "prompts", "chunk"])
        if kind == "decode":
            batch, context, new = _spread(rng, 1, 64), _spread(rng, 20, 8000), 1
        elif kind == "prompts":
            batch = _spread(rng, 1, 8)
            context = new = _spread(rng, 2, 4000 // batch)
        else:
            batch, context, new = _spread(rng, 1, 3), _spread(rng, 1000, 8000), _spread(rng, 2, 600)
        case.update(batch=batch, context=context, new=new)
        if op == "window":
            case.update(layout=rng.choice(["HND", "NHD"]), window=_spread(rng, 16, 4096),
                        sinks=rng.choice([0, 1, 4, 16, 70]))
    return case


@functools.lru_cache(maxsize=64)
def _lengths(batch, context, new):
    """(tokens in the cache after the step, new ones among them) of every request: the first has the case's own
    figures, a batch of whole prompts has nothing cached before, and the others are spread below."""
    rng = random.Random("%d %d %d" % (batch, context, new))
    seq, query = [context], [new]
    for _ in range(1, batch):
        n = context if new == 1 else _spread(rng, 1, new)
        if context == new and new > 1:  # whole prompts
            seq.append(n)
            query.append(n)
        else:
            query.append(1 if new == 1 else n)
            seq.append(rng.randint(query[-1], context))
    return tuple(seq), tuple(query)


def _pages(n):
    return -(-n // PAGE)


# ------------------------------------------------------------------- inputs


class _Draw:
    """Seeded inputs on the GPU."""

    def __init__(self, seed):
        self.dev = torch.device("cuda", torch.cuda.current_device())
        self.g = torch.Generator(device=self.dev).manual_seed(seed)

    def randn(self, *shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=self.g, device=self.dev).mul_(std).add_(mean)

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device=self.dev, dtype=torch.int32)

    def ints(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.dev)


def _table(m, dev):
    inv = 1.0 / (m.theta ** (torch.arange(0, m.d, 2, dtype=torch.float64) / m.d))
    angle = torch.arange(m.maxpos, dtype=torch.float64)[:, None] * inv
    return torch.cat((angle.cos(), angle.sin()), -1).float().to(dev)


_tables = functools.lru_cache(maxsize=8)(lambda model, dev: _table(MODELS[model], dev))


def _offsets(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def _requests(g, case):
    """The step's requests as the attention and the append take them: page list, its offsets, tokens on the last
    page, query offsets, and each new token's request and position."""
    seq, query = _lengths(case["batch"], case["context"], case["new"])
    pages = [_pages(n) for n in seq]
    s = SimpleNamespace(seq=seq, query=query, num_pages=sum(pages) + 3)
    s.kv_indptr, s.qo_indptr = g.ints(_offsets(pages)), g.ints(_offsets(query))
    s.kv_indices = g.perm(s.num_pages)[: sum(pages)].contiguous()
    s.kv_last = g.ints([n - (p - 1) * PAGE for n, p in zip(seq, pages)])
    s.tokens, s.longest, s.most = sum(query), max(seq), max(query)
    lens = torch.tensor(query, device=g.dev)
    s.batch_indices = torch.repeat_interleave(torch.arange(len(seq), device=g.dev), lens)
    first = torch.tensor(seq, device=g.dev) - lens - torch.tensor(_offsets(query)[:-1], device=g.dev)
    s.positions = torch.arange(s.tokens, device=g.dev) + first[s.batch_indices]
    return s


def _kv(g, *shape):
    """Keys or values: N(0, 1) with a few channels of each head well above the rest, as trained models have them."""
    x = g.randn(*shape)
    x[..., 3] *= 4
    x[..., shape[-1] // 2 + 5] *= 3
    return x


def _to_4_bits(x):
    """(codes, scale bytes) of x [..., D] float32; every step is exact but the rounding to a code, ties to even."""
    b = x.unflatten(-1, (-1, 32))
    mantissa, exponent = torch.frexp(b.abs().amax(-1))
    e = (exponent - torch.where(mantissa <= 0.75, 3, 2)).clamp(-126, 127)
    y = torch.ldexp(b, -e[..., None])
    a = y.abs()
    code = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
            + 8 * (y < 0)).flatten(-2)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).to(torch.uint8), (e + 127).to(torch.uint8)


def _from_4_bits(codes, scales):
    """The float32 values that codes [..., D / 2] and scales [..., D / 32] stand for."""
    value = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    scale = torch.ldexp(torch.ones((), device=codes.device), scales.int() - 127)
    return (value[code].unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)


def prepare(case, seed):
    g = _Draw(seed)
    op = case["op"]
    if op == "batch":
        seq, query = _lengths(case["batch"], case["context"], case["new"])
        width = _pages(max(seq)) + 2
        tables = g.perm(len(seq) * width).reshape(len(seq), width).contiguous()
        order = g.perm(len(seq)).long()  # which request has which length
        return SimpleNamespace(op=op, tables=tables, seq=g.ints(seq)[order].contiguous(),
                               query=g.ints(query)[order].contiguous(), tokens=sum(query) + 5)
    m, dtype = MODELS[case["model"]], DTYPES[case["dtype"]]
    if op == "qk_rope":
        t = case["tokens"]
        qkv = g.randn(t, (m.hq + 2 * m.hkv) * m.d).to(dtype)
        q, k, _ = qkv.split([m.hq * m.d, m.hkv * m.d, m.hkv * m.d], -1)
        return SimpleNamespace(op=op, m=m, q=q, k=k, qw=g.randn(m.d, std=0.2, mean=1.0).to(dtype),
                               kw=(g.randn(m.d, std=0.5).exp()).to(dtype), table=_tables(case["model"], g.dev),
                               positions=torch.randint(0, m.maxpos, (t,), generator=g.g, device=g.dev))
    s = _requests(g, case)
    s.op, s.m, s.dtype = op, m, dtype
    if op == "append4":
        s.k, s.v = (_kv(g, s.tokens, m.hkv, m.d).to(dtype) for _ in range(2))
        s.codes = torch.zeros(s.num_pages, 2, m.hkv, PAGE, m.d // 2, dtype=torch.uint8, device=g.dev)
        s.scales = torch.zeros(s.num_pages, 2, m.hkv, PAGE, m.d // 32, dtype=torch.uint8, device=g.dev)
        return s
    s.q = g.randn(s.tokens, m.hq, m.d, std=1.5).to(dtype)
    cache = _kv(g, s.num_pages, 2, m.hkv, PAGE, m.d).to(dtype)
    if op == "attn4":
        s.codes, s.scales = _to_4_bits(cache.float())
    else:
        s.layout, s.window, s.sinks = case["layout"], case["window"], case["sinks"]
        s.cache = cache if s.layout == "HND" else cache.transpose(2, 3).contiguous()
    return s


# --------------------------------------------------------------- plain forms


def _plain_batch(s):
    """The offsets by sums, and each place of the page list and of the token list by a search in them."""
    n, dev = s.seq.numel(), s.seq.device
    zero = torch.zeros(1, dtype=torch.int64, device=dev)
    pages = (s.seq + PAGE - 1) // PAGE
    kv_indptr, qo_indptr = (torch.cat((zero, c.cumsum(0))) for c in (pages, s.query))
    at = torch.arange(s.tables.numel(), device=dev)
    b = torch.searchsorted(kv_indptr[1:], at, right=True).clamp(max=n - 1)
    column = (at - kv_indptr[b]).clamp(max=s.tables.shape[1] - 1)
    kv_indices = torch.where(at < kv_indptr[-1], s.tables[b, column], -1)
    t = torch.arange(s.tokens, device=dev)
    b = torch.searchsorted(qo_indptr[1:], t, right=True).clamp(max=n - 1)
    live = t < qo_indptr[-1]
    position = torch.where(live, s.seq[b] - s.query[b] + t - qo_indptr[b], 0)
    slot = s.tables[b, position // PAGE].long() * PAGE + position % PAGE
    return (qo_indptr.int(), kv_indptr.int(), kv_indices.int(), (s.seq - (pages - 1).clamp(min=0) * PAGE).int(),
            torch.where(live, b, -1).int(), torch.where(live, position, -1), torch.where(live, slot, -1))


def _plain_qk_rope(s):
    angle = s.table[s.positions][:, None]
    c, n = angle.chunk(2, -1)

    def one(x, w):
        x = x.unflatten(-1, (-1, s.m.d)).float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s.m.eps) * w.float()
        a, b = x.chunk(2, -1)
        return torch.cat((a * c - b * n, b * c + a * n), -1).flatten(-2).to(s.q.dtype)

    return one(s.q, s.qw), one(s.k, s.kw)


def _plain_append4(s):
    page = s.kv_indices[s.kv_indptr[s.batch_indices] + s.positions // PAGE].long()
    slot = s.positions % PAGE
    out = []
    for i, x in enumerate((s.k, s.v)):
        codes, scales = _to_4_bits(x.float())
        s.codes[page, i, :, slot], s.scales[page, i, :, slot] = codes, scales
        out.append(_from_4_bits(s.codes[page, i, :, slot], s.scales[page, i, :, slot]).to(s.dtype))
    return tuple(out)


def _plain_attention(s, window, sinks):
    """Every request padded to the longest: gathered keys and values, masked scores, softmax, weighted sum."""
    m, n, dev = s.m, len(s.seq), s.q.device
    j = torch.arange(s.longest, device=dev)
    pages = s.kv_indptr.diff()
    length = (pages - 1) * PAGE + s.kv_last
    at = (s.kv_indptr[:-1, None] + j // PAGE).clamp(max=s.kv_indices.numel() - 1)
    page, slot = s.kv_indices[at].long(), (j % PAGE).expand(n, -1)
    if s.op == "attn4":
        k, v = (_from_4_bits(s.codes[page, i, :, slot], s.scales[page, i, :, slot]) for i in (0, 1))
    elif s.layout == "HND":
        k, v = s.cache[page, 0, :, slot].float(), s.cache[page, 1, :, slot].float()
    else:
        k, v = s.cache[page, 0, slot].float(), s.cache[page, 1, slot].float()
    k, v = (x.permute(0, 2, 1, 3).contiguous() for x in (k, v))  # [request, kv head, key, d]
    i = torch.arange(s.most, device=dev)
    count = s.qo_indptr.diff()
    q = s.q[(s.qo_indptr[:-1, None] + i).clamp(max=s.tokens - 1)].float()
    q = q.unflatten(2, (m.hkv, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [request, kv head, head of it x query, d]
    score = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(m.d ** -0.5).unflatten(2, (-1, s.most))
    position = (length - count)[:, None] + i
    seen = j <= position[..., None]
    if window is not None:
        seen &= (position[..., None] - j < window) | (j < sinks)
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (-1, s.most)) / torch.where(total == 0, 1.0, total)
    t = torch.arange(s.tokens, device=dev)
    o = o.permute(0, 3, 1, 2, 4)[s.batch_indices, t - s.qo_indptr[s.batch_indices]]
    return o.flatten(1).to(s.dtype)


# ---------------------------------------------------------------------- run


@functools.lru_cache(maxsize=None)
def _framework():
    from braidinfer_amd import kernels, layers
    return kernels, layers


def run(s):
    if own:
        kernels, layers = _framework()
        if s.op == "batch":
            return tuple(kernels.build_paged_kv_batch(s.tables, s.seq, s.query, PAGE, s.tokens))
        if s.op == "qk_rope":
            return layers.qk_norm_rope(s.q, s.k, s.qw, s.kw, s.positions, s.table, s.m.eps)
        if s.op == "append4":
            cache = kernels.Fp4KVCache(s.codes, s.scales)
            kernels.append_paged_kv_fp4(s.k, s.v, cache, s.kv_indices, s.kv_indptr, s.batch_indices, s.positions)
            return kernels.gather_paged_kv_fp4(cache, s.kv_indices, s.kv_indptr, s.batch_indices, s.positions, s.dtype)
        if s.op == "attn4":
            return layers.paged_attention(s.q, kernels.Fp4KVCache(s.codes, s.scales), s.kv_indices, s.kv_indptr,
                                          s.kv_last, s.qo_indptr)
        return layers.paged_attention(s.q, s.cache, s.kv_indices, s.kv_indptr, s.kv_last, s.qo_indptr,
                                      window=s.window, num_sinks=s.sinks, kv_layout=s.layout)
    if s.op == "batch":
        return _plain_batch(s)
    if s.op == "qk_rope":
        return _plain_qk_rope(s)
    if s.op == "append4":
        return _plain_append4(s)
    return _plain_attention(s, *((None, 0) if s.op == "attn4" else (s.window, s.sinks)))


def work(case):
    op = case["op"]
    if op == "qk_rope":
        m, t = MODELS[case["model"]], case["tokens"]
        row = (m.hq + m.hkv) * m.d
        return {"bytes": t * (2 * 2 * row + 4 * m.d + 8), "flops": 8 * t * row}
    seq, query = _lengths(case["batch"], case["context"], case["new"])
    tokens, pages = sum(query), sum(_pages(n) for n in seq)
    if op == "batch":  # lengths and used page ids in; offsets, page list, and three words a token out
        width = _pages(max(seq)) + 2
        return {"bytes": 8 * len(seq) + 4 * pages + 12 * len(seq) + 4 * len(seq) * width + 20 * (tokens + 5), "flops": 0}
    m = MODELS[case["model"]]
    if op == "append4":
        row = 2 * m.hkv * m.d
        return {"bytes": tokens * (4 * row + 2 * row * 17 // 32 + 16) + 4 * pages, "flops": 4 * tokens * row}
    window, sinks = (case["window"], case["sinks"]) if op == "window" else (1 << 60, 0)
    pairs = keys = 0
    for n, q in zip(seq, query):
        first = max(0, n - q + 1 - window)  # the first key that the window of any query holds
        keys += n - first + min(sinks, first)
        for p in range(n - q, n):
            low = max(0, p + 1 - window)
            pairs += p + 1 - low + min(sinks, low)
    per_key = 2 * m.hkv * (m.d * 17 // 32 if op == "attn4" else 2 * m.d)
    return {"bytes": keys * per_key + tokens * m.hq * m.d * 4 + 4 * pages, "flops": 4 * m.hq * m.d * pairs}


# -------------------------------------------------------------------- exact


def exact(case, seed):
    """From the definitions, in 64 bits: one request, head and token at a time where that helps."""
    s = prepare(case, seed)
    op = s.op
    if op == "batch":
        seq, query, tables = s.seq.tolist(), s.query.tolist(), s.tables.tolist()
        qo, kv, indices, last, owner, position, slot = [0], [0], [], [], [], [], []
        for b, (n, q) in enumerate(zip(seq, query)):
            used = math.ceil(n / PAGE)
            indices += tables[b][:used]
            kv.append(len(indices))
            last.append((n - 1) % PAGE + 1 if n else 0)
            for p in range(n - q, n):
                owner.append(b)
                position.append(p)
                slot.append(tables[b][p // PAGE] * PAGE + p % PAGE)
            qo.append(len(owner))
        pad = s.tokens - len(owner)
        indices += [-1] * (s.tables.numel() - len(indices))
        word, long = torch.int32, torch.int64
        return tuple(torch.tensor(x, dtype=d) for x, d in (
            (qo, word), (kv, word), (indices, word), (last, word), (owner + [-1] * pad, word),
            (position + [-1] * pad, long), (slot + [-1] * pad, long)))
    d = s.m.d
    if op == "qk_rope":
        cos, sin = (a.unsqueeze(1) for a in s.table.double()[s.positions].split(d // 2, -1))
        out = []
        for x, w in ((s.q, s.qw), (s.k, s.kw)):
            x = x.double().reshape(x.shape[0], -1, d)
            x = w.double() * x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / d + s.m.eps)
            lo, hi = x[..., : d // 2], x[..., d // 2:]
            out.append(torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1).reshape(x.shape[0], -1))
        return tuple(out)
    levels = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=s.kv_last.device)
    if op == "append4":
        out = []
        for x in (s.k, s.v):
            blocks = x.double().reshape(-1, 32)
            most = blocks.abs().max(-1, keepdim=True).values
            power = torch.ceil(torch.log2(most / 6))
            power = torch.where(most > 6 * 2.0 ** power, power + 1, torch.where(most <= 3 * 2.0 ** power, power - 1, power))
            y = blocks / 2.0 ** power
            gap = (y.abs()[..., None] - levels).abs()
            near = gap.min(-1, keepdim=True).values
            even = torch.tensor([0, 1] * 4, device=gap.device)  # of two equally near levels the one with an even code
            code = torch.where(gap == near, even, 2).argmin(-1)
            out.append((levels[code] * y.sign() * 2.0 ** power).reshape(x.shape))
        return tuple(out)
    window, sinks = (s.window, s.sinks) if op == "window" else (None, 0)
    out = torch.zeros(s.tokens, s.m.hq, d, dtype=torch.float64, device=s.q.device)
    group, at, page_at = s.m.hq // s.m.hkv, 0, 0
    for n, q in zip(s.seq, s.query):
        ids = s.kv_indices[page_at: page_at + _pages(n)].long()
        p = torch.arange(n - q, n, device=s.q.device)[:, None]
        j = torch.arange(n, device=s.q.device)
        hidden = j > p
        if window is not None:
            hidden = hidden | ((j <= p - window) & (j >= sinks))
        for h in range(s.m.hkv):
            rows = []
            for i in (0, 1):
                if op == "attn4":
                    raw = s.codes[ids, i, h].reshape(-1, d // 2)[:n].int()
                    raw = torch.stack([raw % 16, raw // 16], -1).reshape(n, d)
                    x = levels[raw % 8] * (1 - 2 * (raw // 8)).double()
                    power = s.scales[ids, i, h].reshape(-1, d // 32)[:n].double() - 127
                    x = x * torch.repeat_interleave(2.0 ** power, 32, -1)
                else:
                    x = s.cache[ids, i, h] if s.layout == "HND" else s.cache[ids, i, :, h]
                    x = x.reshape(-1, d)[:n].double()
                rows.append(x)
            for c in range(h * group, (h + 1) * group):
                z = s.q[at: at + q, c].double() @ rows[0].T / math.sqrt(d)
                z = z.masked_fill(hidden, -math.inf)
                out[at: at + q, c] = torch.softmax(z, -1) @ rows[1]
        at, page_at = at + q, page_at + _pages(n)
    return out.reshape(s.tokens, -1)
