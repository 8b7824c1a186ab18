"""The 8-bit paged cache and the attentions over it, one call each, and attention of requests that share a prefix.

A cached key or value row x of one token and head (D numbers in bfloat16, the largest magnitude of them a) is held as
codes and one fp32 scale:

  int8   code = round(127 x / a), ties to even            value = code a / 127
  fp8    code = round(448 x / a) to E4M3, ties to even    value = code a / 448

A case is one call of one operator:

  write    rows of new tokens into the cache, and the same tokens read back (what the cache now holds)
  read     the cached tokens of requests as bfloat16, packed
  decode   attention of one new token of each request over its cached keys
  prompt   causal attention of packed prompt portions, their own keys and those before them in the cache
  shared   decode attention of groups of requests, each group's first keys in common (and in one place of the cache)

Head layouts are those of this repository's models and tests (query heads, key heads, size of a head). Pages of 16 tokens
are the engine's default, 32 the longer ones of its tests; they are handed out in a random order.
"""
import math

import torch

own = False

LAYOUTS = [(32, 8, 128), (8, 1, 128), (64, 8, 128), (32, 8, 64), (12, 12, 64), (16, 2, 64)]
LARGEST = {"fp8": 448.0, "int8": 127.0}


def _case(name, op, fmt, layout, **kw):
    """`spread`: how the lengths of the case's requests are made (`_lengths`)."""
    return dict(name=name, op=op, fmt=fmt, heads=layout[0], kv=layout[1], dim=layout[2], spread=0, **kw)


def listed():
    return [
        # the cache's part of one decode step of a full batch: a token each of 64 requests
        _case("write decode 64", "write", "fp8", (32, 8, 128), n=64, new_lo=1, new_hi=1, ctx_lo=512, ctx_hi=767, page=16),
        # the rows of a long step of ragged prompts
        _case("write prompts 8k", "write", "int8", (32, 8, 128), n=5, new_lo=1200, new_hi=2048, ctx_lo=0, ctx_hi=0, page=16),
        # one conversation taken out of the cache, to another replica
        _case("read 1x531", "read", "int8", (32, 8, 64), n=1, new_lo=531, new_hi=531, ctx_lo=0, ctx_hi=0, page=16),
        # the prefix cache of a busy server, for a kernel that reads bfloat16
        _case("read 33x2000", "read", "fp8", (32, 8, 128), n=33, new_lo=300, new_hi=4001, ctx_lo=0, ctx_hi=99, page=16),
        # one user on an idle server: latency
        _case("decode 1x640", "decode", "fp8", (32, 8, 128), n=1, new_lo=1, new_hi=1, ctx_lo=639, ctx_hi=639, page=16),
        # the benchmark's load: 64 requests of 512 prompt tokens within their output tokens
        _case("decode 64x640", "decode", "fp8", (32, 8, 128), n=64, new_lo=1, new_hi=1, ctx_lo=511, ctx_hi=766, page=16),
        # one rank of the 70B model: all query heads on one key head, long documents
        _case("decode 9x50k", "decode", "int8", (8, 1, 128), n=9, new_lo=1, new_hi=1, ctx_lo=20000, ctx_hi=80000, page=32),
        # the prompt of a new request that arrives while others run
        _case("prompt 512", "prompt", "fp8", (32, 8, 128), n=1, new_lo=512, new_hi=512, ctx_lo=0, ctx_hi=0, page=16),
        # later portions of long prompts
        _case("prompts 4x2048", "prompt", "int8", (32, 8, 128), n=4, new_lo=1900, new_hi=2048, ctx_lo=1000, ctx_hi=2048, page=16),
        # a chat service: 64 requests behind one long system prompt, the cache in bfloat16
        _case("shared 64x4096", "shared", "bf16", (32, 8, 128), groups=1, n=64, prefix_lo=4096, prefix_hi=4096, ctx_lo=33, ctx_hi=700, page=16),
        # few requests on one document of odd length
        _case("shared 6x1531", "shared", "fp8", (32, 8, 64), groups=1, n=6, prefix_lo=1531, prefix_hi=1531, ctx_lo=1, ctx_hi=60, page=16),
        # documents with many questions each
        _case("shared 5x27 docs", "shared", "fp8", (32, 8, 128), groups=5, n=27, prefix_lo=5000, prefix_hi=30000, ctx_lo=1, ctx_hi=900, page=16),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        c = _drawn(rng)
        if all(work(c)[k] <= most[k] for k in most):
            return c


def _drawn(rng):
    op = rng.choice(["write", "read", "decode", "prompt", "shared"])
    heads, kv, dim = rng.choice(LAYOUTS)
    c = dict(op=op, fmt=rng.choice(["fp8", "int8"]), heads=heads, kv=kv, dim=dim, spread=rng.randrange(1 << 20), page=rng.choice([16, 16, 32]))
    if op in ("write", "read"):
        if rng.random() < 0.4:   # a step of single tokens
            return dict(c, n=_log_uniform(rng, 1, 256), new_lo=1, new_hi=1, ctx_lo=0, ctx_hi=_log_uniform(rng, 16, 2000))
        n = _log_uniform(rng, 1, 33)
        hi = _log_uniform(rng, 2, (9000 if op == "write" else 60000) // n)
        return dict(c, n=n, new_lo=max(1, hi // 3), new_hi=hi, ctx_lo=0, ctx_hi=rng.choice([0, 99]))
    if op == "decode":
        n = _log_uniform(rng, 1, 128)
        hi = _log_uniform(rng, 16, 400000 // max(n, 5))
        return dict(c, n=n, new_lo=1, new_hi=1, ctx_lo=hi // rng.choice([1, 2, 8]), ctx_hi=hi)
    if op == "prompt":
        n = rng.randrange(1, 6)
        hi = _log_uniform(rng, 2, 8192 // n)
        return dict(c, n=n, new_lo=max(1, hi // 2), new_hi=hi, ctx_lo=0, ctx_hi=rng.choice([0, 0, 700, 2000]))
    groups = rng.randrange(1, 6)
    n = _log_uniform(rng, 1, 128 // groups)
    hi = _log_uniform(rng, 64, 60000 // groups)
    return dict(c, fmt=rng.choice(["bf16", "fp8", "int8"]), groups=groups, n=n, prefix_lo=hi // 2, prefix_hi=hi, ctx_lo=1, ctx_hi=_log_uniform(rng, 16, 1000))


# ------------------------------------------------------------------------------------------------ a case's requests and its cache
def _lengths(case, lo, hi, count, salt):
    """`count` lengths from lo to hi, plain values that come from the case alone."""
    return [lo + (case["spread"] + salt + 1 + i * 7919 + (i * i) % 13 * 101) % (hi - lo + 1) if hi > lo else lo for i in range(count)]


def _requests(case):
    """[(new tokens, tokens before them)], and for shared cases the sizes and prefixes of the groups."""
    if case["op"] != "shared":
        new = _lengths(case, case["new_lo"], case["new_hi"], case["n"], 0)
        return list(zip(new, _lengths(case, case["ctx_lo"], case["ctx_hi"], case["n"], 1))), None, None
    sizes = _lengths(case, max(1, case["n"] // 2), case["n"], case["groups"] - 1, 2) + [case["n"]]
    prefixes = _lengths(case, case["prefix_lo"], case["prefix_hi"], case["groups"], 3)
    reqs = []
    for g, (m, p) in enumerate(zip(sizes, prefixes)):
        reqs += [(1, p + t - 1) for t in _lengths(case, case["ctx_lo"], case["ctx_hi"], m, 4 + g)]
    return reqs, sizes, prefixes


def _pages(case, gen):
    """The requests' page tables [S, W] (int32, on the host) and the number of pages; requests of a group have the whole pages of
    their prefix in common, and their own copies of a page that the prefix fills in part."""
    reqs, sizes, prefixes = _requests(case)
    bs = case["page"]
    need = [-(-(q + c) // bs) for q, c in reqs]
    common, first = [0] * len(reqs), list(range(len(reqs)))
    if sizes:
        at = 0
        for m, p in zip(sizes, prefixes):
            for i in range(at, at + m):
                common[i], first[i] = (p // bs if i > at else 0), at
            at += m
    total = sum(n - c for n, c in zip(need, common)) + 1
    order = torch.randperm(total, generator=gen).to(torch.int32)
    tables = torch.zeros(len(reqs), max(need), dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        tables[i, :common[i]] = tables[first[i], :common[i]]
        tables[i, common[i]:n] = order[at:at + n - common[i]]
        at += n - common[i]
    return tables, total


def _rows(n, kv, dim, gen):
    """Keys or values as a model makes them: channels of different strength, some much stronger, tokens too."""
    dev = gen.device
    gain = torch.exp(0.5 * torch.randn(kv, dim, generator=gen, device=dev))
    gain[:, :: dim // 4] *= 3.0
    token = torch.exp(0.2 * torch.randn(n, 1, 1, generator=gen, device=dev))
    return (torch.randn(n, kv, dim, generator=gen, device=dev) * (gain / gain.square().mean(-1, keepdim=True).sqrt()) * token).to(torch.bfloat16)


def prepare(case, seed):
    dev = "cuda"
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device=dev).manual_seed(seed)
    reqs, sizes, prefixes = _requests(case)
    tables, blocks = _pages(case, host)
    bs, kv, dim = case["page"], case["kv"], case["dim"]
    # every slot of the cache holds a row: what no request owns is another's
    k, v = _rows(blocks * bs, kv, dim, gen), _rows(blocks * bs, kv, dim, gen)
    new = sum(q for q, _ in reqs)
    st = dict(case=case, tables=tables.to(dev), reqs=reqs, sizes=sizes, prefixes=prefixes)
    st["lens"] = torch.tensor([q + c for q, c in reqs], dtype=torch.int32, device=dev)
    st["starts"] = torch.tensor([c for _, c in reqs], dtype=torch.int32, device=dev)
    cu = [0]
    for q, _ in reqs:
        cu.append(cu[-1] + q)
    st["cu"], st["cu_host"] = torch.tensor(cu, dtype=torch.int32, device=dev), cu
    slots = torch.cat([tables[i].long()[(c + torch.arange(q)) // bs] * bs + (c + torch.arange(q)) % bs for i, (q, c) in enumerate(reqs)])
    st["slots"] = slots.to(dev, torch.int32)
    if case["op"] == "write":   # the projection's rows, keys and values side by side
        st["new_kv"] = torch.cat([_rows(new, kv, dim, gen), _rows(new, kv, dim, gen)], dim=1)
    if case["op"] in ("decode", "prompt", "shared"):
        st["q"] = (1.3 * torch.randn(new, case["heads"], dim, generator=gen, device=dev)).to(torch.bfloat16)
    if case["fmt"] == "bf16":
        st["kv"] = tuple(x.view(blocks, bs, kv, dim).transpose(1, 2).contiguous() for x in (k, v))
    elif own:
        from xgserve import ops
        cache = ops.QuantKVCache.alloc(blocks, kv, bs, dim, case["fmt"], dev)
        ops.kv_quant_append(k, v, cache, torch.arange(blocks * bs, dtype=torch.int32, device=dev))
        st["kv"] = cache
    else:
        st["kv"] = tuple(x.view(blocks, bs, *x.shape[1:]) for r in (k, v) for x in _quantise(r, case["fmt"]))
    if own and case["op"] == "shared":
        from xgserve import ops
        st["plan"] = ops.shared_prefix_plan(sizes, prefixes, case["heads"], kv, dev)
    return st


# ------------------------------------------------------------------------------------------------ the plain forms
def _quantise(x, fmt):
    """Codes (8 bits) and scales [n, heads] of rows [n, heads, D]. In 64 bits: 127 x / a may lie on the border of two codes."""
    a = x.abs().amax(-1, keepdim=True)
    y = (x.double() * LARGEST[fmt] / a.double()).masked_fill(a == 0, 0)
    codes = y.to(torch.float8_e4m3fn) if fmt == "fp8" else y.round().to(torch.int8)
    return codes, a[..., 0].float() / LARGEST[fmt]


def _rows_at(st, at):
    """Keys and values [n, heads, D] at slots `at` of the cache, in 32 bits."""
    bs = st["case"]["page"]
    pages, offs = at // bs, at % bs
    if st["case"]["fmt"] == "bf16":
        return tuple(x[pages, :, offs].float() for x in st["kv"])
    k, ks, v, vs = st["kv"]
    return k[pages, offs].float() * ks[pages, offs][..., None], v[pages, offs].float() * vs[pages, offs][..., None]


def _tokens(st, i, lo, hi):
    """Keys and values [hi - lo, heads, D] of request i in 32 bits."""
    bs = st["case"]["page"]
    at = torch.arange(lo, hi, device="cuda")
    return _rows_at(st, st["tables"][i].long()[at // bs] * bs + at % bs)


def _attend(q, k, v, seen):
    """q [n, heads, D] over k, v [L, kv, D]; query i sees the first seen[i] keys. All in 32 bits."""
    n, heads, dim = q.shape
    L, kv, _ = k.shape
    g = heads // kv
    qh = q.view(n, kv, g, dim).transpose(0, 1).reshape(kv, n * g, dim)
    s = (torch.matmul(qh, k.permute(1, 2, 0).contiguous()) / math.sqrt(dim)).view(kv, n, g, L)
    s = s.masked_fill((torch.arange(L, device=q.device)[None] >= seen[:, None])[:, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(kv, n * g, L), v.transpose(0, 1).contiguous())
    return o.view(kv, n, g, dim).transpose(0, 1).reshape(n, heads, dim)


def _plain(st):
    case = st["case"]
    op, fmt = case["op"], case["fmt"]
    if op == "write":
        kv, bs, (k, ks, v, vs) = case["kv"], case["page"], st["kv"]
        at = st["slots"].long()
        for x, codes, scales in ((st["new_kv"][:, :kv], k, ks), (st["new_kv"][:, kv:], v, vs)):
            c, s = _quantise(x, fmt)
            codes.view(torch.int8)[at // bs, at % bs] = c.view(torch.int8)
            scales[at // bs, at % bs] = s
    if op in ("write", "read"):
        return tuple(x.to(torch.bfloat16) for x in _rows_at(st, st["slots"].long()))
    out, at = torch.empty_like(st["q"]), 0
    if op == "shared":
        for m, prefix in zip(st["sizes"], st["prefixes"]):
            pk, pv = _tokens(st, at, 0, prefix)
            for i in range(at, at + m):
                L = st["reqs"][i][1] + 1
                sk, sv = _tokens(st, i, prefix, L)
                out[i] = _attend(st["q"][i:i + 1].float(), torch.cat([pk, sk]), torch.cat([pv, sv]), torch.tensor([L], device="cuda"))[0].to(out.dtype)
            at += m
        return out
    for i, (q, c) in enumerate(st["reqs"]):
        k, v = _tokens(st, i, 0, c + q)
        seen = torch.arange(c + 1, c + q + 1, device="cuda")
        out[at:at + q] = _attend(st["q"][at:at + q].float(), k, v, seen).to(out.dtype)
        at += q
    return out


# ------------------------------------------------------------------------------------------------ one call
def run(st):
    if not own:
        return _plain(st)
    from xgserve import ops
    case = st["case"]
    op, scale = case["op"], 1.0 / math.sqrt(case["dim"])
    if op == "write":
        kv = case["kv"]
        ops.kv_quant_append(st["new_kv"][:, :kv], st["new_kv"][:, kv:], st["kv"], st["slots"])
    if op in ("write", "read"):
        return ops.kv_quant_read(st["kv"], st["tables"], st["starts"], st["cu"], st["cu_host"][-1])
    if op == "decode":
        return ops.quant_decode_attention(st["q"], st["kv"], st["tables"], st["lens"], scale)
    if op == "prompt":
        return ops.quant_prefill_attention(st["q"], st["kv"], st["tables"], st["cu"], st["lens"], max(q for q, _ in st["reqs"]), scale)
    return ops.shared_prefix_attention(st["q"], st["kv"], st["tables"], st["lens"], st["plan"], scale)


def work(case):
    reqs, sizes, prefixes = _requests(case)
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    held = 2 * kv * (2 * dim if case["fmt"] == "bf16" else dim + 4)   # bytes of one token in the cache
    new = sum(q for q, _ in reqs)
    if case["op"] == "write":
        return {"bytes": new * (2 * kv * 2 * dim + 4 + held + 2 * kv * 2 * dim), "flops": new * kv * dim * 6}
    if case["op"] == "read":
        return {"bytes": new * (held + 2 * kv * 2 * dim), "flops": new * kv * dim * 2}
    seen = sum(q * c + q * (q + 1) // 2 for q, c in reqs)
    keys = sum(q + c for q, c in reqs)
    if sizes:
        keys -= sum((m - 1) * p for m, p in zip(sizes, prefixes))
    return {"bytes": keys * held + 2 * new * heads * dim * 2, "flops": 4 * heads * dim * seen}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _e4m3(y):
    """The nearest number with 3 bits behind the first and no exponent below -6, the even one of two."""
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    e = torch.where(torch.exp2(e) > y.abs().clamp(min=2.0 ** -6), e - 1, e)
    step = torch.exp2(e - 3)
    return torch.round(y / step) * step


def _held(x, fmt):
    """What the cache stands for after rows x were written to it, in 64 bits."""
    x = x.double()
    if fmt == "bf16":
        return x
    a = x.abs().amax(-1, keepdim=True)
    y = torch.where(a > 0, x * LARGEST[fmt] / torch.where(a > 0, a, 1.0), 0.0)
    return (_e4m3(y) if fmt == "fp8" else torch.round(y)) * a / LARGEST[fmt]


def exact(case, seed):
    dev = "cuda"
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device=dev).manual_seed(seed)
    reqs, sizes, prefixes = _requests(case)
    tables, blocks = _pages(case, host)
    bs, kv, dim, heads, fmt = case["page"], case["kv"], case["dim"], case["heads"], case["fmt"]
    k, v = _rows(blocks * bs, kv, dim, gen), _rows(blocks * bs, kv, dim, gen)
    new = sum(q for q, _ in reqs)
    tables = tables.to(dev).long()
    if case["op"] == "write":
        return _held(_rows(new, kv, dim, gen), fmt), _held(_rows(new, kv, dim, gen), fmt)

    def slots(i, lo, hi):
        at = torch.arange(lo, hi, device=dev)
        return tables[i][at // bs] * bs + at % bs

    if case["op"] == "read":
        at = torch.cat([slots(i, c, c + q) for i, (q, c) in enumerate(reqs)])
        return _held(k[at], fmt), _held(v[at], fmt)
    q = (1.3 * torch.randn(new, heads, dim, generator=gen, device=dev)).to(torch.bfloat16).double()
    out = torch.empty_like(q)
    lead = list(range(len(reqs)))
    if sizes:
        lead = [sum(sizes[:g]) for g, m in enumerate(sizes) for _ in range(m)]
        prefix = [p for m, p in zip(sizes, prefixes) for _ in range(m)]
    row = 0
    for i, (n, c) in enumerate(reqs):
        at = slots(i, 0, n + c) if not sizes else torch.cat([slots(lead[i], 0, prefix[i]), slots(i, prefix[i], n + c)])
        kk, vv = _held(k[at], fmt), _held(v[at], fmt)
        later = torch.arange(n + c, device=dev)[None] > c + torch.arange(n, device=dev)[:, None]
        for h in range(heads):
            s = q[row:row + n, h] @ kk[:, h * kv // heads].T / math.sqrt(dim)
            out[row:row + n, h] = torch.softmax(s.masked_fill(later, -math.inf), -1) @ vv[:, h * kv // heads]
        row += n
    return out
