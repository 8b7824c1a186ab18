"""The 8-bit paged cache: writing, reading back, and the attentions over it, against the formulas in 64 bits.

Tolerances. Codes and scales are exact (a scale: one fp32 rounding), rows read back have one fp32 and one bf16 rounding. An
attention output sum_j p_j v_j rounds every weight p_j (times its value's scale) to bf16 and the result again, each off by at
most 2^-8 of itself, and computes scores in fp32: D products and sums each off by 2^-24 of sum |q k|, which the exponential
turns into a relative error of the weights (and of their sum, hence twice).
"""
import math

import pytest
import torch

from xgserve import ops
from xgserve.ops import kv_quant
from xgserve.ops.attention import DecodeWorkspace

GPU = pytest.param("cuda", marks=pytest.mark.gpu)
DEVICES = pytest.mark.parametrize("dev", ["cpu", GPU])
FORMATS = pytest.mark.parametrize("fmt", ["fp8", "int8"])
E4M3 = sorted({(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)} - {480.0} | {m * 2.0 ** -9 for m in range(8)})


def nearest_e4m3(y):
    """By search in the list of all E4M3 numbers; of two at the same distance the one of even place (0 is the first)."""
    t = torch.tensor(E4M3, dtype=torch.float64)
    a = y.abs()
    hi = torch.searchsorted(t, a).clamp(max=len(E4M3) - 1)
    lo = (hi - 1).clamp(min=0)
    below, above = a - t[lo], t[hi] - a
    pick = torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
    return t[pick] * y.sign()


def held(x, fmt):
    """Codes' values and scales (64 bits) of rows [..., D]."""
    largest = 448.0 if fmt == "fp8" else 127.0
    x = x.double().cpu()
    a = x.abs().amax(-1, keepdim=True)
    bad = ~x.isfinite().all(-1, keepdim=True)
    y = torch.where(bad | (a == 0), 0.0, x * largest / torch.where(bad | (a == 0), 1.0, a))
    code = nearest_e4m3(y) if fmt == "fp8" else torch.round(y)
    return code, torch.where(bad, math.nan, a / largest)


def value(x, fmt):
    if fmt == "bf16":
        return x.double().cpu()
    c, s = held(x, fmt)
    return c * s


def rows(n, heads, D, gen, spread=1.0):
    gain = torch.exp(0.5 * torch.randn(heads, D, generator=gen))
    return (spread * torch.randn(n, heads, D, generator=gen) * gain).to(torch.bfloat16)


def paged(lens, bs, gen, extra=2):
    need = [-(-n // bs) for n in lens]
    total = sum(need) + extra
    order = torch.randperm(total, generator=gen).to(torch.int32)
    table = torch.full((len(lens), max(max(need), 1)), total - 1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, total


def slots_of(table_row, lo, hi, bs):
    at = torch.arange(lo, hi)
    return table_row.long()[at // bs] * bs + at % bs


def spoil(cache):
    """What pages may hold that nobody wrote: E4M3's NaN, and scales that are NaN."""
    cache.k.fill_(0x7F)
    cache.v.fill_(0xFF)
    cache.scales.fill_(math.nan)


def attention(q, k, v, seen, scale):
    """q [n, Hq, D], k, v [L, Hkv, D] in 64 bits, query i sees seen[i] keys -> output, and what bounds its error."""
    n, Hq, D = q.shape
    G = Hq // max(1, k.shape[1])
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for i in range(n):
        L = int(seen[i])
        if L == 0:
            continue
        kk, vv = (x[:L].repeat_interleave(G, dim=1) for x in (k, v))
        s = torch.einsum("hd,lhd->hl", q[i], kk) * scale
        p = torch.softmax(s, -1)
        out[i] = torch.einsum("hl,lhd->hd", p, vv)
        size = torch.einsum("hl,lhd->hd", p, vv.abs())
        work = torch.einsum("hd,lhd->hl", q[i].abs(), kk.abs()).amax(-1)[:, None] * abs(scale)
        bound[i] = size * (2.0 ** -8 + 2 * (D + 16) * 2.0 ** -24 * (1 + work) + 2.0 ** -18) + out[i].abs() * 2.0 ** -8
    return out, bound * 1.01 + 1e-30


def check(got, ref, bound):
    err = (got.double().cpu() - ref).abs()
    worst = (err / bound).max().item() if err.numel() else 0.0
    assert not bool((err > bound).any() | err.isnan().any()), f"off by {worst:.3g} times the bound"


def make(lens, Hkv, D, bs, fmt, dev, gen, fill=None):
    """A cache whose first lens[s] tokens of each table hold rows, and nothing usable elsewhere."""
    table, nb = paged(lens, bs, gen)
    n = sum(lens)
    k, v = rows(n, Hkv, D, gen), rows(n, Hkv, D, gen, 1.5)
    if fill:
        fill(k, v)
    slots = torch.cat([slots_of(table[s], 0, L, bs) for s, L in enumerate(lens)] + [torch.zeros(0, dtype=torch.long)])
    if fmt == "bf16":
        pages = []
        for x in (k, v):
            c = torch.full((nb * bs, Hkv, D), math.nan, dtype=torch.bfloat16)
            c[slots] = x
            pages.append(c.view(nb, bs, Hkv, D).transpose(1, 2).contiguous().to(dev))
        cache = tuple(pages)
    else:
        cache = ops.QuantKVCache.alloc(nb, Hkv, bs, D, fmt, dev)
        spoil(cache)
        ops.kv_quant_append(k.to(dev), v.to(dev), cache, slots.to(dev, torch.int32))
    cu = [0]
    for L in lens:
        cu.append(cu[-1] + L)
    kv, vv = value(k, fmt), value(v, fmt)
    return cache, table.to(dev), [(kv[a:b], vv[a:b]) for a, b in zip(cu, cu[1:])]


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


# ------------------------------------------------------------------------------------------------------------ write and read
def hard_rows(D):
    """Rows at the borders of two codes, and those whose size is out of the ordinary."""
    r = [torch.zeros(D)]
    r.append(torch.arange(D).float() % 256 - 127)
    r[-1][0] = 254.0                                     # 127 x / 254: every odd x lies on a border
    r.append(torch.tensor([17.0, 19, 21, -17, 34, 38, 0.0009765625, 0.0029296875] * (D // 8)))
    r[-1][0] = 448.0                                     # E4M3's borders, those below its smallest normal number too
    r.append(torch.full((D,), -3.3e38))
    r.append(torch.linspace(-3.3e38, 3.3e38, D))
    r.append(torch.arange(D).float() * 9.2e-41)          # below the smallest normal float
    r.append(torch.arange(D).float() * 1.3e-38)
    one = torch.zeros(D)
    one[D - 1] = 9.2e-41
    r.append(one)
    one = torch.full((D,), 1e-30)
    one[3] = 1e30
    r.append(one)
    for m in (129, 151, 213, 255):
        r.append((torch.arange(D) % 200 + 1).float())
        r[-1][1] = m * 128.0 if m > 200 else m
    for bad in (math.inf, -math.inf, math.nan):
        x = torch.linspace(-2, 2, D)
        x[D // 2] = bad
        r.append(x)
    return torch.stack(r).to(torch.bfloat16)


@DEVICES
@FORMATS
@pytest.mark.parametrize("D", [64, 128])
def test_codes_are_those_of_the_formula(dev, fmt, D):
    gen = torch.Generator().manual_seed(D)
    x = torch.cat([hard_rows(D), rows(200, 1, D, gen)[:, 0], torch.randint(-255, 256, (100, D), generator=gen).to(torch.bfloat16)])
    n = x.shape[0]
    cache = ops.QuantKVCache.alloc(-(-n // 32), 1, 32, D, fmt, dev)
    k, v = x[:, None].to(dev), x.flip(0)[:, None].contiguous().to(dev)
    ops.kv_quant_append(k, v, cache, torch.arange(n, dtype=torch.int32, device=dev))
    ko, vo = (o.cpu() for o in kv_quant._order(D, dev))
    slots = torch.arange(n)
    for side, (codes, order, src) in enumerate(((cache.k, ko, x), (cache.v, vo, x.flip(0)))):
        flat = codes.cpu().view(-1, 32 * D)
        raw = flat[(slots // 32)[:, None], ((slots % 32) // 16 * 16 * D)[:, None] + order[slots % 16]]
        got = raw.view(torch.float8_e4m3fn if fmt == "fp8" else torch.int8).double()
        code, scale = held(src, fmt)
        assert torch.equal(got, code)
        sc = cache.scales.cpu()[slots // 32, 0, side, slots % 32].double()
        assert torch.equal(sc.isnan(), scale[:, 0].isnan())
        good = ~sc.isnan()
        assert bool(((sc - scale[:, 0])[good].abs() <= scale[good, 0] * 2.0 ** -24 + 2.0 ** -150).all())
    rk, rv = ops.kv_quant_read(cache, i32([list(range(cache.num_blocks))], dev), i32([0], dev), i32([0, n], dev), n)
    for got, src in ((rk, x), (rv, x.flip(0))):
        want = value(src, fmt)
        got = got[:, 0].double().cpu()
        assert torch.equal(got.isnan(), want.isnan())
        good = ~want.isnan()
        assert bool(((got - want)[good].abs() <= want[good].abs() * (2.0 ** -8 + 2.0 ** -22) + 2.0 ** -133 / 2 + 448 * 2.0 ** -150).all())


@DEVICES
@FORMATS
@pytest.mark.parametrize("Hkv,D,bs", [(8, 128, 16), (1, 128, 48), (3, 64, 16), (12, 64, 32)])
def test_append_takes_any_slots_and_leaves_the_rest(dev, fmt, Hkv, D, bs):
    gen = torch.Generator().manual_seed(7 * Hkv + D)
    nb = 9
    total = nb * bs
    pieces = [torch.arange(5, 18), torch.tensor([-1, total, 2 ** 31 - 1, -2 ** 31]), torch.arange(32, 36), torch.tensor([41, 40, 43, 42]),
              torch.arange(50, 52), torch.arange(56, 59), torch.tensor([61, 62, 63, 64, 65, 66, 67]), torch.arange(total - 9, total),
              torch.tensor([100, 90, 80, -5, 0])]
    for T in (0, 1, 2, 3, 4, 5, None):
        slots = torch.cat(pieces)[:T] if T is not None else torch.cat(pieces)
        T = slots.shape[0]
        big = rows(T, 2 * Hkv + 4, D, gen).to(dev)     # (the projection's rows: k and v beside the queries)
        k, v = big[:, 4:4 + Hkv], big[:, 4 + Hkv:]
        cache = ops.QuantKVCache.alloc(nb, Hkv, bs, D, fmt, dev)
        cache.k.copy_(torch.randint(0, 127, cache.k.shape, generator=gen))
        cache.v.copy_(torch.randint(0, 127, cache.k.shape, generator=gen))
        cache.scales.copy_(torch.rand(cache.scales.shape, generator=gen))
        plain = ops.QuantKVCache(cache.k.cpu().clone(), cache.v.cpu().clone(), cache.scales.cpu().clone(), fmt)
        ops.kv_quant_append(k, v, cache, slots.to(dev, torch.int32))
        for s, t in zip(slots.tolist(), range(T)):     # row by row, through the plain form's parts
            if 0 <= s < total:
                ko, vo = kv_quant._order(D, "cpu")
                for side, (x, codes, order) in enumerate(((k, plain.k, ko), (v, plain.v, vo))):
                    c, sc = held(x[t].cpu(), fmt)
                    raw = c.float().to(torch.float8_e4m3fn).view(torch.uint8) if fmt == "fp8" else c.to(torch.int8).view(torch.uint8)
                    # (a code of -0 stands for a negative number that rounds to 0)
                    if fmt == "fp8":
                        raw = raw | ((x[t].cpu().float() < 0) & (c == 0)).to(torch.uint8) * 128
                    for h in range(Hkv):
                        codes[s // bs, h].view(-1)[(s % bs) // 16 * 16 * D + order[s % 16]] = raw[h]
                    plain.scales[s // bs, :, side, s % bs] = sc[:, 0].float()
        assert torch.equal(cache.k.cpu(), plain.k) and torch.equal(cache.v.cpu(), plain.v)
        torch.testing.assert_close(cache.scales.cpu(), plain.scales, rtol=2.0 ** -23, atol=0)


@pytest.mark.gpu
@FORMATS
@pytest.mark.parametrize("Hkv,D", [(8, 128), (8, 64), (12, 64), (5, 128)])
def test_append_of_many_rows(fmt, Hkv, D):
    """Two heads a wave (an even number of heads), tokens that begin anywhere in a quad, and some of no slot."""
    gen = torch.Generator().manual_seed(11)
    T, bs, nb = 16384 // Hkv + 5, 32, 16384 // Hkv // 32 + 8
    x = rows(T, 2 * Hkv, D, gen)
    slots = torch.cat([torch.arange(3, 1003), torch.tensor([-1, -1]), torch.arange(1026, 1026 + T - 1002)]).to(torch.int32)
    slots[[5, 700]] = -1
    got, want = (ops.QuantKVCache.alloc(nb, Hkv, bs, D, fmt, d) for d in ("cuda", "cpu"))
    big = x.to("cuda")
    ops.kv_quant_append(big[:, :Hkv], big[:, Hkv:], got, slots.to("cuda"))
    ops.kv_quant_append(x[:, :Hkv], x[:, Hkv:], want, slots)
    assert torch.equal(got.k.cpu(), want.k) and torch.equal(got.v.cpu(), want.v)
    torch.testing.assert_close(got.scales.cpu(), want.scales, rtol=2.0 ** -23, atol=0)


@DEVICES
@FORMATS
@pytest.mark.parametrize("Hkv,D,bs", [(8, 128, 16), (2, 64, 48)])
def test_read_takes_any_ranges(dev, fmt, Hkv, D, bs):
    gen = torch.Generator().manual_seed(3)
    lens = [1, 0, 17, 130, 64, 33, 2]
    cache, table, truth = make(lens, Hkv, D, bs, fmt, dev, gen)
    for ranges in ([(0, n) for n in lens], [(0, 1), (0, 0), (16, 1), (15, 100), (31, 33), (32, 1), (1, 1)],
                   [(0, 0)] * 3 + [(129, 1), (0, 0), (7, 20), (0, 0)], [(0, 0)] * 7):
        starts, cu = [a for a, _ in ranges], [0]
        for _, n in ranges:
            cu.append(cu[-1] + n)
        out = tuple(torch.full((cu[-1], Hkv, D), 7.0, dtype=torch.bfloat16, device=dev) for _ in range(2))
        k, v = ops.kv_quant_read(cache, table, i32(starts, dev), i32(cu, dev), cu[-1], out=out)
        assert k is out[0] and v is out[1]
        for s, (a, n) in enumerate(ranges):
            for got, want in zip((k, v), truth[s]):
                want = want[a:a + n]
                err = (got[cu[s]:cu[s + 1]].double().cpu() - want).abs()
                assert bool((err <= want.abs() * (2.0 ** -8 + 2.0 ** -22)).all())


@DEVICES
def test_read_leaves_rows_behind_the_table(dev):
    gen = torch.Generator().manual_seed(4)
    cache, table, truth = make([48], 2, 64, 16, "int8", dev, gen)
    out = tuple(torch.full((40, 2, 64), 7.0, dtype=torch.bfloat16, device=dev) for _ in range(2))
    ops.kv_quant_read(cache, table[:, :2], i32([10], dev), i32([0, 40], dev), 40, out=out)
    for got, want in zip(out, truth[0]):
        err = (got[:22].double().cpu() - want[10:32]).abs()
        assert bool((err <= want[10:32].abs() * (2.0 ** -8 + 2.0 ** -22)).all())
        assert bool((got[22:] == 7.0).all())


@DEVICES
@FORMATS
@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 128), (8, 1, 128), (12, 12, 64)])
def test_rope_kv_quant(dev, fmt, Hq, Hkv, D):
    """q as rope_cache rotates it; the cache as kv_quant_append writes the rotated k."""
    gen = torch.Generator().manual_seed(5)
    T, bs, nb = 37, 16, 8
    qkv = rows(T, Hq + 2 * Hkv, D, gen).view(T, -1).to(dev)
    pos = torch.randint(0, 4000, (T,), generator=gen).to(dev, torch.int32)
    cs = ops.build_cos_sin(D, 4096, 500000.0, device=dev)
    slots = torch.randperm(nb * bs, generator=gen)[:T].to(torch.int32)
    slots[20:33] = torch.arange(96, 109)
    slots[:20] = torch.randperm(96, generator=gen)[:20]
    slots[33:] = torch.arange(120, 124)
    slots[3] = -1
    slots = slots.to(dev)
    ref, kc = qkv.clone(), torch.zeros(nb, Hkv, bs, D, dtype=torch.bfloat16, device=dev)
    vc = torch.zeros_like(kc)
    ops.rope_cache(ref, pos, cs, kc, vc, slots, Hq, Hkv, D)
    cache = ops.QuantKVCache.alloc(nb, Hkv, bs, D, fmt, dev)
    ops.rope_kv_quant(qkv, pos, cs, cache, slots, Hq)
    q = Hq * D
    # the same formula in another order of fp32 operations: two neighbours of bf16 at most
    torch.testing.assert_close(qkv[:, :q].float(), ref[:, :q].float(), rtol=2.0 ** -7, atol=2e-6)
    assert torch.equal(qkv[:, q:], ref[:, q:])
    other = ops.QuantKVCache.alloc(nb, Hkv, bs, D, fmt, dev)
    real = slots >= 0
    at = slots[real].long()
    ops.kv_quant_append(kc[at // bs, :, at % bs].contiguous(), vc[at // bs, :, at % bs].contiguous(), other, slots[real].contiguous())
    assert torch.equal(cache.v, other.v)
    table = i32([list(range(nb))], dev)
    a, b = (ops.kv_quant_read(c, table, i32([0], dev), i32([0, nb * bs], dev), nb * bs)[0].float() for c in (cache, other))
    # k's rotation may round to the neighbour, and its code then too: a step of the code (of the largest, for int8)
    size = b.abs().amax(-1, keepdim=True)
    step = b.abs() * 2.0 ** -3 + size * 2.0 ** -9 if fmt == "fp8" else size / 127
    assert bool(((a - b).abs() <= 1.01 * step + size * 2.0 ** -6).all())
    assert float((a != b).float().mean()) < 0.05


# ----------------------------------------------------------------------------------------------------------------- attention
LENS = [1, 0, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300, 1000]


@DEVICES
@FORMATS
@pytest.mark.parametrize("Hq,Hkv,D,bs", [(32, 8, 128, 16), (8, 1, 128, 32), (12, 12, 64, 16), (6, 2, 64, 48), (20, 1, 128, 16),
                                         (7, 7, 128, 16), (40, 2, 64, 16)])
@pytest.mark.parametrize("splits", [None, 1, 3, 64])
def test_decode(dev, fmt, Hq, Hkv, D, bs, splits):
    gen = torch.Generator().manual_seed(Hq + D)
    cache, table, truth = make(LENS, Hkv, D, bs, fmt, dev, gen)
    big = rows(len(LENS), Hq + 3, D, gen, 1.5).to(dev)
    q = big[:, 3:]
    scale = 1 / math.sqrt(D)
    out = ops.quant_decode_attention(q, cache, table, i32(LENS, dev), scale, num_splits=splits)
    for s, L in enumerate(LENS):
        ref, bound = attention(q[s:s + 1].double().cpu(), *truth[s], [L], scale)
        check(out[s:s + 1], ref, bound)


@DEVICES
@FORMATS
@pytest.mark.parametrize("B,splits", [(3, 7), (64, 2), (65, 3), (130, 1), (300, 2), (300, None)])
def test_decode_of_batches_of_any_lengths(dev, fmt, B, splits):
    """Shares of the batch's keys: one long sequence among short and empty ones, more sequences than lanes of a wave, and of four."""
    gen = torch.Generator().manual_seed(B)
    lens = [(i * 37) % 90 for i in range(B)]
    lens[B // 3], lens[-1] = 1500, 700
    cache, table, truth = make(lens, 1, 64, 16, fmt, dev, gen)
    q = rows(B, 4, 64, gen).to(dev)
    out = ops.quant_decode_attention(q, cache, table, i32(lens, dev), 0.125, num_splits=splits)
    some = range(B) if B < 100 else [0, 1, B // 3, 63, 64, 65, 127, 128, B - 2, B - 1]
    for s in some:
        check(out[s:s + 1], *attention(q[s:s + 1].double().cpu(), *truth[s], [lens[s]], 0.125))
    same = ops.quant_decode_attention(q, cache, table, i32(lens, dev), 0.125, num_splits=splits)
    assert torch.equal(out, same)


@pytest.mark.gpu
@FORMATS
@pytest.mark.parametrize("lens,W,shares", [
    ([(i * 53) % 300 for i in range(120)] + [4000] + [(i * 71) % 280 for i in range(79)], 4096, (400, 16)),   # one is cut
    ([(i * 211) % 2048 for i in range(200)], 4096, (400, 16)),                                                # none is
    ([2049] * 200, 4096, (400, 16)),                                                                          # all are: 17 units each
    ([20000], 20000, (158, 1)), ([16385, 5], 16400, (260, 1))])   # parts at their limit (2 + 2 x ceil(16400 / 128) shares)
def test_decode_where_the_rule_cuts(fmt, lens, W, shares):
    """Automatic shares of wide tables: batches that fill the chip leave sequences of up to 2048 keys whole; 128 parts at most."""
    gen = torch.Generator().manual_seed(len(lens))
    B = len(lens)
    assert kv_quant._shares(None, B, 1, W) == shares
    cache, table, truth = make(lens, 1, 64, 16, fmt, "cuda", gen)
    table = torch.cat([table, table.new_full((B, -(-W // 16) - table.shape[1]), cache.num_blocks - 1)], 1)
    q = rows(B, 4, 64, gen).to("cuda")
    out = ops.quant_decode_attention(q, cache, table, i32(lens, "cuda"), 0.125)
    for s in range(B) if B < 100 else [0, 1, 63, 64, 119, 120, 121, 127, 128, 192, 198, 199]:
        check(out[s:s + 1], *attention(q[s:s + 1].double().cpu(), *truth[s], [lens[s]], 0.125))


@pytest.mark.gpu
@FORMATS
def test_prompts_where_the_rule_cuts(fmt):
    """Automatic parts of a short portion behind many keys, and automatic blocks of 128 rows."""
    gen = torch.Generator().manual_seed(27)
    for Hq, Hkv, new, ctx, cut in ((8, 1, [37, 5], [1500, 0], True), (24, 12, [1900, 1850, 300], [0, 17, 90], False)):
        lens = [a + b for a, b in zip(new, ctx)]
        cache, table, truth = make(lens, Hkv, 64, 16, fmt, "cuda", gen)
        rt = kv_quant._row_tiles(max(new) * Hq // Hkv, len(new) * Hkv)
        blocks = -(-max(new) * (Hq // Hkv) // (16 * rt))
        splits = kv_quant._splits(None, len(new) * Hkv * blocks, table.shape[1] * 16)
        assert (splits > 1 and rt < 8) if cut else (splits == 1 and rt == 8)
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        q = rows(cu[-1], Hq, 64, gen).to("cuda")
        out = ops.quant_prefill_attention(q, cache, table, i32(cu, "cuda"), i32(lens, "cuda"), max(new), 0.125)
        for s, n in enumerate(new):
            for i in sorted({0, 1, n // 3, n // 2, n - 2, n - 1}):
                at = slice(cu[s] + i, cu[s] + i + 1)
                check(out[at], *attention(q[at].double().cpu(), *truth[s], [ctx[s] + i + 1], 0.125))


@DEVICES
def test_decode_into_a_strided_output_with_a_workspace(dev):
    gen = torch.Generator().manual_seed(2)
    lens = [200, 0, 77]
    cache, table, truth = make(lens, 2, 128, 16, "fp8", dev, gen)
    q = rows(3, 8, 128, gen).to(dev)
    big = torch.full((3, 11, 128), 5.0, dtype=torch.bfloat16, device=dev)
    out = ops.quant_decode_attention(q, cache, table, i32(lens, dev), 0.1, num_splits=4, out=big[:, 1:9],
                                     workspace=DecodeWorkspace(3, 8, 128, 4, dev))
    assert out.data_ptr() == big[:, 1:9].data_ptr()
    assert bool((big[:, 0] == 5).all()) and bool((big[:, 9:] == 5).all())
    for s, L in enumerate(lens):
        check(out[s:s + 1], *attention(q[s:s + 1].double().cpu(), *truth[s], [L], 0.1))


@DEVICES
@FORMATS
def test_lengths_behind_the_table_and_pages_outside_the_cache(dev, fmt):
    gen = torch.Generator().manual_seed(12)
    cache, table, truth = make([64, 40], 1, 64, 16, fmt, dev, gen, fill=lambda k, v: v.abs_())
    q = rows(2, 4, 64, gen).to(dev)
    out = ops.quant_decode_attention(q, cache, table, i32([1000, -3], dev), 0.1)
    check(out[:1], *attention(q[:1].double().cpu(), *truth[0], [64], 0.1))
    assert bool((out[1] == 0).all())
    wild = table.clone()
    wild[0, 2:] = i32([1 << 30, -5], dev)
    got = ops.quant_decode_attention(q, cache, wild, i32([64, 40], dev), 0.1)     # some page of the cache instead
    check(got[1:], *attention(q[1:].double().cpu(), *truth[1], [40], 0.1))


@DEVICES
@FORMATS
def test_scores_far_apart(dev, fmt):
    """Scores that rise along the keys, by little and by much, and a first key far above all others."""
    gen = torch.Generator().manual_seed(13)
    L, D = 400, 64
    ramps = [torch.linspace(0, 30, L), torch.linspace(-3000, 3000, L), torch.cat([torch.tensor([900.0]), torch.zeros(L - 1)]),
             torch.linspace(200, -200, L)]

    def fill(k, v):
        k.zero_()
        for s, r in enumerate(ramps):
            k[s * L:(s + 1) * L, 0, 0] = r.to(torch.bfloat16)

    cache, table, truth = make([L] * 4, 1, D, 16, fmt, dev, gen, fill)
    q = torch.zeros(4, 2, D, dtype=torch.bfloat16)
    q[:, 0, 0], q[:, 1, 0] = 1.0, -0.5
    for splits in (1, 3):
        out = ops.quant_decode_attention(q.to(dev), cache, table, i32([L] * 4, dev), 1.0, num_splits=splits)
        for s in range(4):
            check(out[s:s + 1], *attention(q[s:s + 1].double(), *truth[s], [L], 1.0))


@DEVICES
@FORMATS
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("exact", [False, True])
def test_scores_further_down_than_any_mask(dev, fmt, D, exact):
    """All keys alike, and scores of about -2^112. Where the row's largest magnitude is the largest code times a power of two, and softmax's
    scale ln 2 (1 in base 2, to 32 bits), each score has few bits and is exact: the mean of the values; a weight of 1 times the value's
    scale and the output are rounded to bf16, each off by 2^-8 of it at most. Else 32 bits leave a score 2^88 of room, so the weights may be any (a product that is
    rounded at once with the maximum's difference has the part that the maximum lost), and so may those of parts, whose log-sums of
    2^112 and 2^112 + 8 are one number: the output lies among the values."""
    gen = torch.Generator().manual_seed(19)
    lens = [300, 33, 1]

    def fill(k, v):
        k.zero_()
        k[:, :, 0] = kv_quant.LARGEST[fmt] * 2.0 ** 44 if exact else 2.0 ** 50

    cache, table, truth = make(lens, 1, D, 16, fmt, dev, gen, fill)
    q = torch.zeros(3, 4, D, dtype=torch.bfloat16)
    q[..., 0] = -(2.0 ** 62)
    args, scale = (q.to(dev), cache, table), math.log(2.0) if exact else 1.0
    plan = ops.shared_prefix_plan([1, 1, 1], [64, 32, 0], 4, 1, dev)
    outs = [(n, ops.quant_decode_attention(*args, i32(lens, dev), scale, num_splits=n)) for n in (1, 3)]
    outs += [(n, ops.quant_prefill_attention(*args, i32([0, 1, 2, 3], dev), i32(lens, dev), 1, scale, num_splits=n, row_tiles=rt))
             for n, rt in ((1, 1), (3, 1), (1, 2), (1, 8), (3, 8))]
    outs.append((2, ops.shared_prefix_attention(*args, i32(lens, dev), plan, scale)))
    for s in range(3):
        v = truth[s][1][:, 0]
        for parts, out in outs:
            if exact and parts == 1:
                check(out[s], v.mean(0).expand(4, D), ((v.abs().mean(0) + v.mean(0).abs()) * 1.01 * 2.0 ** -8 + 1e-30).expand(4, D))
            else:
                room = v.abs().amax(0) * 1.01 * 2.0 ** -7
                o = out[s].double().cpu()
                assert bool(((o >= v.amin(0) - room) & (o <= v.amax(0) + room)).all())


@DEVICES
@pytest.mark.parametrize("fmt", ["bf16", "fp8", "int8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("first,power", [(-122, -122), (-60, -60), (126, 126), (-110, 40), (0, 126), (126, 0)])
def test_values_of_any_size(dev, fmt, D, first, power):
    """Values of up to 2^(power + 1) (those of a sequence's first 200 tokens: 2^(first + 1)), next to the largest number of bf16 and to the smallest normal one: what is summed is the weights times
    these, and no part of it may leave its type's range where the output does not. Both sides times 2^-power (the output is linear in
    the values); below 2^-126 an output's rounding is half of bf16's smallest number, 2^-134, and an fp32 scale's 2^-150 for a code of up to
    448."""
    gen = torch.Generator().manual_seed(24)
    lens, Hq, unit = [700, 33, 1, 300, 90], 8, 2.0 ** -max(first, power)

    def fill(k, v):
        size = torch.cat([torch.where(torch.arange(n) < 200, 2.0 ** first, 2.0 ** power) for n in lens])[:, None, None]
        v.copy_(v.double().div(v.abs().amax(-1, keepdim=True)).mul(1.5 * size).abs())

    cache, table, truth = make(lens, 2, D, 16, fmt, dev, gen, fill)
    q = rows(len(lens), Hq, D, gen).to(dev)
    assert all(bool((v.abs().amax(-1) >= 1.49 * 2.0 ** min(first, power)).all()) for _, v in truth)

    def hold(out, seen, s):
        k, v = truth[s]
        ref, bound = attention(q[s:s + 1].double().cpu(), k, v * unit, [seen], 0.1)
        got = out.double().cpu() * unit
        check(got, ref, bound + (2.0 ** -134 + 448 * 2.0 ** -150) * unit * 1.01)

    ln = i32(lens, dev)
    plan = ops.shared_prefix_plan([1] * len(lens), [640, 32, 0, 0, 64], Hq, 2, dev)
    outs = [ops.shared_prefix_attention(q, cache, table, ln, plan, 0.1, num_splits=n) for n in (1, 5)]
    if fmt == "bf16":
        wide = ops.shared_prefix_plan([1] * len(lens), [640, 32, 0, 0, 64], Hq, 2, dev)
        wide.wide = kv_quant._prefix_work([1] * len(lens), [640, 32, 0, 0, 64], Hq // 2, 2, 8, 4,
                                          lambda r, w: torch.tensor(r, dtype=torch.int32).reshape(-1, *w).to(dev))
        outs.append(ops.shared_prefix_attention(q, cache, table, ln, wide, 0.1))
    else:
        outs += [ops.quant_decode_attention(q, cache, table, ln, 0.1, num_splits=n) for n in (1, 3)]
        outs += [ops.quant_prefill_attention(q, cache, table, i32(list(range(len(lens) + 1)), dev), ln, 1, 0.1, num_splits=n, row_tiles=rt)
                 for n, rt in ((1, 1), (1, 2), (1, 8), (3, 8))]
    for out in outs:
        for s, L in enumerate(lens):
            hold(out[s:s + 1], L, s)


@DEVICES
@FORMATS
def test_portions_longer_than_their_sequences(dev, fmt):
    """Lengths below a portion's tokens, and below zero: the first token sees the first key, and none sees more than there are."""
    gen = torch.Generator().manual_seed(20)
    cache, table, truth = make([40, 40, 40], 2, 64, 16, fmt, dev, gen)
    q = rows(3 * 35, 4, 64, gen).to(dev)
    for splits, rt in ((1, 1), (1, 2), (3, 2), (1, 8), (3, 8)):
        out = ops.quant_prefill_attention(q, cache, table, i32([0, 35, 70, 105], dev), i32([-5, 0, 20], dev), 35, 0.1,
                                          num_splits=splits, row_tiles=rt)
        assert bool((out[:70] == 0).all())
        check(out[70:], *attention(q[70:].double().cpu(), *truth[2], [min(i + 1, 20) for i in range(35)], 0.1))


@DEVICES
@FORMATS
def test_a_key_that_is_not_finite_reaches_only_those_who_see_it(dev, fmt):
    gen = torch.Generator().manual_seed(14)

    def fill(k, v):
        k[50, 0, 3] = math.inf
        v[100 + 70, 1, 5] = math.nan

    lens = [100, 100, 100]
    cache, table, truth = make(lens, 2, 64, 16, fmt, dev, gen, fill)
    q = rows(3, 4, 64, gen).to(dev)
    out = ops.quant_decode_attention(q, cache, table, i32(lens, dev), 0.1).cpu()
    assert bool(out[0, :2].isnan().all()) and bool(out[0, 2:].isfinite().all())
    assert bool(out[1, 2:].isnan().all()) and bool(out[1, :2].isfinite().all()) and bool(out[2].isfinite().all())
    n = 60                                # tokens 40 .. 100 of each: those before the key do not see it
    qp = rows(3 * n, 4, 64, gen).to(dev)
    for rt, s in ((rt, s) for rt in (1, 2, 8) for s in range(3)):
        got = ops.quant_prefill_attention(qp, cache, table, i32([0, n, 2 * n, 3 * n], dev), i32(lens, dev), n, 0.1, row_tiles=rt).cpu()
        for i in range(n):
            seen = 40 + i + 1
            bad = [s == 0 and seen > 50, s == 1 and seen > 70]
            for h in range(2):
                o = got[s * n + i, 2 * h:2 * h + 2]
                if bad[h]:
                    assert bool(o.isnan().all())
                else:
                    kk, vv = (x[:seen, h:h + 1] for x in truth[s])
                    check(o[None], *attention(qp[s * n + i:s * n + i + 1, 2 * h:2 * h + 2].double().cpu(), kk, vv, [seen], 0.1))


@DEVICES
@FORMATS
@pytest.mark.parametrize("Hq,Hkv,D,bs", [(32, 8, 128, 16), (8, 1, 128, 32), (12, 12, 64, 16), (6, 2, 64, 48), (20, 1, 128, 16)])
@pytest.mark.parametrize("splits,rt", [(None, None), (1, 1), (1, 2), (5, 2), (1, 8), (3, 8)])
def test_prompts(dev, fmt, Hq, Hkv, D, bs, splits, rt):
    gen = torch.Generator().manual_seed(Hq * 3 + D)
    new, ctx = [1, 0, 5, 33, 17, 64, 3, 130], [0, 9, 0, 31, 200, 64, 500, 2]
    lens = [a + b for a, b in zip(new, ctx)]
    cache, table, truth = make(lens, Hkv, D, bs, fmt, dev, gen)
    cu = [2]                                   # rows before the first portion and behind the last one belong to nobody
    for n in new:
        cu.append(cu[-1] + n)
    q = rows(cu[-1] + 3, Hq, D, gen, 1.5).to(dev)
    scale = 1 / math.sqrt(D)
    out = torch.full_like(q, 9.0)
    ops.quant_prefill_attention(q, cache, table, i32(cu, dev), i32(lens, dev), max(new), scale, num_splits=splits, out=out,
                                row_tiles=rt)
    assert bool((out[:2] == 9).all()) and bool((out[cu[-1]:] == 9).all())
    for s, n in enumerate(new):
        a, b = cu[s], cu[s + 1]
        if n:
            check(out[a:b], *attention(q[a:b].double().cpu(), *truth[s], [ctx[s] + i + 1 for i in range(n)], scale))


def groups_of(sizes, prefixes, tails, Hkv, D, bs, fmt, dev, gen, fill=None):
    """Sequences in groups; a group's whole pages of the prefix are common, and only its first sequence's table is right below the
    prefix: the others' first pages are somebody else's."""
    lens = [p + t for m, p, tt in zip(sizes, prefixes, tails) for t in tt]
    cache, table, truth = make(lens, Hkv, D, bs, fmt, dev, gen, fill)
    seqs, at = [], 0
    for m, p in zip(sizes, prefixes):
        for i in range(m):
            seqs.append(tuple(torch.cat([truth[at][j][:p], truth[at + i][j][p:]]) for j in (0, 1)))
            if i and p // bs:
                table[at + i, :p // bs] = table[at + i, :p // bs].flip(0)
        at += m
    return cache, table, lens, seqs


@DEVICES
@pytest.mark.parametrize("fmt", ["bf16", "fp8", "int8"])
@pytest.mark.parametrize("Hq,Hkv,D,bs", [(32, 8, 128, 16), (8, 1, 128, 32), (12, 12, 64, 16), (6, 2, 64, 48), (20, 1, 128, 16)])
@pytest.mark.parametrize("splits,wide", [(None, False), (1, False), (5, False), (None, True), (3, True)])
def test_shared_prefix(dev, fmt, Hq, Hkv, D, bs, splits, wide, monkeypatch):
    if wide:
        monkeypatch.setattr(kv_quant, "WIDE_ROWS", 0)
        monkeypatch.setattr(kv_quant, "WIDE_TILES", 0)
    gen = torch.Generator().manual_seed(Hq * 5 + D)
    sizes, prefixes = [3, 1, 5, 17, 2], [100, 0, 33, 64, 400]
    tails = [[5, 1, 40], [70], [1, 2, 3, 4, 100], list(range(1, 18)), [0, 9]]
    cache, table, lens, seqs = groups_of(sizes, prefixes, tails, Hkv, D, bs, fmt, dev, gen)
    q = rows(len(lens), Hq, D, gen, 1.5).to(dev)
    plan = ops.shared_prefix_plan(sizes, prefixes, Hq, Hkv, dev)
    assert (plan.wide is not None) == wide
    scale = 1 / math.sqrt(D)
    out = ops.shared_prefix_attention(q, cache, table, i32(lens, dev), plan, scale, num_splits=splits)
    for s, L in enumerate(lens):
        check(out[s:s + 1], *attention(q[s:s + 1].double().cpu(), *seqs[s], [L], scale))


@DEVICES
@pytest.mark.parametrize("fmt", ["bf16", "fp8", "int8"])
def test_shared_prefix_of_sequences_shorter_than_it(dev, fmt):
    gen = torch.Generator().manual_seed(21)
    sizes, prefixes = [6, 2], [90, 50]
    cache, table, lens, seqs = groups_of(sizes, prefixes, [[1] * 6, [1] * 2], 2, 64, 16, fmt, dev, gen)
    q = rows(8, 8, 64, gen).to(dev)
    plan = ops.shared_prefix_plan(sizes, prefixes, 8, 2, dev)
    short = [91, 0, 1, 32, 90, 89, 0, 0]
    out = ops.shared_prefix_attention(q, cache, table, i32(short, dev), plan, 0.2)
    for s, L in enumerate(short):
        check(out[s:s + 1], *attention(q[s:s + 1].double().cpu(), *seqs[s], [L], 0.2))


@DEVICES
@pytest.mark.parametrize("fmt", ["bf16", "fp8", "int8"])
@pytest.mark.parametrize("D,Hq", [(128, 8), (64, 24), (64, 2)])
@pytest.mark.parametrize("wide", [False, True])
def test_a_value_that_is_not_finite_reaches_only_those_who_see_it(dev, fmt, D, Hq, wide, monkeypatch):
    """Sequences shorter than their prefix beside longer ones; behind the second group's, pages that were never written."""
    if wide:
        monkeypatch.setattr(kv_quant, "WIDE_ROWS", 0)
        monkeypatch.setattr(kv_quant, "WIDE_TILES", 0)
    gen = torch.Generator().manual_seed(23)

    def fill(k, v):
        v[40, 0, 3] = math.inf
        v[95, 1, D - 1] = -math.inf
        v[200, 1, 7] = math.nan
        v[201, 1, 6] = math.nan
        v[299, 0, 17] = math.inf

    sizes, prefixes = [12, 3], [300, 64]
    tails = [[10, 1] + [0] * 10, [1, 1, 1]]
    cache, table, lens, seqs = groups_of(sizes, prefixes, tails, 2, D, 16, fmt, dev, gen, fill)
    short = [310, 301, 300, 299, 41, 40, 39, 200, 201, 0, 96, 64] + [65, 30, 1]
    q = rows(len(short), Hq, D, gen).to(dev)
    plan = ops.shared_prefix_plan(sizes, [300, 200], Hq, 2, dev)
    assert (plan.wide is not None) == wide
    out = ops.shared_prefix_attention(q, cache, table, i32(short, dev), plan, 0.1)
    for s, L in enumerate(short):
        ref, bound = attention(q[s:s + 1].double().cpu(), *seqs[s], [L], 0.1)
        got = out[s:s + 1].double().cpu()
        assert torch.equal(got.isnan(), ref.isnan()) and torch.equal(got[ref.isinf()], ref[ref.isinf()])
        good = ref.isfinite()
        check(got[good], ref[good], bound[good])


@DEVICES
@pytest.mark.parametrize("fmt", ["bf16", "fp8", "int8"])
@pytest.mark.parametrize("Hq,D,sizes,rt", [(8, 128, [3, 2], 1), (8, 64, [4, 2], 1), (12, 128, [9, 2], 2), (40, 64, [5, 2], 2),
                                           (8, 128, [33, 3], 8), (8, 64, [33, 3], 8)])
def test_many_tiles_of_a_shared_prefix(dev, fmt, Hq, D, sizes, rt, monkeypatch):
    """Workgroups with far more 32-key tiles than waves, of common and own keys: tiles that all rows see, then those behind the end of
    the group's shortest sequence, in whose midst is an infinity that some see; the second group has whole tiles only."""
    monkeypatch.setattr(kv_quant, "PREFIX_WGS", 4)
    wide = rt == 8
    monkeypatch.setattr(kv_quant, "WIDE_ROWS", 0 if wide else 1 << 30)
    monkeypatch.setattr(kv_quant, "WIDE_TILES", 0)
    gen = torch.Generator().manual_seed(25)
    prefixes, at = ([1500, 900], 777) if wide else ([3000, 1700], 1777)
    tails = [[600, 1] + [45] * (sizes[0] - 2), [500] + [3] * (sizes[1] - 1)]

    def fill(k, v):
        v[at - 1, 0, 3] = math.inf
        v[at + 40, 1, D - 1] = -math.inf
        v[at + 300, 1, 7] = math.nan
        v[prefixes[0] + 580, 0, 5] = math.inf

    cache, table, lens, seqs = groups_of(sizes, prefixes, tails, 2, D, 16, fmt, dev, gen, fill)
    short = list(lens)
    short[1:3] = [at, at + 41]
    q = rows(len(lens), Hq, D, gen).to(dev)
    plan = ops.shared_prefix_plan(sizes, prefixes, Hq, 2, dev)
    assert plan.work.row_tiles == (1 if sizes[0] * Hq // 2 <= 16 else 2) and (plan.wide is not None) == wide
    if wide and fmt == "bf16":
        assert plan.wide.row_tiles == 8
    for work in (plan.work, plan.wide) if wide else (plan.work,):
        assert max(it[4] - it[3] for it in work.items.tolist()) > 16 * 32
    out = ops.shared_prefix_attention(q, cache, table, i32(short, dev), plan, 0.1, num_splits=1)
    cut = ops.shared_prefix_attention(q, cache, table, i32(short, dev), plan, 0.1, num_splits=3)
    for s in [0, 1, 2, sizes[0] - 1] + list(range(sizes[0], len(lens))):
        ref, bound = attention(q[s:s + 1].double().cpu(), *seqs[s], [short[s]], 0.1)
        good = ref.isfinite()
        assert good.all() == (s >= sizes[0])
        for o in (out, cut):
            got = o[s:s + 1].double().cpu()
            assert torch.equal(got.isnan(), ref.isnan()) and torch.equal(got[ref.isinf()], ref[ref.isinf()])
            check(got[good], ref[good], bound[good])


@DEVICES
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("splits", [1, 2, 3, 5])
def test_an_infinity_in_any_part(dev, D, splits):
    """bf16: a part of a row's keys whose output is infinite, the first, one in the midst or the last of 2 to 6."""
    gen = torch.Generator().manual_seed(26)
    lens, at = [700] * 6, [0, 70, 199, 300, 500, 699]

    def fill(k, v):
        for s, x in enumerate(at):
            v[700 * s + x, s % 2, 5] = math.inf * (1 - 2 * (s % 3 == 0))

    cache, table, truth = make(lens, 2, D, 16, "bf16", dev, gen, fill)
    q = rows(6, 8, D, gen).to(dev)
    plan = ops.shared_prefix_plan([1] * 6, [128] * 6, 8, 2, dev)
    out = ops.shared_prefix_attention(q, cache, table, i32(lens, dev), plan, 0.1, num_splits=splits)
    for s in range(6):
        ref, bound = attention(q[s:s + 1].double().cpu(), *truth[s], [700], 0.1)
        got, good = out[s:s + 1].double().cpu(), ref.isfinite()
        assert int((~good).sum()) == 4 and torch.equal(got[~good], ref[~good])
        check(got[good], ref[good], bound[good])


def test_work_of_a_plan():
    """Every (block of rows, 32 keys) of every group is in one item, in blocks of either size."""
    sizes, prefixes, G, Hkv = [40, 1, 9, 3], [30000, 0, 9001, 31], 4, 8
    plan = ops.shared_prefix_plan(sizes, prefixes, G * Hkv, Hkv, "cpu")
    assert plan.wide is not None and plan.slots == max(plan.work.slots, plan.wide.slots)
    assert ops.shared_prefix_plan([40], [200], G * Hkv, Hkv, "cpu").wide is None
    assert ops.shared_prefix_plan([9], [30000], G * Hkv, Hkv, "cpu").wide is None
    for work in (plan.work, plan.wide):
        at = 0
        for n, p in zip(sizes, prefixes):
            items = [it for it in work.items.tolist() if it[0] == at]
            blocks = -(-n * G // (16 * work.row_tiles))
            assert all(it[1] == n for it in items) and {it[2] for it in items} == (set(range(blocks)) if p else set())
            for b in range(blocks if p else 0):
                mine = sorted((it[3], it[4], it[5]) for it in items if it[2] == b)
                assert mine[0][0] == 0 and mine[-1][1] == p and all(x[1] == y[0] and x[1] % 32 == 0 for x, y in zip(mine, mine[1:]))
                assert [x[2] for x in mine] == list(range(len(mine)))
                assert work.counts[at:at + n].tolist() == [len(mine)] * n and len(mine) <= work.slots
            at += n


@DEVICES
def test_nothing_shared_is_decode(dev):
    gen = torch.Generator().manual_seed(22)
    lens = [65, 3, 0, 200]
    cache, table, truth = make(lens, 2, 128, 16, "int8", dev, gen)
    q = rows(4, 8, 128, gen).to(dev)
    plan = ops.shared_prefix_plan([1, 3], [0, 0], 8, 2, dev)
    assert plan.slots == 0 and plan.work.items.shape[0] == 0
    a = ops.shared_prefix_attention(q, cache, table, i32(lens, dev), plan, 0.1, num_splits=2)
    b = ops.quant_decode_attention(q, cache, table, i32(lens, dev), 0.1, num_splits=2)
    assert torch.equal(a, b)


@DEVICES
@FORMATS
def test_a_conversation(dev, fmt):
    """Prompts written and read by portions, forked behind a common prefix, then decoded step by step."""
    gen = torch.Generator().manual_seed(30)
    Hq, Hkv, D, bs, scale = 8, 2, 128, 16, 1 / math.sqrt(128)
    nb = 40
    cache = ops.QuantKVCache.alloc(nb, Hkv, bs, D, fmt, dev)
    spoil(cache)
    kept_k, kept_v = torch.zeros(nb * bs, Hkv, D, dtype=torch.float64), torch.zeros(nb * bs, Hkv, D, dtype=torch.float64)

    def write(slots, k, v):
        ops.kv_quant_append(k.to(dev), v.to(dev), cache, slots.to(dev, torch.int32))
        kept_k[slots.long()], kept_v[slots.long()] = value(k, fmt), value(v, fmt)

    first = torch.arange(10)
    for lo, hi in ((0, 70), (70, 71), (71, 96)):      # a prompt of 96 tokens by portions
        n = hi - lo
        write(slots_of(first, lo, hi, bs), rows(n, Hkv, D, gen), rows(n, Hkv, D, gen))
        q = rows(n, Hq, D, gen).to(dev)
        out = ops.quant_prefill_attention(q, cache, first[None].to(dev, torch.int32), i32([0, n], dev), i32([hi], dev), n, scale)
        at = slots_of(first, 0, hi, bs)
        check(out, *attention(q.double().cpu(), kept_k[at], kept_v[at], [lo + i + 1 for i in range(n)], scale))
    tables = torch.stack([torch.cat([first[:6], torch.arange(10 + 4 * i, 14 + 4 * i)]) for i in range(5)])
    plan = ops.shared_prefix_plan([5], [96], Hq, Hkv, dev)
    for step in range(20):                            # five answers to it
        L = 96 + step + 1
        slots = torch.stack([slots_of(t, L - 1, L, bs)[0] for t in tables])
        write(slots, rows(5, Hkv, D, gen), rows(5, Hkv, D, gen))
        q = rows(5, Hq, D, gen).to(dev)
        a = ops.shared_prefix_attention(q, cache, tables.to(dev, torch.int32), i32([L] * 5, dev), plan, scale)
        b = ops.quant_decode_attention(q, cache, tables.to(dev, torch.int32), i32([L] * 5, dev), scale)
        for s in range(5):
            at = slots_of(tables[s], 0, L, bs)
            ref = attention(q[s:s + 1].double().cpu(), kept_k[at], kept_v[at], [L], scale)
            check(a[s:s + 1], *ref)
            check(b[s:s + 1], *ref)
    k, v = ops.kv_quant_read(cache, tables.to(dev, torch.int32), i32([90] * 5, dev), i32([0, 26, 52, 78, 104, 130], dev), 130)
    at = torch.cat([slots_of(t, 90, 116, bs) for t in tables])
    for got, want in ((k, kept_k[at]), (v, kept_v[at])):
        assert bool(((got.double().cpu() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -22)).all())


# ------------------------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    bf, f32, i = torch.bfloat16, torch.float32, torch.int32
    z = lambda *s, dtype=bf: torch.zeros(*s, dtype=dtype)  # noqa: E731
    c = ops.QuantKVCache.alloc(4, 2, 16, 64, "fp8", "cpu")
    for bad in (dict(fmt="fp4"), dict(head_dim=96), dict(block_size=24), dict(block_size=0), dict(num_blocks=0),
                dict(num_blocks=1 << 29)):
        a = dict(num_blocks=1, num_kv_heads=1, block_size=16, head_dim=64, fmt="int8", device="meta")
        with pytest.raises(ValueError):
            ops.QuantKVCache.alloc(**{**a, **bad})
    with pytest.raises(ValueError):
        ops.QuantKVCache(c.k, c.v, c.scales[:, :, :1], "fp8")
    with pytest.raises(ValueError):
        ops.QuantKVCache(c.k.transpose(0, 2), c.v.transpose(0, 2), c.scales, "fp8")
    with pytest.raises(TypeError):
        ops.QuantKVCache(c.k.view(torch.int8), c.v, c.scales, "fp8")
    with pytest.raises(ValueError):
        ops.QuantKVCache(c.k, torch.zeros(c.v.numel() + 8, dtype=torch.uint8)[8:].view(c.v.shape), c.scales, "fp8")

    rows3, slots = z(3, 2, 64), z(3, dtype=i)
    for k, v, s, e in ((rows3.float(), rows3, slots, TypeError), (rows3, rows3.half(), slots, TypeError),
                       (rows3, rows3[:2], slots, ValueError), (z(3, 1, 64), z(3, 1, 64), slots, ValueError),
                       (rows3, rows3, slots.long(), TypeError), (rows3, rows3, slots[:2], ValueError),
                       (z(3, 64, 2).transpose(1, 2), rows3, slots, ValueError), (z(2, 3, 64).transpose(0, 1), rows3, slots, ValueError),
                       (z(3, 129)[:, 1:].unflatten(1, (2, 64)), rows3, slots, ValueError)):
        with pytest.raises(e):
            ops.kv_quant_append(k, v, c, s)
    cs = z(8, 64, dtype=f32)
    for qkv, pos, table, e in ((z(3, 6 * 64 - 1), slots, cs, ValueError), (z(1, 6 * 64).expand(3, -1), slots, cs, ValueError),
                               (z(3, 6 * 64), slots.long(), cs, TypeError),
                               (z(3, 6 * 64), slots[:2], cs, ValueError), (z(3, 6 * 64), slots, cs.double(), TypeError),
                               (z(3, 6 * 64), slots, z(8, 32, dtype=f32), ValueError)):
        with pytest.raises(e):
            ops.rope_kv_quant(qkv, pos, table, c, slots, 2)

    bt, ln = z(2, 3, dtype=i), z(2, dtype=i)
    cu = z(3, dtype=i)
    for a, e in (((bt.long(), ln, cu, 1), TypeError), ((bt, ln[:1], cu, 1), ValueError), ((bt, ln, cu[:2], 1), ValueError),
                 ((bt, ln, cu, -1), ValueError), ((bt.t().contiguous().t(), ln, cu, 1), ValueError)):
        with pytest.raises(e):
            ops.kv_quant_read(c, *a)
    with pytest.raises(ValueError):
        ops.kv_quant_read(c, bt, ln, cu, 1, out=(z(1, 2, 64), z(2, 2, 64)))

    q = z(2, 4, 64)
    for args, kw, e in (((q.float(), c, bt, ln), {}, TypeError), ((z(2, 3, 64), c, bt, ln), {}, ValueError),
                        ((z(2, 4, 128), c, bt, ln), {}, ValueError), ((z(4, 2, 64).transpose(0, 1), c, bt, ln), {}, ValueError),
                        ((q, c, bt[:1], ln), {}, ValueError), ((q, c, bt, ln.long()), {}, TypeError),
                        ((q, c, bt[:, :0], ln), {}, ValueError), ((q, c, bt, ln), dict(num_splits=0), ValueError),
                        ((q, c, bt, ln), dict(num_splits=65), ValueError), ((q, c, bt, ln), dict(out=z(2, 4, 32)), ValueError),
                        ((q, c, bt, ln), dict(out=z(1, 4, 64).expand(2, -1, -1)), ValueError),
                        ((z(2, 0, 64), c, bt, ln), {}, ValueError),
                        ((q, c, bt, ln), dict(out=z(2, 4, 64, dtype=f32)), TypeError)):
        with pytest.raises(e):
            ops.quant_decode_attention(*args, 0.1, **kw)
    for args, e in (((q, c, bt, cu[:2], ln, 1), ValueError), ((q, c, bt, cu.long(), ln, 1), TypeError), ((q, c, bt, cu, ln, -1), ValueError),
                    ((q, c, bt[:1], cu, ln, 1), ValueError)):
        with pytest.raises(e):
            ops.quant_prefill_attention(*args, 0.1)
    with pytest.raises(ValueError):
        ops.quant_prefill_attention(q, c, bt, cu, ln, 1, 0.1, row_tiles=4)

    for a in (([1], [1, 2], 4, 2), ([0], [1], 4, 2), ([1], [-1], 4, 2), ([1], [1], 3, 2), ([1], [1], 4, 0)):
        with pytest.raises(ValueError):
            ops.shared_prefix_plan(*a, device="cpu")
    plan = ops.shared_prefix_plan([2], [20], 4, 2, "cpu")
    pages = z(4, 2, 16, 64)
    for args, e in (((z(3, 4, 64), c, z(3, 3, dtype=i), z(3, dtype=i), plan), ValueError), ((z(2, 2, 64), c, bt, ln, plan), ValueError),
                    ((q, c, bt[:, :1], ln, plan), ValueError), ((q, (pages.float(), pages.float()), bt, ln, plan), TypeError),
                    ((q, (pages, pages[:2]), bt, ln, plan), ValueError), ((q, (z(4, 2, 8, 64),) * 2, bt, ln, plan), ValueError)):
        with pytest.raises(e):
            ops.shared_prefix_attention(*args, 0.1)
    assert ops.shared_prefix_attention(z(0, 4, 64), c, bt[:0], ln[:0], ops.shared_prefix_plan([], [], 4, 2, "cpu"), 0.1).shape == (0, 4, 64)


# ----------------------------------------------------------------------------------------------------------------- GPU only
@pytest.mark.gpu
def test_a_workspace_too_small_is_refused():
    dev = "cuda"
    c = ops.QuantKVCache.alloc(4, 2, 16, 64, "fp8", dev)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=dev)
    bt, ln = torch.zeros(2, 3, dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
    with pytest.raises(ValueError):
        ops.quant_decode_attention(q, c, bt, ln, 0.1, num_splits=3, workspace=DecodeWorkspace(2, 4, 64, 2, dev))
    with pytest.raises(ValueError):
        ops.quant_decode_attention(q.cpu(), c, bt, ln, 0.1)
    with pytest.raises(ValueError):
        ops.quant_decode_attention(q, c, bt.cpu(), ln, 0.1)


@pytest.mark.gpu
def test_captured_and_replayed_on_another_stream():
    dev, gen = "cuda", torch.Generator().manual_seed(40)
    Hq, Hkv, D, bs, B = 8, 2, 128, 16, 6
    lens = [130, 97, 100, 260, 96, 111]
    cache, table, truth = make(lens, Hkv, D, bs, "fp8", dev, gen)
    table[1:3, :6] = table[0, :6]
    q, k, v = rows(B, Hq, D, gen).to(dev), rows(B, Hkv, D, gen).to(dev), rows(B, Hkv, D, gen).to(dev)
    sl = i32(lens, dev)
    slots = torch.stack([slots_of(table[s].cpu(), n - 1, n, bs)[0] for s, n in enumerate(lens)]).to(dev, torch.int32)
    plan = ops.shared_prefix_plan([3, 3], [96, 0], Hq, Hkv, dev)

    def step():
        ops.kv_quant_append(k, v, cache, slots)
        a = ops.quant_decode_attention(q, cache, table, sl, 0.1, num_splits=3)
        b = ops.shared_prefix_attention(q, cache, table, sl, plan, 0.1, num_splits=2)
        p = ops.quant_prefill_attention(q, cache, table, cu, sl, 2, 0.1, num_splits=2)
        return (a, b, p) + ops.kv_quant_read(cache, table, sl - 1, torch.arange(B + 1, dtype=torch.int32, device=dev), B)

    cu = i32([0, 1, 2, 3, 4, 5, 6], dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held_out = step()
    for i in range(4):
        for t, n in ((q, Hq), (k, Hkv), (v, Hkv)):
            t.copy_(rows(B, n, D, gen))
        sl.copy_(i32([n - (i % 2) for n in lens], dev))
        want = [t.clone() for t in step()]
        cache.k.fill_(0) if i == 3 else None
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held_out, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
@FORMATS
def test_a_cache_behind_32_bits(fmt):
    """Pages whose bytes lie past 2^32, and slots past what a product of 32 bits holds."""
    dev, gen = "cuda", torch.Generator().manual_seed(41)
    Hq, Hkv, D, bs, nb = 16, 8, 128, 16, 280_000
    cache = ops.QuantKVCache.alloc(nb, Hkv, bs, D, fmt, dev)
    assert cache.k.numel() > 1 << 32
    L = 90
    table = i32([[nb - 1, 3, nb - 7, nb - 2, 270_001, 269_999], [0, nb - 3, 1, 262_144, 262_143, 262_145]], dev)
    slots = torch.cat([slots_of(table[s].cpu(), 0, L, bs) for s in (0, 1)]).to(dev, torch.int32)
    k, v = rows(2 * L, Hkv, D, gen), rows(2 * L, Hkv, D, gen)
    ops.kv_quant_append(k.to(dev), v.to(dev), cache, slots)
    rk, rv = ops.kv_quant_read(cache, table, i32([0, 0], dev), i32([0, L, 2 * L], dev), 2 * L)
    tk, tv = value(k, fmt), value(v, fmt)
    for got, want in ((rk, tk), (rv, tv)):
        assert bool(((got.double().cpu() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -22)).all())
    q = rows(2, Hq, D, gen).to(dev)
    out = ops.quant_decode_attention(q, cache, table, i32([L, L], dev), 0.1)
    for s in (0, 1):
        check(out[s:s + 1], *attention(q[s:s + 1].double().cpu(), tk[s * L:(s + 1) * L], tv[s * L:(s + 1) * L], [L], 0.1))
