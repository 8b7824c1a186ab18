"""The engine on an 8-bit KV cache: the attention layer on it, whole generations, prefix pages, sizes and refusals."""
import math
import os
import socket
from dataclasses import replace

import pytest
import torch

from tests.test_kv_quant import attention, check, i32, rows
from xgserve import ops
from xgserve.core.errors import CacheDeserialization
from xgserve.engine import EngineConfig, LLMEngine, SamplingParams
from xgserve.engine.kv_io import deserialize, serialize
from xgserve.models import build_model, get_config
from xgserve.models.base import AttnMeta, PagedAttention
from xgserve.ops import kv_quant
from xgserve.server.config import load_config

GPU = pytest.param("cuda", marks=pytest.mark.gpu)
DEVICES = pytest.mark.parametrize("dev", ["cpu", GPU])
FORMATS = pytest.mark.parametrize("fmt", ["fp8", "int8"])


def _engine(fmt, **kw):
    base = dict(model="llama-tiny", device="cpu", dtype="bfloat16", num_blocks=64, max_num_seqs=4, max_num_batched_tokens=64,
                use_graphs=False, kv_cache_dtype=fmt)
    return LLMEngine(EngineConfig(**{**base, **kw}))


@DEVICES
@FORMATS
@pytest.mark.parametrize("parts", [0, 1, 3, 8])
@pytest.mark.parametrize("Hq,Hkv,D,rope", [(8, 2, 128, True), (4, 4, 64, False), (8, 2, 64, True)])
def test_attention_layer(dev, fmt, parts, Hq, Hkv, D, rope):
    """A mixed step (three decode rows, two prompt portions): its rows into the cache, its attention from it. parts: the projection
    as partial sums, rounded to bf16 once after the rotation."""
    gen = torch.Generator().manual_seed(50 + parts)
    bs, nb = 16, 24
    attn = PagedAttention(Hq, Hkv, D, use_rope=rope)
    cache = ops.QuantKVCache.alloc(nb, Hkv, bs, D, fmt, dev)
    before, new = [40, 0, 17, 20, 0], [1, 1, 1, 13, 30]
    tables = torch.randperm(nb, generator=gen)[:20].view(5, 4)
    cs = ops.build_cos_sin(D, 128, 10000.0, device=dev)
    for s, n in enumerate(before):
        at = torch.arange(n)
        slots = (tables[s][at // bs] * bs + at % bs).to(dev, torch.int32)
        ops.kv_quant_append(rows(n, Hkv, D, gen).to(dev), rows(n, Hkv, D, gen).to(dev), cache, slots)
    pos = torch.cat([torch.arange(b, b + n) for b, n in zip(before, new)])
    seq = torch.cat([torch.full((n,), s) for s, n in enumerate(new)])
    slots = tables[seq, pos // bs] * bs + pos % bs
    T = len(pos)
    meta = AttnMeta(num_tokens=T, num_decodes=3, positions=pos.to(dev, torch.int32), slot_mapping=slots.to(dev, torch.int32),
                    dec_block_tables=i32(tables[:3].tolist(), dev), dec_seq_lens=i32([b + 1 for b in before[:3]], dev), num_splits=2,
                    pre_block_tables=i32(tables[3:].tolist(), dev), pre_qsl=i32([0, 13, 43], dev),
                    pre_seq_lens=i32([33, 30], dev), pre_max_q=30)
    x = rows(T, Hq + 2 * Hkv, D, gen).view(T, -1)
    if parts:
        share = torch.randn(parts, T, x.shape[1], generator=gen)
        share[0] += x.float() - share.sum(0)
        pend = ops.PendingSum(share.to(dev), parts)
        full = share.double().sum(0)
        out = attn.from_partials(pend, meta, cache, cs)
    else:
        full = x.double()
        out = attn(x.to(dev), meta, cache, cs)
    out = out.view(T, Hq, D)
    q = full[:, :Hq * D].view(T, Hq, D)
    if rope:
        c = cs.cpu().double()[pos]
        a, b = q[..., :D // 2], q[..., D // 2:]
        co, si = c[:, None, :D // 2], c[:, None, D // 2:]
        q = torch.cat([a * co - b * si, b * co + a * si], -1)
    plain = ops.QuantKVCache(cache.k.cpu(), cache.v.cpu(), cache.scales.cpu(), fmt)
    for t in range(T):
        L = int(pos[t]) + 1
        at = torch.arange(L)
        k, v = (r.double() for r in kv_quant._rows_ref(plain, tables[seq[t]][at // bs] * bs + at % bs))
        ref, bound = attention(q[t:t + 1], k, v, [L], attn.scale)
        # q's rounding to bf16 moves every score by at most 2^-8 of sum |q k|: weights by that, twice
        G = Hq // Hkv
        work = torch.einsum("hd,lhd->hl", q[t].abs(), k.abs().repeat_interleave(G, 1)).amax(-1)[:, None] * attn.scale
        p = torch.softmax(torch.einsum("hd,lhd->hl", q[t], k.repeat_interleave(G, 1)) * attn.scale, -1)
        size = torch.einsum("hl,lhd->hd", p, v.abs().repeat_interleave(G, 1))
        check(out[t:t + 1], ref, bound + size * torch.expm1(2 * work * (2.0 ** -8 + parts * 2.0 ** -20)))


@FORMATS
def test_generation_and_prefix_pages(fmt):
    sp = SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True)
    prompts = [[1] + list(range(20, 60)), [1] + list(range(20, 52)) + [7, 8], [1, 2, 3]]
    a = _engine(fmt)
    outs = a.generate(prompts, sp)
    assert [len(o) for o in outs] == [6, 6, 6]
    assert _engine(fmt, enable_prefix_cache=False).generate(prompts, sp) == outs
    assert _engine(fmt, max_num_batched_tokens=16).generate(prompts, sp) == outs      # prompts by portions
    entry = a.export_prefix(prompts[0])
    assert entry.token_count == 32 and entry.kv.dtype == torch.uint8
    back = deserialize(serialize(entry))
    assert back.equivalent(entry) and back.meta == {"kv_cache_dtype": fmt}
    b = _engine(fmt)
    assert b.import_prefix(back) == 2
    again = b.export_prefix(prompts[0])
    assert again.equivalent(entry)
    assert b.generate(prompts, sp) == outs
    other = _engine("int8" if fmt == "fp8" else "fp8")
    with pytest.raises(ValueError, match="KV dtype"):
        other.import_prefix(back)
    with pytest.raises(ValueError, match="KV dtype"):
        _engine(None).import_prefix(back)
    back.kv = back.kv.float()
    with pytest.raises(ValueError, match="uint8"):
        b.import_prefix(back)
    with pytest.raises(CacheDeserialization):
        deserialize(serialize(entry)[:-1])


def test_sizes():
    wide, small = _engine(None), _engine("int8")
    D = wide.mcfg.head_dim
    assert small.runner.kv_bytes() * 2 * D == wide.runner.kv_bytes() * (D + 4)
    assert small._block_bytes() * small.num_blocks == small.runner.kv_bytes()
    assert wide._block_bytes() * wide.num_blocks == wide.runner.kv_bytes()


def test_refusals():
    with pytest.raises(ValueError, match="bfloat16"):
        _engine("fp8", dtype="float32")
    with pytest.raises(ValueError, match="page layout"):
        _engine("fp8", model="bazurax-tiny", block_size=4)
    with pytest.raises(ValueError, match="format"):
        _engine("fp4")
    with pytest.raises(Exception, match="kv_cache_dtype"):
        load_config(None, cli=["worker.kv_cache_dtype=int4"])
    with pytest.raises(Exception, match="bf16 activations"):
        load_config(None, cli=["worker.kv_cache_dtype=int8", "worker.quantization=fp32"])
    assert load_config(None, cli=["worker.kv_cache_dtype=int8"]).worker.kv_cache_dtype == "int8"


@pytest.mark.gpu
@FORMATS
def test_engine_on_the_gpu(fmt):
    """Graphs, eager steps and prompts by portions give the same tokens, and each is near the top of the fp32 model's logits on the
    same tokens. An E4M3 number is off by at most 2^-4 of itself, so an attention output by about that share of itself (int8: of the
    largest number by 2^-8): half a deviation of the logits, where a wrong kernel's token is several below the top."""
    from xgserve.models.reference import reference_logits
    cfg = replace(get_config("llama3-8b"), num_layers=2, name="llama3-8b-2l")
    model = build_model(cfg, device="cuda:0", seed=3)
    prompts = [[128000] + list(range(1000, 1100)), [128000, 5, 6, 7], [128000] + list(range(300, 331))]
    sp = SamplingParams(max_tokens=8, temperature=0.0, ignore_eos=True)

    def run(**kw):
        base = dict(model=cfg.name, device="cuda:0", num_blocks=256, max_num_seqs=8, max_num_batched_tokens=1024, max_model_len=512,
                    graph_batch_sizes=[1, 2, 4], kv_cache_dtype=fmt)
        return LLMEngine(EngineConfig(**{**base, **kw}), model=model).generate(prompts, sp)

    outs = run()
    assert run(use_graphs=False) == outs
    for p, o in zip(prompts, outs):
        ref = reference_logits(model, p + o[:-1]).float()
        for i, tok in enumerate(o):
            row = ref[len(p) - 1 + i]
            assert float(row.max() - row[tok]) <= 0.5 * float(row.std())


@pytest.mark.gpu
def test_no_workspace_that_nothing_uses():
    """An engine on an 8-bit cache holds its pages, and no buffer for the parts of the bf16 cache's decode attention."""
    held = {}
    for fmt in (None, "fp8"):
        r = _engine(fmt, device="cuda:0", max_num_seqs=64).runner
        held[fmt] = r.workspace
        assert (r.kv_quant is None) == (fmt is None)
    assert held[None] is not None and held["fp8"] is None


PROMPTS = [[1] + list(range(20, 60)), [1, 5, 6, 7, 8], [1] + list(range(20, 52)) + [7, 8]]


def _near_the_top(model, prompts, outs):
    """As test_engine_on_the_gpu: each token within half a deviation of the fp32 model's logits on the same tokens."""
    from xgserve.models.reference import reference_logits
    for p, o in zip(prompts, outs):
        ref = reference_logits(model, p + o[:-1]).float()
        for i, tok in enumerate(o):
            row = ref[len(p) - 1 + i]
            assert tok < len(row) and float(row.max() - row[tok]) <= 0.5 * float(row.std())


@FORMATS
@pytest.mark.parametrize("name", ["llama-tiny", "mixtral-tiny", "gpt2-tiny"])
def test_families(fmt, name):
    """Whole generations of each family that is served from the 8-bit cache, prompts whole and by portions."""
    sp = SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True)
    eng = _engine(fmt, model=name)
    outs = eng.generate(PROMPTS, sp)
    assert [len(o) for o in outs] == [6, 6, 6]
    assert all(isinstance(c, ops.QuantKVCache) and c.fmt == fmt and bool((c.scales > 0).any()) for c in eng.runner.kv_caches)
    _near_the_top(eng.model, PROMPTS, outs)
    _near_the_top(eng.model, PROMPTS, _engine(fmt, model=name, max_num_batched_tokens=16).generate(PROMPTS, sp))


def _rank(rank, world, port, ck, fmt, q):
    os.environ.update(RANK=str(rank), WORLD_SIZE=str(world), LOCAL_RANK=str(rank), MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    torch.set_num_threads(1)
    try:
        from xgserve.parallel.state import destroy_distributed, init_distributed
        init_distributed(tp_size=world, backend="gloo", device=torch.device("cpu"), timeout_s=120)
        eng = _engine(fmt, model="llama-tiny-gqa8", checkpoint=ck, tp=world, max_model_len=256)
        outs = None
        if rank == 0:
            outs = eng.generate(PROMPTS, SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True))
            eng.stop_followers()
        else:
            eng.follower_loop()
        c = eng.runner.kv_caches[0]
        q.put((rank, None, outs, (c.fmt, c.num_kv_heads, bool((c.scales > 0).any()))))
        destroy_distributed()
    except Exception as e:  # noqa: BLE001 - reported to the parent
        q.put((rank, repr(e), None, None))


@FORMATS
def test_ranks_of_a_group(fmt, tmp_path):
    """Two ranks, each with an 8-bit cache of its own kv heads."""
    from xgserve.models import save_checkpoint
    full = build_model(get_config("llama-tiny-gqa8"), device="cpu", dtype=torch.bfloat16, seed=11)
    ck = str(tmp_path / "ckpt")
    save_checkpoint(full, ck)
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = torch.multiprocessing.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_rank, args=(r, 2, port, ck, fmt, q)) for r in range(2)]
    for p in procs:
        p.start()
    try:
        res = {r[0]: r[1:] for r in (q.get(timeout=240) for _ in procs)}
    finally:
        for p in procs:
            p.join(timeout=60)
            if p.is_alive():
                p.kill()
    assert [res[r][0] for r in (0, 1)] == [None, None]
    assert [res[r][2] for r in (0, 1)] == [(fmt, full.cfg.num_kv_heads // 2, True)] * 2
    _near_the_top(full, PROMPTS, res[0][1])
