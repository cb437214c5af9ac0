"""A paged cache held in 8 bits: the references that run on a CPU, against the
definition in 64 bits, and what they refuse."""
import math

import pytest
import torch

from xllm_service_amd import ops

from kv8_oracle import Cache, attend, layout, same, slots_of


def rows(T, heads, dim, seed, big=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, heads, dim, generator=g) * big
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("dim", [64, 128])
def test_write_begins_goes_on_and_grows(dim):
    cache = ops.kv8_cache(4, 2, dim)
    want = Cache(4, 2, dim)
    for step, slots in enumerate([
            list(range(16, 16 + 21)),            # page 1 whole, page 2 begun
            [37], [38], [39, 40],                # page 2 goes on
            [-1, 41, -1, 4 * 16, 10 ** 9, -7],   # skipped: no slot of the cache
            [0, 1], [2, 2],                      # two for one slot: the later
            [16, 18]]):                          # page 1 anew, with a gap
        # each step's are larger: scales grow over pages that go on
        k, v = (rows(len(slots), 2, dim, 10 * step + i, 3.0 ** step)
                for i in range(2))
        ops.reshape_and_cache_kv8(k, v, *cache, torch.tensor(slots))
        want.write(k, v, slots)
        got = Cache(4, 2, dim).load(*cache)
        for i in range(2):
            assert same(got.x[i], want.x[i])
        assert same(got.scale, want.scale)


def test_scale_borders():
    """Powers of two at the borders 448 * 2^e, zeros, and what is not finite."""
    k = torch.zeros(16, 1, 64, dtype=torch.bfloat16)
    v = k.clone()
    for big, scale in ((448.0, 1.0), (450.0, 2.0), (224.0, 0.5), (0.0, 2.0 ** -126),
                       (2.0 ** -133, 2.0 ** -126), (3.3e38, 2.0 ** 120)):
        cache = ops.kv8_cache(1, 1, 64)
        k[3, 0, 5], v[2, 0, 1] = big, -big
        k[4, 0, 6], v[1, 0, 0] = math.inf, math.nan
        ops.reshape_and_cache_kv8(k, v, *cache, torch.arange(16))
        assert cache[2].tolist() == [[[scale, scale]]]
        assert cache[0].float().isnan().sum() == 1
        assert cache[1].float().isnan().sum() == 1


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
def test_the_largest_values_stay_finite(kind):
    """448 * 2^120 is not: the largest values are 240 * 2^120."""
    most = torch.finfo(kind).max
    for big in (most, -most, 3.3e38, 3.2e38):
        x = torch.full((3, 1, 64), big, dtype=kind)
        cache = ops.kv8_cache(1, 1, 64)
        ops.reshape_and_cache_kv8(x, x, *cache, torch.arange(3))
        assert cache[2].tolist() == [[[2.0 ** 120] * 2]]
        k = cache[0].float().transpose(2, 3).reshape(16, 64)[:3] * 2.0 ** 120
        v = cache[1].float()[0, 0, :, :3] * 2.0 ** 120
        for y in (k, v):
            assert y.to(torch.bfloat16).isfinite().all()
            assert ((y / x.flatten()[0].float() - 1).abs() <= 2.0 ** -4).all()


@pytest.mark.parametrize("per", [1, 3])
def test_attention_of_the_references(per):
    lens, new, dim = [0, 1, 17, 40], [2, 1, 5, 40], 64
    table, pages = layout(lens, 2, 1)
    old = [0] * 4
    cache = ops.kv8_cache(pages, 2, dim)
    slots = slots_of(table, old, lens)
    k, v = rows(len(slots), 2, dim, 2, 2.0), rows(len(slots), 2, dim, 3)
    ops.reshape_and_cache_kv8(k, v, *cache, torch.tensor(slots))
    ref = Cache(pages, 2, dim).load(*cache)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = rows(cu[-1] + 2, 2 * per, dim, 4).float()
    out = torch.full_like(q, 7.0)
    ops.paged_attn_prefill_kv8(q, *cache, table, torch.tensor(cu).int(),
                               torch.tensor(lens).int(), 0.125, out=out)
    want, *_ = attend(q, ref.values(0), ref.values(1), table, cu, lens, 0.125)
    assert torch.allclose(out[:-2].double(), want[:-2], atol=1e-5)
    assert (out[-2:] == 7.0).all()               # behind the last sequence
    assert (out[:2] == 0).all()                  # no keys
    got = ops.paged_attn_decode_kv8(q[:4], *cache, table,
                                    torch.tensor(lens).int(), 0.125)
    want, *_ = attend(q[:4], ref.values(0), ref.values(1), table,
                      list(range(5)), lens, 0.125)
    assert torch.allclose(got.double(), want, atol=1e-5)


def test_values_that_are_not_finite():
    """A NaN among a sequence's values is seen by the rows that see it, and by no
    others; nor is what a page holds behind its last token."""
    lens, dim = [40, 70], 64
    table, pages = layout(lens, 2, 8)
    cache = ops.kv8_cache(pages, 2, dim)
    slots = slots_of(table, [0, 0], lens)
    k, v = rows(len(slots), 2, dim, 2), rows(len(slots), 2, dim, 3)
    v[40 + 20, 1, 5] = math.inf                   # the second one's token 20
    k[40 + 30, 0, 7] = math.nan                   # and 30
    ops.reshape_and_cache_kv8(k, v, *cache, torch.tensor(slots))
    cache[1].view(torch.uint8)[table[0, 2], :, :, 8:] = 0x7f
    q = rows(110, 4, dim, 4).float()
    got = ops.paged_attn_prefill_kv8(q, *cache, table, torch.tensor([0, 40, 110]).int(),
                                     torch.tensor(lens).int(), 0.1)
    assert got[:60].isfinite().all()
    assert got[60:, 2:, 5].isnan().all()
    got[60:, 2:, 5] = 0.0
    assert got[:70].isfinite().all() and got[:, 2:].isfinite().all()
    assert got[70:, :2].isnan().all()
    got = ops.paged_attn_decode_kv8(q[:2], *cache, table,
                                    torch.tensor([40, 20]).int(), 0.1)
    assert got.isfinite().all()
    got = ops.paged_attn_decode_kv8(q[:2], *cache, table,
                                    torch.tensor([40, 21]).int(), 0.1)
    assert got[1, 2:, 5].isnan().all() and got[0].isfinite().all()


def test_attention_reads_the_pages_of_its_tables(monkeypatch):
    """Not the pool: what is made of pages in 32 bits is as large as the sequences."""
    from xllm_service_amd.ops import ref
    lens, dim = [40, 0, 70], 64
    table, pages = layout(lens, 300, 8)
    cache = ops.kv8_cache(pages, 2, dim)
    most, plain = [], ref.kv8_values

    def values(k_cache, v_cache, kv_scale):
        most.append(k_cache.shape[0])
        return plain(k_cache, v_cache, kv_scale)
    monkeypatch.setattr(ref, "kv8_values", values)
    n = torch.tensor(lens).int()
    ops.paged_attn_decode_kv8(rows(3, 4, dim, 4), *cache, table, n, 0.1)
    ops.paged_attn_prefill_kv8(rows(7, 4, dim, 4), *cache, table,
                               torch.tensor([0, 2, 4, 7]).int(), n, 0.1)
    assert most and max(most) <= 5


def plan_of(table, old, new, free, room):
    """Token by token, page by page."""
    table = [list(map(int, r)) for r in table]
    slots, pos, cu, at = [], [], [0], 0
    for i, (a, b) in enumerate(zip(old, new)):
        a = max(a, 0)
        for p in range(a, max(b, a)):
            if p % 16 == 0:
                if at < len(free) and p // 16 < len(table[i]):
                    table[i][p // 16] = free[at]
                at += 1
            first = -(-a // 16)
            ok = p // 16 < len(table[i]) and (
                p // 16 < first or at <= len(free))
            slots.append(table[i][p // 16] * 16 + p % 16 if ok else -1)
            pos.append(p)
        cu.append(len(slots))
    more = room - len(slots)
    return table, (slots + [-1] * more)[:room], (pos + [0] * more)[:room], \
        [min(c, room) for c in cu], [at]


@pytest.mark.parametrize("old,new,free,width,room", [
    ([0], [1], 1, 1, 1), ([15, 16, 17], [16, 17, 18], 5, 3, 3),
    ([0, 5, 40, 3], [33, 5, 100, 2], 20, 8, 100),
    ([7, 0], [7, 0], 3, 2, 4), ([], [], 2, 2, 3),
    ([0, 0], [40, 40], 4, 3, 80),           # pages run out
    ([0, 10], [50, 60], 9, 2, 200),         # tables too narrow
    ([0, 3], [20, 20], 9, 4, 25),           # too little room
    ([-3], [5], 2, 2, 5)])
def test_tables_from_lengths(old, new, free, width, room):
    g = torch.Generator().manual_seed(0)
    table = torch.randint(100, 200, (len(old), width), generator=g).int()
    ids = torch.randperm(50, generator=g)[:free].int()
    want = plan_of(table, old, new, ids.tolist(), room)
    got = ops.extend_block_tables(table, torch.tensor(old).int(),
                                  torch.tensor(new).int(), ids, room)
    assert table.tolist() == want[0]
    assert [t.tolist() for t in got] == list(want[1:])
    assert [t.dtype for t in got] == [torch.int64, torch.int64, torch.int32,
                                      torch.int32]


def test_tables_from_lengths_of_any_size():
    most = 2 ** 31 - 1
    old = torch.tensor([3, 0, most, most]).int()
    new = torch.tensor([40, most, most, -most]).int()
    table = torch.zeros(4, 3, dtype=torch.int32)
    slots, pos, cu, used = ops.extend_block_tables(
        table, old, new, torch.arange(1, 8).int(), 100)
    # lengths count as 2^24 - 1 at most, which is 2^20 pages
    assert table.tolist() == [[0, 1, 2], [3, 4, 5], [0, 0, 0], [0, 0, 0]]
    assert pos.tolist() == [*range(3, 40), *range(63)]
    assert cu.tolist() == [0, 37, 100, 100, 100]
    assert used.tolist() == [2 + 2 ** 20]
    with pytest.raises(RuntimeError):
        ops.extend_block_tables(table, old, new, table[0], 2 ** 20 + 1)


def test_a_run_of_them():
    """Three steps of two sequences: planned, written and attended, against the
    same over all tokens at once."""
    table = torch.zeros(2, 4, dtype=torch.int32)
    free = torch.tensor([5, 2, 7, 0, 3, 6, 1, 4]).int()
    cache = ops.kv8_cache(8, 1, 64)
    want = Cache(8, 1, 64)
    lens, seed = torch.zeros(2, dtype=torch.int32), 0
    for grow in ([20, 0], [1, 30], [1, 1]):
        new = lens + torch.tensor(grow).int()
        slots, pos, cu, used = ops.extend_block_tables(table, lens, new, free,
                                                       sum(grow))
        free = free[int(used):]
        k, v, q = (rows(sum(grow), n, 64, seed + i) for i, n in
                   enumerate((1, 1, 2)))
        seed += 3
        ops.reshape_and_cache_kv8(k, v, *cache, slots)
        want.write(k, v, slots.tolist())
        out = ops.paged_attn_prefill_kv8(q.float(), *cache, table, cu, new, 0.1)
        ref, *_ = attend(q, want.values(0), want.values(1), table, cu.tolist(),
                         new.tolist(), 0.1)
        assert torch.allclose(out.double(), ref, atol=1e-5)
        lens = new


def test_refusals():
    k8, v8, s = ops.kv8_cache(3, 2, 64)
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    at = torch.zeros(4, dtype=torch.long)
    tab = torch.zeros(4, 1, dtype=torch.int32)
    lens = torch.ones(4, dtype=torch.int32)

    def no(f, *args):
        with pytest.raises(RuntimeError):
            f(*args)
    no(ops.kv8_cache, 3, 2, 96)
    w = ops.reshape_and_cache_kv8
    no(w, x, x, k8, v8, s, at[:3])
    no(w, x, x[:3], k8, v8, s, at)
    no(w, x[:, :1], x, k8, v8, s, at)
    no(w, x, x, k8, v8, s, at.int())
    no(w, x, x, k8.view(torch.uint8), v8, s, at)
    no(w, x, x, k8, v8, s.double(), at)
    no(w, x, x, k8[:2], v8, s, at)
    no(w, x, x, v8, k8, s, at)
    d = ops.paged_attn_decode_kv8
    no(d, x[:, :1], k8, v8, s, tab, lens, 1.0)
    no(d, x[..., :32], k8, v8, s, tab, lens, 1.0)
    no(d, x, k8, v8, s, tab.long(), lens, 1.0)
    no(d, x, k8, v8, s, tab[:3], lens, 1.0)
    no(d, x, k8, v8, s, tab, lens[:3], 1.0)
    no(d, torch.zeros(4, 34, 64), k8, v8, s, tab, lens, 1.0)
    cu = torch.tensor([0, 4]).int()
    p = ops.paged_attn_prefill_kv8
    no(p, x, k8, v8, s, tab, cu.long(), lens, 1.0)
    no(p, x, k8, v8, s, tab[:0], cu, lens, 1.0)
    no(p, x, k8, v8, s[:2], tab, cu, lens, 1.0)


# ---- the engine over such a cache --------------------------------------------
def engine(model="llama-tiny", **kw):
    from xllm_service_amd.engine.engine import LLMEngine
    return LLMEngine(model, device="cpu", seed=3, max_num_seqs=4, **kw)


PROMPTS = [[5, 9, 2, 7] * 9, [3], list(range(40, 75))]


@pytest.mark.parametrize("model", ["llama-tiny", "opt-125m"])
def test_engine(model):
    """Prompts in chunks and tokens behind them, pages that are shared, and blocks
    that move as bytes."""
    from xllm_service_amd.engine.sampling import SamplingParams
    sp = SamplingParams(max_tokens=6, ignore_eos=True)
    eng = engine(model, max_kv_blocks=40, kv_cache_dtype="fp8",
                 max_batched_tokens=16)
    out = eng.generate(PROMPTS, sp)
    assert [len(o) for o in out] == [6] * 3
    assert eng.generate(PROMPTS, sp) == out          # over pages of before
    assert all(len(c) == 3 for c in eng.runner.kv_caches)
    other = engine(model, max_kv_blocks=40, kv_cache_dtype="fp8")
    other.import_block_bytes([4, 2], eng.export_block_bytes([0, 1]))
    for a, b in zip(eng.runner.paged_tensors(), other.runner.paged_tensors()):
        assert torch.equal(a[:2].view(torch.uint8), b[[4, 2]].view(torch.uint8))
    with pytest.raises(ValueError):
        engine(model, max_kv_blocks=8).import_block_bytes(
            [0], eng.export_block_bytes([0]))


def test_engine_first_logits():
    """Logits over 8-bit pages are near those over 32-bit ones: values are off by
    2^-4 of themselves at most, and what attention adds to a row by as much of the
    sum of their sizes."""
    from xllm_service_amd.engine.metadata import AttnMetadata
    outs = []
    for kind in (None, "fp8"):
        eng = engine(max_kv_blocks=8, kv_cache_dtype=kind)
        T = 37
        meta = AttnMetadata(
            T, 0, torch.arange(T), cu_q=torch.tensor([0, T]).int(),
            prefill_seq_lens=torch.tensor([T]).int(),
            prefill_block_tables=torch.arange(3).int()[None])
        attn = eng.model.layers[0].attn
        x = torch.randn(T, eng.cfg.hidden_size,
                        generator=torch.Generator().manual_seed(1))
        attn.o_proj = torch.nn.Identity()
        with torch.inference_mode():
            outs.append(attn(x, torch.arange(T), eng.runner.kv_caches[0], meta,
                             eng.model.cos_sin))
            kv = attn.qkv_proj(x)
    heads = eng.cfg.num_kv_heads * eng.cfg.head_dim
    k, v = kv[:, -2 * heads:-heads], kv[:, -heads:]
    q = kv[:, :-2 * heads]
    # a score moves by at most 2^-4 |q| |k| (and the least step of a page)
    off = 2.0 ** -4 * q.unflatten(1, (-1, 64)).norm(dim=-1).max() \
        * k.unflatten(1, (-1, 64)).norm(dim=-1).max() / 8
    bound = (2.0 ** -4 + 2 * off) * v.abs().max() + 2.0 ** -9 * v.abs().max()
    diff = (outs[0] - outs[1]).abs().max()
    assert 0 < diff < bound


@pytest.mark.parametrize("kind", [None, "fp8"])
def test_engine_imports_blocks_of_its_cache(kind):
    """Too few bytes change nothing; an 8-bit cache takes those of its blocks alone,
    others what is behind them as well, as they did."""
    eng = engine(max_kv_blocks=8, kv_cache_dtype=kind)
    tensors = eng.runner.paged_tensors()
    for i, c in enumerate(tensors):
        c.fill_(1 + i % 3)
    data = eng.export_block_bytes([1, 2])
    for c in tensors:
        c.fill_(7)
    with pytest.raises(ValueError, match="another cache"):
        eng.import_block_bytes([3, 4], data[:-1])
    assert all((c == 7).all() for c in tensors)
    if kind is not None:
        with pytest.raises(ValueError, match="another cache"):
            eng.import_block_bytes([3, 4], data + b"x")
        assert all((c == 7).all() for c in tensors)
    eng.import_block_bytes([3, 4], data if kind else data + b"beyond")
    for i, c in enumerate(tensors):
        assert (c[3:5] == 1 + i % 3).all() and (c[:3] == 7).all()


@pytest.fixture
def anyio_backend():
    return "asyncio"


@pytest.mark.anyio
@pytest.mark.parametrize("kinds", [("fp8", "fp8"), ("fp8", None), (None, "fp8")])
async def test_workers_of_a_pair(kinds):
    """Prompt and tokens on two workers: blocks of 8 bits move between equal caches; of
    a pair of different ones the request ends before its prompt is computed."""
    from tests.test_service_integration import (http_client, make_master,
                                                wait_for, worker_kwargs)
    from xllm_service_amd.engine.worker import Worker
    master = make_master(policy="RR")
    await master.start(serve_http=False)
    pair = [Worker(name, role, **worker_kwargs(
        master, engine_kwargs=dict(seed=11, kv_cache_dtype=kind)))
        for name, role, kind in zip(("p0", "d0"), ("PREFILL", "DECODE"), kinds)]
    try:
        for w in pair:
            await w.start()
        await wait_for(lambda: master.scheduler.has_available_instances()
                       and "d0" in pair[0].peers and "p0" in pair[1].peers)
        assert pair[0].peers["d0"].kv_cache_dtype == (kinds[1] or "")
        client = await http_client(master)
        r = await client.post("/v1/completions", json={
            "model": "llama-tiny", "prompt": list(range(50, 90)),
            "max_tokens": 6, "temperature": 0.0, "ignore_eos": True})
        await client.aclose()
        if kinds[0] == kinds[1]:
            assert r.status_code == 200, r.text
            assert r.json()["usage"]["completion_tokens"] == 6
        else:
            assert r.status_code != 200 and "cache" in r.text, r.text
            assert pair[0].engine.stats.steps == 0
            for w in pair:
                bm = w.engine.block_manager
                assert bm.num_free == bm.num_blocks
    finally:
        for w in pair:
            await w.stop()
        await master.stop()


@pytest.mark.parametrize("tier", ["dram", "ssd"])
def test_engine_swaps(tier, tmp_path):
    """Preempted sequences' pages go to the host's memory or to files, and come back
    with their scales: the tokens are those of a pool that holds all of them."""
    import os

    from xllm_service_amd.engine.sampling import SamplingParams
    g = torch.Generator().manual_seed(17)
    prompts = [torch.randint(0, 500, (60,), generator=g).tolist() for _ in range(2)]
    sp = SamplingParams(max_tokens=8, ignore_eos=True)
    want = engine(max_kv_blocks=64, kv_cache_dtype="fp8",
                  enable_prefix_caching=False).generate(prompts, sp)
    spool = str(tmp_path / "spool")
    kw = dict(swap_space_mb=0, ssd_swap_dir=spool) if tier == "ssd" else {}
    # two sequences of four blocks, each of which needs a fifth
    eng = engine(max_kv_blocks=9, kv_cache_dtype="fp8",
                 enable_prefix_caching=False, **kw)
    assert (eng.cpu_block_manager is None) == (tier == "ssd")
    assert eng.generate(prompts, sp) == want
    assert eng.scheduler.num_swap_outs > 0 and eng.scheduler.num_swap_ins > 0
    assert eng.block_manager.num_free == eng.block_manager.num_blocks
    if tier == "ssd":
        assert os.listdir(spool) == []
    else:
        assert eng.cpu_block_manager.num_free == eng.cpu_block_manager.num_blocks


def test_engine_of_several_ranks_does_not_swap(tmp_path):
    with pytest.raises(ValueError, match="several ranks"):
        engine(kv_cache_dtype="fp8", tp_size=2, ssd_swap_dir=str(tmp_path))


@pytest.mark.parametrize("heads,kv_heads,good", [
    (32, 2, True), (34, 2, False), (17, 1, False)])
def test_query_heads_per_key_head(heads, kv_heads, good):
    import dataclasses

    from xllm_service_amd.engine.cache_spec import PagedKV8, default_specs
    from xllm_service_amd.models.config import get_config
    cfg = dataclasses.replace(get_config("llama-tiny"), num_heads=heads,
                              num_kv_heads=kv_heads)
    if good:
        assert isinstance(default_specs(cfg, kv_heads, "fp8")[0], PagedKV8)
    else:
        with pytest.raises(ValueError, match="16 query heads"):
            default_specs(cfg, kv_heads, "fp8")
    assert len(default_specs(cfg, kv_heads)) == cfg.num_layers


def test_engine_holds_twice_the_blocks_and_refuses():
    from xllm_service_amd.engine.cache_spec import default_specs
    from xllm_service_amd.models.config import get_config
    cfg = get_config("llama-3-8b")
    two = [sum(s.block_bytes(16, 2) for s in default_specs(cfg, 8, kind))
           for kind in (None, "fp8")]
    assert 1.98 < two[0] / two[1] <= 2.0
    for model, kind in (("llama-tiny", "int8"), ("qwen2-vl-tiny", "fp8"),
                        ("zokanex-tiny", "fp8")):
        with pytest.raises(ValueError):
            engine(model, max_kv_blocks=8, kv_cache_dtype=kind)
