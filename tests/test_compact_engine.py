"""Engines with a compact cache, without a GPU: the cache manager's books where requests evict, the arrays of a step, the options and what refuses them."""
from __future__ import annotations

import numpy as np
import pytest

from conftest import TINY_CONFIGS
from pylon_b200.cache import CacheError, CacheManager
from pylon_b200.cache.manager import group_page_counts
from pylon_b200.config import EngineConfig
from pylon_b200.engine.step import StepEntry, StepFunction, StepLayout
from pylon_b200.parts.base import CacheNeed, CompactCache, KVNeed


def evicting(keep=10, page_size=4, num_pages=32, kv_heads=(2, 2)):
    needs = [CacheNeed(kv=KVNeed(heads, 32, compact=CompactCache(4, 32, keep, 1, 2))) for heads in kv_heads]
    return CacheManager(needs, [None] * len(needs), page_size=page_size, num_pages=num_pages, max_requests=4)


@pytest.mark.parametrize("kv_heads", [(2, 2), (2, 3, 2)])      # one group of layers, two
def test_requests_hold_what_they_may_keep(kv_heads):
    cache = evicting(kv_heads=kv_heads)                       # keep 10, slack 2
    a, b = cache.open("a", 200), cache.open("b", 200)
    most = cache.lifetime_pages(200, 7)
    seen = {id(a): 0, id(b): 0}
    for count in (7, 7, 1, 1, 1, 7, 1, 1, 1, 1, 1, 1, 3):
        over = cache.evict([a, b])
        for request in (a, b):
            held = request.length - request.evicted
            assert held < 12 and (request not in over or held == 10)
            assert all(len(table) == -(-held // 4) for table in request.tables)
        cache.prepare([(a, count), (b, 1)])
        assert all(len(a.tables[g]) <= most[g] for g in range(len(cache.groups)))
        assert a.length - a.evicted + count <= cache.most_held(200, count)
        cache.commit(a)
        cache.commit(b)
        seen[id(a)] += count
        seen[id(b)] += 1
        assert (a.length, b.length) == (seen[id(a)], seen[id(b)])
        cache.check()
    assert cache.evict([b, b, a]) and cache.evict([b, b, a]) == []
    cache.prepare([(a, 2)])
    assert cache.evict([a]) == []                             # in the middle of a step: nothing
    cache.rollback(a)
    held = a.length - a.evicted
    assert len(a.tables[0]) == -(-held // 4)
    cache.close(a)
    cache.close(b)
    assert cache.free_pages() == [32] * len(cache.groups) and cache.evict([a]) == []
    again = cache.open("a", 20)
    assert again.evicted == 0


def test_a_request_is_not_shorter_than_the_pool_says():
    needs = [CacheNeed(kv=KVNeed(2, 32, compact=CompactCache(4, 32, 100, 4, 10)))]
    counts = group_page_counts(needs, 16, 1 << 20, 3, 100_000, 64)
    assert counts[needs[0].kv] == 3 * -(-(100 + 25 + 64) // 16)
    assert group_page_counts(needs, 16, 1 << 20, 3, 90, 64)[needs[0].kv] == 3 * 6


def test_bytes_of_a_token():
    packed = KVNeed(8, 128, compact=CompactCache(4, 64))
    assert packed.row_bytes(2) == 8 * (128 + 2 * 2 * 2) and not packed.bounded
    assert KVNeed(8, 128, compact=CompactCache(16, keep=100)).row_bytes(2) == 8 * 128 * 4 + 64
    assert KVNeed(8, 128, value_dim=64).row_bytes(4) == 8 * 192 * 4


def test_layers_that_evict_by_different_rules_are_refused():
    needs = [CacheNeed(kv=KVNeed(2, 32, compact=CompactCache(4, 32, keep))) for keep in (10, None)]
    with pytest.raises(ValueError, match="same rule"):
        CacheManager(needs, [None, None], page_size=4, num_pages=8, max_requests=1)


@pytest.mark.parametrize("padded", [False, True])
def test_the_arrays_of_a_step(padded):
    cache = evicting()
    a, b = cache.open("a", 100), cache.open("b", 100)
    for count in (9, 9):
        cache.evict([a, b])
        cache.prepare([(a, count), (b, 1)])
        cache.commit(a)
        cache.commit(b)
    cache.evict([a, b])
    assert (a.length, a.evicted, b.length, b.evicted) == (18, 8, 2, 0)
    entries = [StepEntry(b, [5], (0,)), StepEntry(a, [6, 7, 8], (2,))]
    cache.prepare([(entry.request, len(entry.tokens)) for entry in entries])
    layout = StepLayout(tokens=6 if padded else 4, rows=4 if padded else 2, logits=2, table_widths=(4,), evicts=True)
    buffer = np.full(layout.total, -9, dtype=np.int32)
    filler = StepFunction.__new__(StepFunction)
    filler.cache = cache
    off = layout.offsets
    if padded:
        filler.fill_padded(entries[:1], entries[1:], entries, layout, buffer, 2)
        assert list(buffer[off["kv_len"] : off["kv_len"] + 4]) == [3, 0, 13, 0]
        assert list(buffer[off["cache_slots"] : off["cache_slots"] + 6]) == [2, 10, 11, 12, 0, 0]
    else:
        assert filler.fill(entries, layout, buffer) == (3, 13)
        assert list(buffer[off["kv_len"] : off["kv_len"] + 2]) == [3, 13]
        assert list(buffer[off["cache_slots"] : off["cache_slots"] + 4]) == [2, 10, 11, 12]
    assert list(buffer[off["positions"] : off["positions"] + 4]) == [2, 18, 19, 20]
    for request in (a, b):
        cache.commit(request)
    ones = [StepEntry(a, [1], (0,)), StepEntry(b, [1], (0,))]
    cache.evict([a, b])
    cache.prepare([(a, 1), (b, 1)])
    layout = StepLayout(tokens=2, rows=2, logits=2, table_widths=(4,), evicts=True)
    buffer = np.full(layout.total, -9, dtype=np.int32)
    assert filler.fill(ones, layout, buffer) == (1, 11)
    off = layout.offsets
    assert list(buffer[off["cache_slots"] : off["cache_slots"] + 2]) == [10, 3] and list(buffer[off["kv_len"] : off["kv_len"] + 2]) == [11, 4]
    assert list(buffer[off["positions"] : off["positions"] + 2]) == [21, 3]


@pytest.mark.parametrize("options, message", [
    (dict(cache_bits=8), "cache_bits"), (dict(cache_bits=4.0), "cache_bits"), (dict(cache_keep=0), "cache_keep"), (dict(cache_keep=2.5), "cache_keep"),
    (dict(cache_keep=4), "always kept"), (dict(cache_keep=20, cache_keep_recent=17), "always kept"), (dict(cache_keep=20, cache_keep_first=-1), "cache_keep_first"),
    (dict(cache_keep=20, cache_keep_recent=-1), "cache_keep_recent"),
])
def test_options_that_are_refused(options, message):
    with pytest.raises(ValueError, match=message):
        EngineConfig(**options)


def test_options_that_are_taken(monkeypatch):
    assert EngineConfig().cache_bits == 16 and EngineConfig().cache_keep is None
    assert EngineConfig(cache_bits=4, cache_keep=400).keep_recent == 100
    assert EngineConfig(cache_keep=5).keep_recent == 1
    monkeypatch.setenv("PYLON_B200_CACHE_BITS", "4")
    monkeypatch.setenv("PYLON_B200_CACHE_KEEP", "512")
    config = EngineConfig.from_env()
    assert (config.cache_bits, config.cache_keep) == (4, 512)


def mixer(**options):
    from pylon_b200.parts.attention import GroupedQueryAttention

    fields = dict(width=64, n_heads=4, n_kv_heads=2, head_dim=64)
    fields.update(options)
    return GroupedQueryAttention(**fields)


def test_what_a_mixer_refuses():
    for group, head_dim in ((64, 128), (64, 64), (32, 96), (32, 32)):
        part = mixer(head_dim=head_dim)
        part.compact_cache(CompactCache(4))
        assert part.cache_need().kv.compact.group == group
    with pytest.raises(ValueError, match="multiple of 32"):
        mixer(head_dim=48).compact_cache(CompactCache(4))
    with pytest.raises(ValueError, match="multiple of 16"):
        mixer(head_dim=24).compact_cache(CompactCache(keep=10))
    with pytest.raises(ValueError, match="window"):
        mixer(window=32).compact_cache(CompactCache(keep=10))
    mixer(window=32).compact_cache(CompactCache(4))
    for options in (dict(softcap=5.0), dict(chunk=16), dict(value_dim=32), dict(output_gate="heads"), dict(bias=True)):
        with pytest.raises(ValueError, match="compact cache"):
            mixer(**options).compact_cache(CompactCache(4))


def test_a_model_refuses_for_its_mixers():
    from pylon_b200.config import ARCHITECTURES, Qwen3Config
    from pylon_b200.models.decoder import DecoderModel

    architecture = next(entry for entry in ARCHITECTURES.values() if entry.config_class is Qwen3Config)
    model = DecoderModel(architecture.build_spec(Qwen3Config(**TINY_CONFIGS["tinyA"]), 64))
    with pytest.raises(ValueError, match="multiple of 32"):
        model.compact_caches(CompactCache(4))
    model.compact_caches(CompactCache(keep=20))
    assert all(need.kv.keep == 20 for need in model.cache_needs())


def sized_engine(monkeypatch, total, **options):
    """An engine without weights on a device of ``total`` bytes, 1 GB of them taken: what its pool is sized by."""
    import torch

    from pylon_b200.config import ARCHITECTURES, Qwen3Config
    from pylon_b200.engine.engine import Engine
    from pylon_b200.kernels import ops
    from pylon_b200.models.decoder import DecoderModel

    architecture = next(entry for entry in ARCHITECTURES.values() if entry.config_class is Qwen3Config)
    fields = dict(TINY_CONFIGS["tinyC"], max_position_embeddings=40_960)
    engine = Engine.__new__(Engine)
    engine.device, engine.spec = None, architecture.build_spec(Qwen3Config(**fields), None)
    engine.config = EngineConfig(dtype="bfloat16", page_size=64, max_batch_size=500, prefill_chunk_size=2048, max_gpu_utilization=1.0, **options)
    engine.model = DecoderModel(engine.spec)
    if engine.config.cache_bits == 4 or engine.config.cache_keep:
        engine.model.compact_caches(CompactCache(engine.config.cache_bits, keep=engine.config.cache_keep))
    for block in engine.model.blocks:
        block.mixer.w_qkv = torch.zeros(1, dtype=torch.bfloat16)
    monkeypatch.setattr(ops, "_multiprocessors", lambda device: 148)
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device: (total - (1 << 30), total))
    needs = engine.model.cache_needs()
    return engine, needs, engine._pool_pages(needs, torch.bfloat16, 64)


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("bits, keep", [(16, None), (4, None), (4, 600), (16, 600)])
def test_the_pool_leaves_room_for_workspaces(bits, keep, graphs, monkeypatch):
    """Pages take what is left of the device's share after the weights, a step's activations and what a compact cache's operators take for a while."""
    from pylon_b200.kernels import ops

    total, fields = 6 << 30, TINY_CONFIGS["tinyC"]
    engine, needs, pages = sized_engine(monkeypatch, total, cuda_graphs=graphs, cache_bits=bits, cache_keep=keep)
    compact = CompactCache(bits, keep=keep)
    held = sum(pages[need.kv] * 64 * need.kv.row_bytes(2) for need in needs)
    heads, kv_heads, d = fields["num_attention_heads"], fields["num_key_value_heads"], fields["head_dim"]
    longest = 40_960 if keep is None else min(40_960, keep + compact.slack + 2048 + 256 + 1000)
    room = ops.compact_cache_workspace(1000, 2048 + 256 + 1000, longest, heads, kv_heads, d, 2, bits == 4, 64 if keep else 0, 148)
    assert room > (1 << 29 if bits == 4 else 1 << 24 if keep else -1)
    room = room * (2 if graphs else 1) if bits == 4 or keep else 0
    left = total - (1 << 30) - 2048 * engine.spec.width * 64 - room
    assert held <= left
    if keep is None:   # (an evicting pool is no larger than what its requests may hold)
        assert held > left - (1 << 20)


@pytest.mark.parametrize("keep", [600, 20_000, 40_000])
def test_a_pool_that_evicts_takes_what_there_is(keep, monkeypatch):
    """Requests that may keep more than the device has room for share what it has, as requests that keep everything do."""
    from pylon_b200.cache.manager import group_page_counts

    engine, needs, pages = sized_engine(monkeypatch, 6 << 30, cache_keep=keep)
    most = group_page_counts(needs, 64, 500 * 40_960, 500, 40_960, 2048)
    for need in needs:
        assert 0 < pages[need.kv] <= most[need.kv]
    held = sum(pages[need.kv] * 64 * need.kv.row_bytes(2) for need in needs)
    assert held <= 5 << 30 and (keep == 600 or held > 3 << 30)
