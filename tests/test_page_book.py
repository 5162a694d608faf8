"""Shared pages of the paged caches on host pools (CPU): forks, copy on write, truncation,
eviction and compaction against plain lists of tokens, and their refusals. The device runs the
same bookkeeping with one copy kernel (tests/test_gpu_pages.py)."""

from __future__ import annotations

import random

import pytest
import torch

import fastest_flash_attention_amd as ffa

H, D, P = 2, 8, 4


def _cache(pages=40):
    return ffa.PagedKVCache(max_pages=pages, page_size=P, num_heads=H, head_dim=D, dtype=torch.float32)


def _tokens(n, start):
    """n distinct tokens: K and V [H, n, D]."""
    k = torch.arange(start, start + n, dtype=torch.float32)[None, :, None].expand(H, n, D).contiguous()
    return k, -k


def _invariants(cache, held=0):
    """Every page is free or owned, never both, with as many owners as tables that hold it."""
    owners = {}
    for seq in cache.sequences.values():
        assert len(seq["page_table"]) >= -(-seq["len"] // P)
        for page in seq["page_table"]:
            if page >= 0:
                owners[page] = owners.get(page, 0) + 1
    assert len(set(cache.free_pages)) == len(cache.free_pages)
    assert not set(cache.free_pages) & set(owners)
    assert len(cache.free_pages) + len(owners) + held == cache.max_pages
    assert cache._owners == {p: n for p, n in owners.items() if n > 1}


def _check(cache, want):
    for s, tokens in want.items():
        k, v = cache.get_kv(s)
        if not tokens:
            assert k is None
            continue
        assert k[0, :, 0].tolist() == tokens and torch.equal(v, -k) and k.shape == (H, len(tokens), D)


@pytest.mark.parametrize("seed", range(12))
def test_random_operations_match_lists(seed):
    rng = random.Random(seed)
    cache, want, clock = _cache(), {}, 1
    for step in range(250):
        kind = rng.choice(["append", "append", "batch", "fork", "truncate", "free", "compact"])
        ids = sorted(want)
        if kind == "append" or not ids:
            s, n = rng.randrange(8), rng.choice([1, 1, 2, 5, 9])
            room = len(cache.free_pages) * P
            if n + 2 * P > room:
                continue
            cache.append_tokens(s, *_tokens(n, clock))
            want[s] = want.get(s, []) + list(range(clock, clock + n))
            clock += n
        elif kind == "batch":
            some, n = rng.sample(ids, rng.randint(1, len(ids))), rng.choice([1, 1, 3])
            if len(cache.free_pages) < 2 * len(some):
                continue
            parts = [_tokens(n, clock + i * n) for i in range(len(some))]
            cache.append_batch(some, torch.stack([k for k, _ in parts]), torch.stack([v for _, v in parts]))
            for i, s in enumerate(some):
                want[s] = want[s] + list(range(clock + i * n, clock + (i + 1) * n))
            clock += n * len(some)
        elif kind == "fork":
            s, t = rng.choice(ids), rng.randrange(8, 16)
            if t in want:
                with pytest.raises(ValueError):
                    cache.fork_sequence(s, t)
                continue
            cache.fork_sequence(s, t)
            want[t] = list(want[s])
        elif kind == "truncate":
            s = rng.choice(ids)
            n = rng.randint(0, len(want[s]))
            cache.truncate_sequence(s, n)
            want[s] = want[s][:n]
        elif kind == "free":
            s = rng.choice(ids)
            cache.free_sequence(s)
            del want[s]
        else:
            moved = cache.compact()
            used = cache.max_pages - len(cache.free_pages)
            assert cache.free_pages == list(range(used, cache.max_pages)) and moved >= 0
        _invariants(cache)
        _check(cache, want)


def test_fork_copies_the_last_page_once():
    """Three owners of a partly filled page: two copies, the last owner writes in place."""
    cache = _cache()
    cache.append_tokens(0, *_tokens(6, 1))
    cache.fork_sequence(0, 1)
    cache.fork_sequence(0, 2)
    free = cache.num_free_pages
    k, v = (torch.stack(x) for x in zip(*(_tokens(1, 100 + i) for i in range(3))))
    cache.append_batch([0, 1, 2], k, v)
    assert cache.num_free_pages == free - 2
    tables = [cache.sequences[s]["page_table"] for s in range(3)]
    assert len({t[0] for t in tables}) == 1 and len({t[1] for t in tables}) == 3
    _check(cache, {i: [1, 2, 3, 4, 5, 6, 100 + i] for i in range(3)})
    _invariants(cache)


def test_failed_copy_leaves_the_page_shared():
    cache = _cache()
    cache.append_tokens(0, *_tokens(6, 1))
    cache.fork_sequence(0, 1)
    before = {s: list(q["page_table"]) for s, q in cache.sequences.items()}, list(cache.free_pages)

    def fails(src, dst):
        raise RuntimeError("no copy")
    cache._copy = fails
    with pytest.raises(RuntimeError, match="no copy"):
        cache.append_tokens(1, *_tokens(1, 50))
    assert before == ({s: q["page_table"] for s, q in cache.sequences.items()}, cache.free_pages)
    del cache._copy
    cache.append_tokens(1, *_tokens(1, 50))
    _check(cache, {0: [1, 2, 3, 4, 5, 6], 1: [1, 2, 3, 4, 5, 6, 50]})
    _invariants(cache)


def test_full_pages_stay_shared():
    cache = _cache()
    cache.append_tokens(0, *_tokens(8, 1))
    cache.fork_sequence(0, 1)
    cache.append_tokens(1, *_tokens(1, 50))
    assert cache.sequences[0]["page_table"] == cache.sequences[1]["page_table"][:2]
    cache.free_sequence(0)
    _check(cache, {1: [1, 2, 3, 4, 5, 6, 7, 8, 50]})
    _invariants(cache)


def test_fork_leaves_pages_without_tokens_to_the_first():
    """A page taken ahead of its tokens (an append that failed) is not written by both."""
    cache = _cache()
    cache.append_tokens(0, *_tokens(4, 1))
    cache.sequences[0]["page_table"].append(cache.allocate_page())
    cache.fork_sequence(0, 1)
    cache.append_tokens(0, *_tokens(1, 50))
    cache.append_tokens(1, *_tokens(1, 60))
    _check(cache, {0: [1, 2, 3, 4, 50], 1: [1, 2, 3, 4, 60]})
    _invariants(cache)


def test_out_of_pages_appends_nothing():
    cache = _cache(pages=3)
    cache.append_tokens(0, *_tokens(5, 1))
    cache.fork_sequence(0, 1)
    cache.append_tokens(2, *_tokens(4, 20))  # the last free page
    before = {s: (list(q["page_table"]), q["len"]) for s, q in cache.sequences.items()}
    with pytest.raises(RuntimeError, match="out of physical pages"):
        cache.append_tokens(1, *_tokens(1, 9))  # its shared page would have to be copied
    with pytest.raises(RuntimeError, match="out of physical pages"):
        cache.append_batch([7, 0], *(t[None].expand(2, -1, -1, -1) for t in _tokens(1, 9)))
    assert before == {s: (q["page_table"], q["len"]) for s, q in cache.sequences.items()}
    _check(cache, {0: [1, 2, 3, 4, 5], 1: [1, 2, 3, 4, 5], 2: [20, 21, 22, 23]})


def test_evict_keeps_sinks_and_window():
    cache = _cache()
    cache.append_tokens(0, *_tokens(30, 1))
    table = list(cache.sequences[0]["page_table"])
    # tokens 0-4 (sinks: pages 0, 1) and 20-29 (window: pages 5-7) stay
    assert cache.evict(0, 10, 5) == 3
    assert cache.sequences[0]["page_table"] == table[:2] + [-1, -1, -1] + table[5:]
    assert cache.evict(0, 10, 5) == 0
    _invariants(cache)
    with pytest.raises(ValueError, match="evicted"):
        cache.get_kv(0)
    cache._check_seen([0], 10, 5)
    cache._check_seen([0], 10, 8)
    for window, sinks in ((11, 5), (10, 9), (None, 5)):
        with pytest.raises(ValueError, match="evicted"):
            cache._check_seen([0], window, sinks)
    with pytest.raises(ValueError, match="evicted"):
        cache.truncate_sequence(0, 17)
    cache.append_tokens(0, *_tokens(3, 90))
    assert cache.sequences[0]["len"] == 33
    cache.free_sequence(0)
    assert cache.num_free_pages == cache.max_pages


def test_evict_of_a_fork_leaves_the_other():
    cache = _cache()
    cache.append_tokens(0, *_tokens(20, 1))
    cache.fork_sequence(0, 1)
    free = cache.num_free_pages
    assert cache.evict(1, 4) == 4 and cache.num_free_pages == free
    _check(cache, {0: list(range(1, 21))})
    cache.compact()
    _check(cache, {0: list(range(1, 21))})
    _invariants(cache)


def test_compaction_leaves_pages_outside_sequences():
    cache = _cache(pages=10)
    cache.append_tokens(0, *_tokens(12, 1))
    held = cache.allocate_page()  # page 3, the caller's
    cache.append_tokens(1, *_tokens(8, 50))
    cache.k_pages[held] = 7.0
    cache.free_sequence(0)
    assert cache.compact() == 2 and cache.sequences[1]["page_table"] == [0, 1]  # were 4, 5
    assert torch.all(cache.k_pages[held] == 7.0) and held not in cache.free_pages
    _check(cache, {1: list(range(50, 58))})
    _invariants(cache, held=1)


def test_refusals():
    cache = _cache()
    cache.append_tokens(0, *_tokens(5, 1))
    with pytest.raises(KeyError):
        cache.fork_sequence(3, 4)
    with pytest.raises(ValueError):
        cache.fork_sequence(0, 0)
    for n in (-1, 6):
        with pytest.raises(ValueError):
            cache.truncate_sequence(0, n)
    with pytest.raises(ValueError):
        cache.evict(0, 0)
    with pytest.raises(ValueError):
        cache.evict(0, 4, -1)
    for src, dst, err in (([0], [40], IndexError), ([-1], [2], IndexError), ([0, 1], [2, 2], ValueError),
                          ([0, 1], [1, 2], ValueError), ([0], [1, 2], ValueError)):
        with pytest.raises(err):
            cache.copy_pages(src, dst)
    k, v = _tokens(1, 1)
    with pytest.raises(ValueError, match="twice"):
        cache.append_batch([0, 0], torch.stack([k, k]), torch.stack([v, v]))
    with pytest.raises(ValueError, match="batch"):
        cache.append_batch([0], torch.stack([k, k]), torch.stack([v, v]))
    with pytest.raises(ValueError, match="rotary"):
        cache.append_batch([0], k[None], v[None], q=k[None])
    with pytest.raises(RuntimeError, match="ROCm"):
        cache.append_batch([0], k[None], v[None], q=k[None], rotary=ffa.FastestFlashRotary(8))
    with pytest.raises(RuntimeError, match="ROCm"):
        ffa.fastest_flash_copy_pages(cache.k_pages, cache.v_pages, [0], [1])
    with pytest.raises(ValueError):
        ffa.fastest_flash_copy_pages(cache.k_pages, cache.v_pages[:3], [0], [1])


def test_latent_cache_shares_pages():
    cache = ffa.MLALatentCache(max_pages=12, page_size=4, latent_dim=8, rope_dim=4, dtype=torch.float32)
    rows = torch.arange(6 * 12, dtype=torch.float32).view(6, 12)
    cache.append(0, rows[:, :8], rows[:, 8:])
    cache.fork_sequence(0, 1)
    new = torch.full((1, 12), -1.0)
    cache.append(1, new[:, :8], new[:, 8:])
    cache.append(0, new[:, :8] * 2, new[:, 8:] * 2)

    def rows_of(s):
        seq = cache.sequences[s]
        return cache.pages[seq["page_table"]].flatten(0, 1)[:seq["len"]]

    assert torch.equal(rows_of(0), torch.cat([rows, 2 * new])) and torch.equal(rows_of(1), torch.cat([rows, new]))
    cache.truncate_sequence(0, 2)
    cache.free_sequence(0)
    cache.compact()
    assert torch.equal(rows_of(1), torch.cat([rows, new]))
    cache.free_sequence(1)
    assert sorted(cache.free_pages) == list(range(12))
