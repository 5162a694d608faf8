"""Page copies and forked sequences on the GPU: bit for bit against indexed copies, and decode
over forked, compacted and evicted caches against caches that own their pages."""

from __future__ import annotations

import random

import pytest
import torch

import fastest_flash_attention_amd as ffa
from tests.gpu_util import require_gpu, say, seeded

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("shape,dt", [
    ((9, 2, 16, 128), BF16),
    ((40, 8, 64, 128), FP16),   # pages of 128 KiB: many pieces
    ((9, 1, 3, 6), FP16),       # 36-byte pages
    ((9, 1, 3, 5), FP16),       # 30-byte pages
    ((9, 3, 5, 33), FP32),
    ((12, 7, 40), BF16),        # one pool of rows, the latent cache's shape
])
def test_copy_pages(shape, dt):
    require_gpu()
    k, v = seeded(shape, dt, 1).cuda(), seeded(shape, dt, 2).cuda()
    ids = torch.randperm(shape[0], generator=torch.Generator().manual_seed(3)).tolist()
    n = shape[0] // 2
    src, dst = ids[:n], ids[n:2 * n]
    src[0] = src[-1]  # a source may serve twice
    for second in (v, None):
        a, b = k.clone(), v.clone()
        say(f"copy pages {shape} {dt} {'two pools' if second is not None else 'one pool'}")
        ffa.fastest_flash_copy_pages(a, b if second is not None else None, src, dst)
        want = k.clone()
        want[dst] = k[src]
        assert torch.equal(a, want)
        want = v.clone()
        if second is not None:
            want[dst] = v[src]
        assert torch.equal(b, want)
        as_tensors = [torch.tensor(x, dtype=torch.int32).cuda() for x in (src, dst)]
        c, d = k.clone(), v.clone()
        ffa.fastest_flash_copy_pages(c, d if second is not None else None, *as_tensors)
        assert torch.equal(a, c) and torch.equal(b, d)


def test_copy_leaves_out_bad_pairs():
    require_gpu()
    k, v = seeded((6, 2, 4, 8), BF16, 1).cuda(), seeded((6, 2, 4, 8), BF16, 2).cuda()
    k0, v0 = k.clone(), v.clone()
    src = torch.tensor([0, -1, 6, 1, 2 ** 31 - 1, 5], dtype=torch.int32).cuda()
    dst = torch.tensor([3, 4, 2, -7, 2, 5], dtype=torch.int32).cuda()
    say("copy pages with ids outside the pool")
    ffa.fastest_flash_copy_pages(k, v, src, dst)
    k0[3], v0[3] = k0[0], v0[0]
    assert torch.equal(k, k0) and torch.equal(v, v0)
    ffa.fastest_flash_copy_pages(k, v, [], [])
    for args, err in (((k, v, [0], [6]), IndexError), ((k, v, [0], [0]), ValueError),
                      ((k, v, src.long(), dst), TypeError), ((k, v, src, [1]), TypeError),
                      ((k, v, src, dst[:2]), ValueError), ((k, v.half(), [0], [1]), ValueError),
                      ((k[:, :1], v[:, :1], [0], [1]), ValueError)):
        with pytest.raises(err):
            ffa.fastest_flash_copy_pages(*args)
    assert torch.equal(k, k0)


def test_copy_in_a_graph():
    require_gpu()
    k, v = seeded((10, 2, 16, 64), BF16, 1).cuda(), seeded((10, 2, 16, 64), BF16, 2).cuda()
    src, dst = (torch.tensor(x, dtype=torch.int32).cuda() for x in ([0, 1], [5, 6]))
    say("copy pages capture")
    ffa.fastest_flash_copy_pages(k, v, src, dst)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ffa.fastest_flash_copy_pages(k, v, src, dst)
    for rep in range(3):
        k.copy_(seeded(k.shape, BF16, 10 + rep))
        v.copy_(seeded(v.shape, BF16, 20 + rep))
        src.copy_(torch.tensor([rep, 9], dtype=torch.int32))
        want_k, want_v = k.clone(), v.clone()
        want_k[[5, 6]], want_v[[5, 6]] = k[[rep, 9]], v[[rep, 9]]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(k, want_k) and torch.equal(v, want_v), f"replay {rep}"


@pytest.mark.parametrize("seed", range(3))
def test_forked_cache_decodes_like_owned_pages(seed):
    """Random forks, appends, truncations and compactions: decode equals that of a cache whose
    sequences were appended whole, bit for bit (the same kernels over other pages)."""
    require_gpu()
    rng, H, D, page, dt = random.Random(seed), 2, 64, 8, FP16
    cache = ffa.PagedKVCache(120, page, H, D, dtype=dt, device="cuda")
    have = {}
    say(f"forked cache {seed}")
    for s in range(3):
        k, v = (seeded((H, 5 + 9 * s, D), dt, 10 * s + i).cuda() for i in range(2))
        cache.append_tokens(s, k, v)
        have[s] = (k, v)
    for step in range(25):
        s = rng.choice(sorted(have))
        kind = rng.choice(["fork", "batch", "batch", "truncate", "compact", "append"])
        if kind == "fork" and len(have) < 7:
            t = max(have) + 1
            cache.fork_sequence(s, t)
            have[t] = have[s]
        elif kind == "truncate" and have[s][0].size(1) > 3:
            n = rng.randint(1, have[s][0].size(1))
            cache.truncate_sequence(s, n)
            have[s] = tuple(x[:, :n] for x in have[s])
        elif kind == "compact":
            cache.compact()
        elif kind in ("batch", "append"):
            ids = sorted(have) if kind == "batch" else [s]
            k, v = (seeded((len(ids), H, 1, D), dt, 1000 + 2 * step + i).cuda() for i in range(2))
            if kind == "batch":
                cache.append_batch(ids, k, v)
            else:
                cache.append_tokens(s, k[0], v[0])
            for i, t in enumerate(ids):
                have[t] = tuple(torch.cat([x, y[i]], dim=1) for x, y in zip(have[t], (k, v)))
    ids = sorted(have)
    whole = ffa.PagedKVCache(400, page, H, D, dtype=dt, device="cuda")
    for t in ids:
        assert all(torch.equal(x, y) for x, y in zip(cache.get_kv(t), have[t]))
        whole.append_tokens(t, *have[t])
    q = seeded((len(ids), 4, D), dt, 5).cuda()
    for x, y in zip(cache.decode(q, ids, return_lse=True), whole.decode(q, ids, return_lse=True)):
        assert torch.equal(x, y)


def test_evicted_cache_decodes_within_its_window():
    require_gpu()
    H, D, page, dt = 2, 64, 8, BF16
    for dt in (BF16, FP32):
        cache = ffa.PagedKVCache(80, page, H, D, dtype=dt, device="cuda")
        for s, n in enumerate((100, 37, 3)):
            cache.append_tokens(s, *(seeded((H, n, D), dt, 3 * s + i).cuda() for i in range(2)))
        q = seeded((3, 4, D), dt, 9).cuda()
        say(f"evicted cache {dt}")
        want = cache.decode(q, [0, 1, 2], sliding_window=20, return_lse=True)
        assert [cache.evict(s, 20) for s in range(3)] == [10, 2, 0]
        cache.k_pages[cache.free_pages] = float("nan")  # other sequences' business by now
        got = cache.decode(q, [0, 1, 2], sliding_window=20, return_lse=True)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        with pytest.raises(ValueError, match="evicted"):
            cache.decode(q, [0, 1, 2])
