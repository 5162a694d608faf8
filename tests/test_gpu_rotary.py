"""Rotary positions and the rotated batched append on the GPU against float64.

Error bound of one value m (a cos - b sin): cos and sin are off by at most 2^-23 (two units in
the last place of sincospi) + 2^-25 (their correction) + 2^-24 (the product with m), the product
and the sum round by 2^-24 each: below (|a| + |b|) |m| 2^-21 together, then one rounding to the
type, half a step of the value.
"""

from __future__ import annotations

import pytest
import torch

import fastest_flash_attention_amd as ffa
from tests.gpu_util import require_gpu, say, seeded

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _ref(x, pos, freq, interleaved, m=1.0, sign=1.0):
    """(value, |a| + |b|) in float64 on the CPU: x [B, H, S, D], pos [B or 1, S]."""
    x, freq = x.detach().double().cpu(), freq.double().cpu()
    n = freq.numel()
    ang = pos.double().cpu()[:, None, :, None] * freq * sign
    cos, sin = ang.cos() * m, ang.sin() * m
    y, size = x.clone(), torch.zeros_like(x)
    ia = torch.arange(0, 2 * n, 2) if interleaved else torch.arange(n)
    ib = ia + 1 if interleaved else ia + n
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * cos - b * sin, b * cos + a * sin
    size[..., ia] = size[..., ib] = (a.abs() + b.abs()) * abs(m)
    return y, size


def _close(got, ref, what):
    y, size = ref
    got = got.detach()
    tol = size * 2.0 ** -21 + (y.abs() + size * 2.0 ** -21) * (torch.finfo(got.dtype).eps / 2)
    off = (got.double().cpu() - y).abs()
    # fp16 values below its normal range step by 2^-24
    tol = tol + (2.0 ** -25 if got.dtype == FP16 else 0.0) * (size > 0)
    worst = (off - tol).max().item() if off.numel() else -1.0
    assert worst <= 0, f"{what}: off by {off.max().item():.3e}, {worst:.3e} over the bound"


CASES = [
    # B, Hq, Hk, S, D, R, dtype, interleaved
    (2, 4, 2, 33, 128, 128, BF16, False),
    (2, 4, 2, 33, 128, 128, BF16, True),
    (1, 3, 1, 7, 96, 48, FP16, True),
    (1, 3, 1, 7, 96, 48, FP16, False),
    (3, 2, 2, 5, 80, 20, BF16, False),     # ten pairs: two at a time
    (3, 2, 2, 5, 80, 20, BF16, True),
    (1, 1, 1, 1, 64, 64, BF16, False),
    (2, 5, 1, 9, 6, 2, FP16, False),       # rows of 12 bytes
    (2, 5, 1, 9, 7, 4, FP16, True),        # rows of 14 bytes
    (2, 3, 3, 17, 33, 10, FP32, False),
    (2, 3, 3, 17, 64, 64, FP32, True),
    (1, 40, 8, 700, 128, 64, BF16, False),  # several heads a thread
    (1, 2, 2, 300, 256, 256, FP16, True),
]


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_rotary_matches_float64(case):
    require_gpu()
    B, Hq, Hk, S, D, R, dt, il = case
    freq = ffa.rotary_frequencies(R, device="cuda")
    q, k = seeded((B, Hq, S, D), dt, 1).cuda(), seeded((B, Hk, S, D), dt, 2).cuda()
    for off in (0, 131071):
        say(f"rotary {case} offset {off}")
        yq, yk = ffa.fastest_flash_rotary(q, k, freq, q_offset=off, interleaved=il)
        pos = torch.arange(off, off + S)[None]
        assert yq.shape == q.shape and yq.dtype == dt and yq.data_ptr() != q.data_ptr()
        _close(yq, _ref(q, pos, freq, il), "q")
        _close(yk, _ref(k, pos, freq, il), "k")
        assert torch.equal(yq[..., R:], q[..., R:])


@pytest.mark.parametrize("dt", [torch.int32, torch.int64])
def test_positions_and_magnitude(dt):
    require_gpu()
    B, S, D = 3, 50, 64
    freq = ffa.rotary_frequencies(64, scaling="yarn", factor=8.0, original_max_position=1024, device="cuda")
    q = seeded((B, 2, S, D), BF16, 3).cuda()
    far = torch.randint(-1000, 2 ** 30, (B, S), generator=torch.Generator().manual_seed(4)).to(dt).cuda()
    for pos in (far, far[:1], far[0], far[:1].expand(B, S), far.t().contiguous().t()):
        say(f"rotary positions {tuple(pos.shape)} {pos.stride()}")
        y, none = ffa.fastest_flash_rotary(q, None, freq, positions=pos, magnitude=1.3)
        full = (pos if pos.dim() == 2 else pos[None]).expand(B, S)
        assert none is None
        _close(y, _ref(q, full, freq, False, m=1.2999999523162842), "positions")


def test_strides_and_layouts():
    """Views of a packed projection, padded and misaligned rows, broadcast batches, 3D."""
    require_gpu()
    B, S, D, dt = 2, 21, 64, BF16
    freq = ffa.rotary_frequencies(32, device="cuda")
    pos = torch.arange(S)[None]
    packed = seeded((B, S, 6 * D + 3), dt, 5).cuda()
    say("rotary packed rows at odd offsets")
    q = packed[..., 1:1 + 4 * D].unflatten(-1, (4, D)).transpose(1, 2)   # odd row stride and offset
    k = packed[..., 4 * D:6 * D].unflatten(-1, (2, D)).transpose(1, 2)
    for il in (False, True):
        yq, yk = ffa.fastest_flash_rotary(q, k, freq, interleaved=il)
        _close(yq, _ref(q, pos, freq, il), "q")
        _close(yk, _ref(k, pos, freq, il), "k")
    say("rotary token-major keeps its order")
    t = seeded((B, S, 4, D), dt, 6).cuda().transpose(1, 2)
    assert ffa.fastest_flash_rotary(t, None, freq)[0].stride() == t.stride()
    say("rotary dim-major, broadcast, 3D")
    d = seeded((B, 4, D, S), dt, 7).cuda().transpose(2, 3)
    _close(ffa.fastest_flash_rotary(d, None, freq)[0], _ref(d, pos, freq, False), "dim stride")
    e = seeded((1, 4, S, D), dt, 8).cuda().expand(B, -1, -1, -1)
    _close(ffa.fastest_flash_rotary(e, None, freq)[0], _ref(e, pos, freq, False), "broadcast")
    x = seeded((B, S, D), dt, 9).cuda()
    y, z = ffa.fastest_flash_rotary(x, x, freq)
    assert y.shape == x.shape and torch.equal(y, z)
    for shape in ((0, 2, 4, D), (2, 2, 0, D), (2, 0, 4, D)):
        assert ffa.fastest_flash_rotary(torch.zeros(shape, dtype=dt, device="cuda"), None, freq)[0].shape == shape


@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("dt", [BF16, FP32])
def test_gradients(dt, il):
    """Against the formula (the rotation back) and against differences: the map is linear, so a
    difference quotient has no error of its own but the values' rounding."""
    require_gpu()
    B, H, S, D, R, m = 2, 3, 19, 48, 32, 1.25
    freq = ffa.rotary_frequencies(R, device="cuda")
    pos = torch.randint(0, 5000, (B, S), generator=torch.Generator().manual_seed(1)).cuda()
    q, k = (seeded((B, H, S, D), dt, s).cuda().requires_grad_() for s in (11, 12))
    dq, dk = (seeded((B, H, S, D), dt, s).cuda() for s in (13, 14))
    say(f"rotary gradients {dt} {il}")
    yq, yk = ffa.fastest_flash_rotary(q, k, freq, positions=pos, interleaved=il, magnitude=m)
    gq, gk = torch.autograd.grad((yq, yk), (q, k), (dq, dk))
    _close(gq, _ref(dq, pos, freq, il, m, -1.0), "dq")
    _close(gk, _ref(dk, pos, freq, il, m, -1.0), "dk")
    # one of the two, a broadcast gradient
    only = torch.autograd.grad(ffa.fastest_flash_rotary(q, k.detach(), freq, positions=pos,
                                                        interleaved=il, magnitude=m)[0].sum(), q)[0]
    _close(only, _ref(torch.ones_like(q), pos, freq, il, m, -1.0), "ones")
    if dt == FP32:
        h = seeded((B, H, S, D), dt, 15).cuda()
        with torch.no_grad():
            up, down = (ffa.fastest_flash_rotary(q + s * h, None, freq, positions=pos, interleaved=il,
                                                 magnitude=m)[0].double() for s in (1.0, -1.0))
        slope = ((up - down) / 2 * dq.double()).sum()
        want = (gq.double() * h.double()).sum()
        # the rounding of q +- h and of the outputs: 2^-22 of each term's size
        size = (dq.double().abs() * (up.abs() + down.abs() + (q.detach().abs() + h.abs()).double() * 2 * m)).sum()
        assert abs(slope - want) <= size * 2.0 ** -22
        twice = torch.autograd.grad(torch.autograd.grad(
            ffa.fastest_flash_rotary(q, None, freq, positions=pos, interleaved=il, magnitude=m)[0], q,
            dq.requires_grad_(), create_graph=True)[0], dq, h)[0]
        _close(twice, _ref(h, pos, freq, il, m), "second order")


def _pool(P, H, page, D, dt, seed):
    return seeded((P, H, page, D), dt, seed).cuda(), seeded((P, H, page, D), dt, seed + 1).cuda()


@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("n,page,il", [(1, 16, False), (1, 5, True), (7, 4, False), (40, 16, True)])
def test_append_matches_loop(dt, n, page, il):
    """Rows reach their slots, padding rows and bad pages are left out, and nothing else of the
    pools changes."""
    require_gpu()
    B, Hq, H, D, R, P, width = 5, 6, 2, 64, 32, 60, 12
    g = torch.Generator().manual_seed(n)
    at = torch.tensor([0, 3, page, -2, page * width - 2], dtype=torch.int32)
    counts = torch.tensor([n, max(n - 1, 0), n, n, n], dtype=torch.int32)
    bt = torch.randperm(P, generator=g)[:B * width].view(B, width).to(torch.int32)
    bt[2, 1] = -1 if n == 1 else bt[2, 1]
    bt[2, 2] = P
    q, k, v = (seeded((B, n, h, D), dt, s).cuda().transpose(1, 2) for h, s in ((Hq, 1), (H, 2), (H, 3)))
    freq = ffa.rotary_frequencies(R, device="cuda")
    for rotate in (True, False):
        kp, vp = _pool(P, H, page, D, dt, 9)
        k0, v0 = kp.clone(), vp.clone()
        say(f"append {dt} n {n} page {page} rotate {rotate}")
        how = dict(q=q, inv_freq=freq, interleaved=il, magnitude=0.5) if rotate else {}
        yq = ffa.fastest_flash_paged_append(k, v, kp, vp, bt.cuda(), at.cuda(), counts=counts.cuda(), **how)
        pos = at.long()[:, None] + torch.arange(n)
        if rotate:
            _close(yq, _ref(q, pos, freq, il, 0.5), "q")
            want, size = _ref(k, pos, freq, il, 0.5)
        else:
            assert yq is None
        touched = torch.zeros(P, page, dtype=torch.bool)
        for b in range(B):
            for j in range(n):
                t = int(pos[b, j])
                if t < 0 or j >= counts[b] or t // page >= width:
                    continue
                phys = int(bt[b, t // page])
                if not 0 <= phys < P:
                    continue
                touched[phys, t % page] = True
                assert torch.equal(vp[phys, :, t % page], v[b, :, j])
                if rotate:
                    _close(kp[phys, :, t % page], (want[b, :, j], size[b, :, j]), f"k {b} {j}")
                else:
                    assert torch.equal(kp[phys, :, t % page], k[b, :, j])
        keep = ~touched.cuda()[:, None, :, None].expand_as(kp)
        assert torch.equal(kp[keep], k0[keep]) and torch.equal(vp[keep], v0[keep])
        if n == 1:  # the same rows given without the token dim
            k2, v2 = k0.clone(), v0.clone()
            y2 = ffa.fastest_flash_paged_append(k[:, :, 0], v[:, :, 0], k2, v2, bt.cuda(), at.cuda(),
                                                counts=counts.cuda(), **dict(how, **({"q": q[:, :, 0]} if rotate else {})))
            assert torch.equal(k2, kp) and torch.equal(v2, vp)
            assert y2 is None or torch.equal(y2, yq[:, :, 0])


def test_cache_append_batch_equals_single_appends():
    """PagedKVCache.append_batch with rotation: what rotating and appending one by one gives."""
    require_gpu()
    H, D, page, dt = 2, 64, 8, BF16
    rot = ffa.FastestFlashRotary(64, scaling="linear", factor=2.0, device="cuda")
    one = ffa.PagedKVCache(64, page, H, D, dtype=dt, device="cuda")
    many = ffa.PagedKVCache(64, page, H, D, dtype=dt, device="cuda")
    lens = [0, 5, 8, 31]
    for s, n in enumerate(lens):
        k, v = seeded((H, n, D), dt, 20 + s).cuda(), seeded((H, n, D), dt, 30 + s).cuda()
        for cache in (one, many):
            cache.append_tokens(s, k, v)
    for step, n in enumerate((1, 1, 13)):
        q, k, v = (seeded((4, h, n, D), dt, 40 + 3 * step + i).cuda() for i, h in enumerate((4, H, H)))
        say(f"append_batch step {step}")
        yq = many.append_batch([0, 1, 2, 3], k, v, q=q, rotary=rot)
        for s in range(4):
            at = one.sequences.get(s, {"len": 0})["len"]
            rq, rk = rot(q[s:s + 1], k[s:s + 1], q_offset=at)
            assert torch.equal(yq[s], rq[0])
            one.append_tokens(s, rk[0], v[s])
    for s in range(4):
        for x, y in zip(one.get_kv(s), many.get_kv(s)):
            assert torch.equal(x, y)


def test_graph_replays_and_streams():
    """Rotation and append captured once, replayed over refilled inputs with eager work between;
    the same calls on another stream."""
    require_gpu()
    B, Hq, H, D, page, P, dt = 3, 4, 2, 128, 16, 24, BF16
    freq = ffa.rotary_frequencies(D, device="cuda")
    q, k, v = (seeded((B, h, 1, D), dt, s).cuda() for h, s in ((Hq, 1), (H, 2), (H, 3)))
    kp, vp = _pool(P, H, page, D, dt, 4)
    bt = torch.randperm(P, generator=torch.Generator().manual_seed(5)).view(B, -1).to(torch.int32).cuda()
    at = torch.tensor([0, 5, 127], dtype=torch.int32).cuda()

    def calls():
        y = ffa.fastest_flash_paged_append(k, v, kp, vp, bt, at, q=q, inv_freq=freq)
        return y, *ffa.fastest_flash_rotary(q, k, freq, q_offset=7)

    say("rotary capture")
    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = calls()
    for rep in range(3):
        for t, s in ((q, 50), (k, 60), (v, 70)):
            t.copy_(seeded(t.shape, dt, s + rep))
        at.copy_(torch.tensor([rep, 16 * rep + 15, 100 - rep], dtype=torch.int32))
        for t in outs:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        got, pools = [t.clone() for t in outs], (kp.clone(), vp.clone())
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            want = calls()
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), f"replay {rep}"
        assert torch.equal(pools[0], kp) and torch.equal(pools[1], vp)


def test_gpu_refusals():
    require_gpu()
    q = torch.zeros(2, 2, 4, 8, device="cuda", dtype=BF16)
    f = ffa.rotary_frequencies(8, device="cuda")
    for bad, err in ((f.float(), TypeError), (f.cpu(), RuntimeError), (ffa.rotary_frequencies(10, device="cuda"), ValueError)):
        with pytest.raises(err):
            ffa.fastest_flash_rotary(q, None, bad)
    pos = torch.zeros(2, 4, device="cuda", dtype=torch.int32)
    for kw, err in ((dict(positions=pos.float()), TypeError), (dict(positions=pos[:, :3]), ValueError),
                    (dict(positions=pos.cpu()), RuntimeError), (dict(positions=pos, q_offset=1), ValueError),
                    (dict(positions=torch.zeros(3, 4, device="cuda", dtype=torch.int32)), ValueError),
                    (dict(magnitude=float("nan")), ValueError)):
        with pytest.raises(err):
            ffa.fastest_flash_rotary(q, None, f, **kw)
    with pytest.raises(TypeError):
        ffa.fastest_flash_rotary(q.double(), None, f)
    pool = torch.zeros(4, 2, 4, 8, device="cuda", dtype=BF16)
    bt, at = torch.zeros(2, 2, device="cuda", dtype=torch.int32), torch.zeros(2, device="cuda", dtype=torch.int32)
    for args, err in (((q, q, pool, pool.half(), bt, at), TypeError), ((q, q, pool, pool, bt[:1], at), ValueError),
                      ((q, q, pool, pool, bt, at[:1]), ValueError), ((q, q, pool, pool, bt.cpu(), at), RuntimeError),
                      ((q, q, pool.transpose(1, 2), pool, bt, at), ValueError)):
        with pytest.raises(err):
            ffa.fastest_flash_paged_append(*args)


def test_offsets_past_32_bits():
    """Rows and pages past 4 GiB of a tensor or pool: the same as those at its beginning."""
    require_gpu()
    say("rotary past 4 GiB")
    S, H, D = 270000, 64, 128
    q = torch.empty(1, S, H, D, dtype=BF16, device="cuda").transpose(1, 2)
    tail = seeded((1, H, 37, D), BF16, 1).cuda()
    q[:, :, :-37].zero_()
    q[:, :, -37:] = tail
    assert q.numel() * 2 > 1 << 32
    freq = ffa.rotary_frequencies(D, device="cuda")
    got, _ = ffa.fastest_flash_rotary(q, None, freq)
    want, _ = ffa.fastest_flash_rotary(tail, None, freq, q_offset=S - 37)
    assert torch.equal(got[:, :, -37:], want) and not got[:, :, :-37].any()
    del q, got
    P, page, Hkv = 34000, 64, 8
    pools = [torch.empty(P, Hkv, page, D, dtype=BF16, device="cuda") for _ in range(2)]
    small = [torch.empty(4, Hkv, page, D, dtype=BF16, device="cuda") for _ in range(2)]
    assert pools[0].numel() * 2 > 1 << 32
    k, v = (seeded((1, Hkv, 100, D), BF16, s).cuda() for s in (2, 3))
    at = torch.tensor([40], dtype=torch.int32, device="cuda")
    far = torch.tensor([[P - 2, 3, P - 1]], dtype=torch.int32, device="cuda")
    near = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    for x in (*pools, *small):
        x[-4:].zero_()
        x[:4].zero_()
    say("append, copy and decode past 4 GiB")
    ffa.fastest_flash_paged_append(k, v, *pools, far, at, inv_freq=freq)
    ffa.fastest_flash_paged_append(k, v, *small, near, at, inv_freq=freq)
    ffa.fastest_flash_copy_pages(*pools, [P - 2, 3], [P - 3, P - 4])
    ffa.fastest_flash_copy_pages(*small, [2], [3])
    for a, b in zip(pools, small):
        assert torch.equal(a[P - 2], b[2]) and torch.equal(a[3], b[0]) and torch.equal(a[P - 1], b[1])
        assert torch.equal(a[P - 3], b[3]) and torch.equal(a[P - 4], b[0])
    lens = torch.tensor([140], dtype=torch.int32, device="cuda")
    x = seeded((1, 16, D), BF16, 4).cuda()
    how = dict(sliding_window=50, sink_tokens=45, max_context_len=140)
    a, _ = ffa.fastest_flash_paged_decode(x, *pools, far, lens, **how)
    b, _ = ffa.fastest_flash_paged_decode(x, *small, near, lens, **how)
    assert torch.equal(a, b) and a.any()


def test_refused_append_changes_nothing():
    """A query or rotation that does not fit is refused before pages are taken."""
    require_gpu()
    say("refused append")
    cache = ffa.PagedKVCache(max_pages=6, page_size=4, num_heads=2, head_dim=16, dtype=torch.bfloat16,
                             device="cuda")
    kv = torch.ones(2, 2, 4, 16, dtype=torch.bfloat16, device="cuda")
    rot = ffa.FastestFlashRotary(16, device="cuda")
    cache.append_batch([0, 1], kv, kv)
    before = {s: (list(q["page_table"]), q["len"]) for s, q in cache.sequences.items()}, list(cache.free_pages)
    for q in (kv.float(), kv[:, :, :3], kv[:1], kv.cpu(), kv[..., :8]):
        with pytest.raises(ValueError, match="does not match"):
            cache.append_batch([0, 5], kv, kv, q=q, rotary=rot)
    with pytest.raises(RuntimeError, match="rotary module is on"):
        cache.append_batch([0, 5], kv, kv, rotary=ffa.FastestFlashRotary(16))
    assert before == ({s: (q["page_table"], q["len"]) for s, q in cache.sequences.items()}, cache.free_pages)
