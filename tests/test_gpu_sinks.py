"""Sliding-window attention with sinks on the GPU against float64: prefill (whole, split, over a
cache), gradients, paged decode, and the modules over a paged cache."""

from __future__ import annotations

import math

import pytest
import torch

import fastest_flash_attention_amd as ffa
from fastest_flash_attention_amd.kernels import _lib
from fastest_flash_attention_amd.ops.attention_forward import launch_prefill, prepare_prefill
from tests import sinks_ref as ref
from tests.gpu_util import require_gpu, say, seeded

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _qkv(B, Hq, Hkv, S, N, D, dt, seed=0):
    return (seeded((B, Hq, S, D), dt, seed).cuda(), seeded((B, Hkv, N, D), dt, seed + 1).cuda(),
            seeded((B, Hkv, N, D), dt, seed + 2).cuda())


def _opt(causal, W, N, cap):
    return (dict(causal=causal, sliding_window=W, sink_tokens=N, softcap=cap),
            dict(causal=causal, window=W, sinks=N, softcap=cap))


FORWARD = [
    # B, Hq, Hkv, S, D, dtype, causal, window, sinks, softcap
    (1, 2, 1, 1, 64, BF16, True, 1, 1, None),
    (1, 2, 1, 2, 64, BF16, True, 1, 1, None),        # row 1: itself and the sink
    (2, 4, 2, 197, 64, FP16, True, 20, 4, None),
    (1, 2, 2, 300, 128, BF16, True, 64, 1, None),
    (1, 2, 2, 300, 128, BF16, True, 64, 33, 30.0),
    (1, 2, 1, 517, 128, FP16, True, 100, 64, None),  # a whole tile of sinks
    (1, 2, 1, 517, 128, BF16, True, 100, 130, None),
    (1, 1, 1, 700, 128, BF16, True, 300, 4, None),   # the window's fast steps
    (1, 1, 1, 700, 128, BF16, True, 333, 200, 20.0),
    (1, 1, 1, 1000, 64, BF16, True, 500, 70, None),  # an odd number of sink tiles ahead of them
    (1, 1, 1, 1000, 64, BF16, True, 500, 70, 25.0),
    (1, 2, 1, 600, 32, FP16, True, 150, 5, None),
    (1, 2, 1, 600, 32, FP16, True, 150, 5, 15.0),
    (1, 1, 1, 400, 192, BF16, True, 130, 40, None),
    (1, 1, 1, 400, 192, FP16, True, 130, 40, 30.0),
    (1, 1, 1, 400, 256, BF16, True, 130, 3, None),
    (1, 1, 1, 400, 256, BF16, True, 130, 3, 30.0),
    (1, 1, 1, 300, 72, BF16, True, 50, 9, None),     # padded head_dim
    (1, 1, 1, 300, 65, FP16, True, 50, 9, None),
    (1, 2, 1, 300, 128, BF16, False, 40, 6, None),   # one-sided window without causal
    (1, 2, 1, 300, 64, BF16, True, 300, 6, None),    # the window reaches every key
    (1, 2, 1, 300, 64, BF16, True, 40, 1000, None),  # every key a sink
    (1, 2, 1, 300, 64, BF16, True, None, 8, None),   # no window: sinks change nothing
    (1, 2, 1, 250, 64, FP32, True, 30, 5, None),
    (1, 2, 1, 250, 128, FP32, True, 70, 40, 20.0),
    (1, 1, 1, 200, 192, FP32, True, 30, 33, None),
    (1, 1, 1, 200, 256, FP32, False, 30, 5, 20.0),
]


@pytest.mark.parametrize("case", FORWARD, ids=[str(i) for i in range(len(FORWARD))])
def test_forward(case):
    require_gpu()
    B, Hq, Hkv, S, D, dt, causal, W, N, cap = case
    q, k, v = _qkv(B, Hq, Hkv, S, S, D, dt)
    ours, theirs = _opt(causal, W, N, cap)
    say(f"sinks forward {case}")
    o, lse = ffa.fastest_flash_attn_forward(q, k, v, num_kv_heads=Hkv, return_lse=True, **ours)
    r = ref.batch(q, k, v, **theirs)
    ref.check(o, r, "o", str(case))
    ref.check(lse, r, "lse", str(case))


PAST = [
    # B, Hq, Hkv, S, Skv, D, dtype, causal, window, sinks, softcap: the last rows' windows lie past
    # the keys, in the tile of the last sinks or behind it
    (1, 2, 1, 418, 5, 64, BF16, True, 7, 8, None),
    (2, 2, 2, 475, 225, 40, FP16, True, 4, 363, None),
    (1, 4, 1, 361, 1, 128, BF16, True, 109, 5, 20.0),
    (1, 2, 1, 431, 195, 136, BF16, True, 33, 226, None),
    (1, 2, 1, 300, 114, 256, FP16, False, 11, 146, None),
    (1, 2, 1, 300, 300, 128, BF16, False, 1, 3, None),
    (1, 2, 1, 500, 130, 128, BF16, True, 30, 129, None),
    (1, 3, 1, 113, 70, 64, FP32, True, 3, 386, 20.0),
    (1, 2, 1, 418, 5, 128, FP32, True, 7, 8, None),
    (1, 2, 1, 150, 20, 192, FP32, True, 7, 8, None),
    (64, 32, 32, 200, 5, 32, FP32, True, 7, 4, None),  # the 128-row fp32 kernel
]


@pytest.mark.parametrize("case", PAST, ids=[str(i) for i in range(len(PAST))])
def test_rows_past_the_keys(case):
    """More rows than keys: rows whose window holds no key see the sinks alone."""
    require_gpu()
    B, Hq, Hkv, S, Skv, D, dt, causal, W, N, cap = case
    q, k, v = _qkv(B, Hq, Hkv, S, Skv, D, dt)
    do = seeded((B, Hq, S, D), dt, 9).cuda()
    ours, theirs = _opt(causal, W, N, cap)
    say(f"sinks past the keys {case}")
    o, lse = ffa.fastest_flash_attn_forward(q, k, v, num_kv_heads=Hkv, return_lse=True, **ours)
    grads = ffa.fastest_flash_attn_backward(do, q, k, v, o, lse, **ours)
    b = slice(B - 1, B)
    r = ref.batch(q[b], k[b], v[b], dout=do[b], **theirs)
    ref.check(o[b], r, "o", str(case))
    ref.check(lse[b], r, "lse", str(case))
    for name, g in zip(("dq", "dk", "dv"), grads):
        ref.check(g[b], r, name, str(case))


def test_large_fp32_grid():
    """The 128-row fp32 kernel (2048 workgroups or more)."""
    require_gpu()
    B, H, S, D = 64, 32, 40, 32
    q, k, v = _qkv(B, H, H, S, S, D, FP32)
    ours, theirs = _opt(True, 5, 3, None)
    say("sinks fp32 grid of 2048")
    o, lse = ffa.fastest_flash_attn_forward(q, k, v, return_lse=True, **ours)
    pick = [0, 17, 63]
    r = ref.batch(q[pick], k[pick], v[pick], **theirs)
    ref.check(o[pick], r, "o", "fp32 grid")
    ref.check(lse[pick], r, "lse", "fp32 grid")


CACHED = [
    # B, Hq, Hkv, Sq, cached, D, dtype, causal, window, sinks, softcap
    (2, 8, 2, 1, 3000, 128, BF16, True, 1000, 4, None),
    (2, 8, 2, 1, 3000, 128, BF16, True, 1000, 200, 30.0),
    (1, 4, 4, 7, 2500, 64, FP16, True, 64, 70, None),
    (1, 4, 1, 130, 1500, 128, BF16, True, 500, 4, None),
    (1, 4, 1, 130, 1500, 128, BF16, True, 2000, 4, None),    # the window reaches every key
    (1, 2, 2, 40, 700, 192, BF16, True, 300, 290, 20.0),     # sinks and window meet
    (1, 2, 2, 40, 700, 256, FP16, True, 300, 500, None),     # sinks inside the window
    (1, 2, 1, 300, 20, 64, BF16, True, 50, 64, None),        # sinks past the cache
    (1, 2, 1, 100, 4096, 64, BF16, True, 16, 513, None),     # sinks in several ranges
    (1, 2, 1, 3, 50, 64, BF16, True, 1, 1, None),
    (1, 2, 1, 300, 2000, 128, BF16, False, 400, 10, None),
    (1, 2, 1, 20, 900, 64, FP32, True, 100, 5, None),        # joined, unseen rows left out
    (2, 64, 64, 140, 900, 128, BF16, True, 64, 4, None),     # too many workgroups to split: joined
]


@pytest.mark.parametrize("case", CACHED, ids=[str(i) for i in range(len(CACHED))])
def test_over_a_cache(case):
    require_gpu()
    B, Hq, Hkv, S, Sc, D, dt, causal, W, N, cap = case
    q, k, v = _qkv(B, Hq, Hkv, S, S, D, dt)
    kc, vc = seeded((B, Hkv, Sc, D), dt, 11).cuda(), seeded((B, Hkv, Sc, D), dt, 12).cuda()
    ours, theirs = _opt(causal, W, N, cap)
    say(f"sinks over a cache {case}")
    o, lse = ffa.fastest_flash_attn_forward(q, k, v, num_kv_heads=Hkv, kv_cache=(kc, vc), return_lse=True,
                                            **ours)
    heads = slice(0, 2) if Hq == 64 else slice(None)
    kv_heads = slice(0, 2) if Hq == 64 else slice(None)
    r = ref.batch(q[:, heads], torch.cat([kc, k], dim=2)[:, kv_heads], torch.cat([vc, v], dim=2)[:, kv_heads],
                  off=Sc, **theirs)
    ref.check(o[:, heads], r, "o", str(case))
    ref.check(lse[:, heads], r, "lse", str(case))


@pytest.mark.parametrize("case", [
    (1, 2, 2, 4500, 64, BF16, 2500, 100, None),
    (1, 2, 1, 4500, 128, BF16, 2500, 4, 30.0),
    (1, 1, 1, 5000, 256, FP16, 3000, 700, None),
], ids=["d64", "d128", "d256"])
def test_split_without_a_cache(case):
    require_gpu()
    B, Hq, Hkv, S, D, dt, W, N, cap = case
    q, k, v = _qkv(B, Hq, Hkv, S, S, D, dt)
    ours, theirs = _opt(True, W, N, cap)
    call = prepare_prefill(q, k, v, num_kv_heads=Hkv, return_lse=True, **ours)
    assert call.args.workspace_bytes > 0  # split
    say(f"sinks split {case}")
    launch_prefill(call)
    r = ref.batch(q, k, v, **theirs)
    ref.check(call.out, r, "o", str(case))
    ref.check(call.lse, r, "lse", str(case))


def test_rows_without_a_key():
    """More queries than keys: the rows before the first key see nothing."""
    require_gpu()
    for dt, D in ((BF16, 64), (BF16, 128), (FP32, 64), (FP16, 256)):
        q, k, v = _qkv(1, 2, 1, 150, 40, D, dt)
        kc, vc = seeded((1, 1, 7, D), dt, 21).cuda(), seeded((1, 1, 7, D), dt, 22).cuda()
        say(f"sinks rows without a key {dt} {D}")
        o, lse = ffa.fastest_flash_attn_forward(q, k, v, causal=True, sliding_window=9, sink_tokens=3,
                                                num_kv_heads=1, kv_cache=(kc, vc), return_lse=True)
        r = ref.batch(q, torch.cat([kc, k], 2), torch.cat([vc, v], 2), off=47 - 150, causal=True, window=9,
                      sinks=3)
        assert torch.isneginf(lse[:, :, :103]).all() and (o[:, :, :103] == 0).all()
        ref.check(o, r, "o", "no key")
        ref.check(lse, r, "lse", "no key")
        # fewer keys than queries, not causal: rows past the window see the sinks alone
        o, lse = ffa.fastest_flash_attn_forward(q, k, v, sliding_window=9, sink_tokens=3, num_kv_heads=1,
                                                return_lse=True)
        r = ref.batch(q, k, v, causal=False, window=9, sinks=3)
        ref.check(o, r, "o", "few keys")
        ref.check(lse, r, "lse", "few keys")


def test_low_scores_keep_their_lse():
    """No floor is added to the softmax sum: rows whose scores are all far below 0."""
    require_gpu()
    q, k, v = _qkv(1, 1, 1, 200, 200, 64, BF16)
    q, k = q.abs() * 6, -k.abs() * 6
    say("sinks low scores")
    o, lse = ffa.fastest_flash_attn_forward(q, k, v, causal=True, sliding_window=30, sink_tokens=4, return_lse=True)
    r = ref.batch(q, k, v, causal=True, window=30, sinks=4)
    assert r["lse"].max() < -69
    # (scores of this size are off by more in fp32: |s| 2^-20)
    ref.check(lse, r, "lse", "low scores", lse_abs=float(r["lse"].abs().max()) * 2.0 ** -16)


def test_strides_and_broadcast():
    require_gpu()
    B, Hq, Hkv, S, D, dt = 2, 4, 2, 210, 64, BF16
    ours, theirs = _opt(True, 40, 6, None)
    q = seeded((B, S, Hq, D), dt, 1).cuda().transpose(1, 2)
    k = seeded((1, S, Hkv, D), dt, 2).cuda().transpose(1, 2)
    v = seeded((1, S, Hkv, D), dt, 3).cuda().transpose(1, 2)
    say("sinks broadcast keys")
    o, lse = ffa.fastest_flash_attn_forward(q, k, v, num_kv_heads=Hkv, return_lse=True, **ours)
    r = ref.batch(q, k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1), **theirs)
    ref.check(o, r, "o", "broadcast")
    say("sinks narrow v")  # padded: no kernels of its own
    q, k, v = _qkv(1, 2, 2, 300, 300, 192, dt)
    o, _ = ffa.fastest_flash_attn_forward(q, k, v[..., :128], **ours)
    r = ref.batch(q, k, torch.nn.functional.pad(v[..., :128], (0, 64)), **theirs)
    ref.check(o, r, "o", "narrow v")


TRAIN = [
    # B, Hq, Hkv, S, D, dtype, causal, window, sinks, softcap
    (1, 2, 1, 1, 64, BF16, True, 1, 1, None),
    (2, 4, 2, 197, 64, FP16, True, 20, 4, None),
    (1, 4, 1, 300, 128, BF16, True, 64, 33, None),
    (1, 2, 2, 517, 128, BF16, True, 100, 130, 30.0),   # two key tiles of sinks
    (1, 8, 1, 700, 64, BF16, True, 50, 5, None),       # parts of the sinks' sweeps
    (1, 8, 2, 900, 128, BF16, True, 40, 1, 20.0),
    (1, 8, 1, 700, 128, FP16, False, 50, 140, None),
    (1, 4, 2, 400, 192, BF16, True, 60, 9, None),
    (1, 8, 1, 500, 192, BF16, True, 30, 9, 25.0),
    (1, 2, 1, 400, 256, BF16, True, 60, 9, None),
    (1, 2, 1, 300, 256, FP16, True, 60, 150, 25.0),
    (1, 2, 1, 200, 80, BF16, True, 30, 5, None),
    (1, 2, 1, 200, 64, BF16, True, 30, 500, None),     # every key a sink
    (1, 2, 1, 200, 64, BF16, True, 200, 5, None),      # the window reaches every key
    (1, 2, 1, 250, 64, FP32, True, 30, 5, None),
    (1, 4, 2, 250, 64, FP32, True, 30, 40, 20.0),
    (1, 2, 1, 200, 128, FP32, True, 30, 5, None),
    (1, 2, 1, 150, 192, FP32, True, 20, 5, None),
    (1, 2, 1, 150, 160, FP32, False, 20, 40, 20.0),
    (4, 16, 16, 220, 64, FP32, True, 20, 5, None),     # two fp32 workgroups per CU
]


@pytest.mark.parametrize("case", TRAIN, ids=[str(i) for i in range(len(TRAIN))])
def test_gradients(case):
    require_gpu()
    B, Hq, Hkv, S, D, dt, causal, W, N, cap = case
    q, k, v = (t.requires_grad_() for t in _qkv(B, Hq, Hkv, S, S, D, dt))
    do = seeded((B, Hq, S, D), dt, 9).cuda()
    ours, theirs = _opt(causal, W, N, cap)
    say(f"sinks gradients {case}")
    out = ffa.fastest_flash_attn_func(q, k, v, num_kv_heads=Hkv, **ours)
    grads = torch.autograd.grad(out, (q, k, v), do)
    b = slice(0, 1)  # the reference of one batch entry
    r = ref.batch(q[b].detach(), k[b].detach(), v[b].detach(), dout=do[b], **theirs)
    ref.check(out[b], r, "o", str(case))
    for name, g in zip(("dq", "dk", "dv"), grads):
        assert g.dtype == dt
        ref.check(g[b], r, name, str(case))
    again = torch.autograd.grad(ffa.fastest_flash_attn_func(q, k, v, num_kv_heads=Hkv, **ours), (q, k, v), do)
    assert all(torch.equal(x, y) for x, y in zip(grads, again))


def test_gradients_by_differences():
    """A directional difference quotient of the float64 reference's own loss against the kernel's
    gradients: what the formula in the reference cannot show."""
    require_gpu()
    B, Hq, Hkv, S, D = 1, 2, 1, 90, 32
    q, k, v = (t.requires_grad_() for t in _qkv(B, Hq, Hkv, S, S, D, FP32))
    do = seeded((B, Hq, S, D), FP32, 9).cuda()
    kw = dict(causal=True, window=11, sinks=3, softcap=20.0)
    say("sinks gradients by differences")
    out = ffa.fastest_flash_attn_func(q, k, v, causal=True, sliding_window=11, sink_tokens=3, softcap=20.0,
                                      num_kv_heads=Hkv)
    grads = torch.autograd.grad(out, (q, k, v), do)
    for i, x in enumerate((q, k, v)):
        d = seeded(x.shape, FP32, 30 + i).double()
        h = 1e-5
        loss = []
        for s in (h, -h):
            args = [t.detach().double().cpu() + (s * d if t is x else 0.0) for t in (q, k, v)]
            loss.append((ref.batch(*args, **kw)["o"] * do.double().cpu()).sum())
        slope = ((loss[0] - loss[1]) / (2 * h)).item()
        got = (grads[i].double().cpu() * d).sum().item()
        # h^2 terms and cancellation: 1e-6 of the loss' scale; the kernel's own error as in the bounds
        size = (grads[i].double().cpu().abs() * d.abs()).sum().item()
        assert abs(slope - got) <= 1e-5 * size, (i, slope, got)


def test_backward_q_offset():
    """Rows of a chunk: gradients for queries at an offset over all keys."""
    require_gpu()
    for D, dt in ((128, BF16), (64, FP32)):
        S, N, off = 70, 400, 330
        q, k, v = _qkv(1, 4, 2, S, N, D, dt)
        do = seeded((1, 4, S, D), dt, 9).cuda()
        kw = dict(causal=True, window=40, sinks=6)
        r = ref.batch(q, k, v, dout=do, off=off, **kw)
        o = r["o"].to(dt).cuda()
        lse = r["lse"].float().cuda()[..., None]
        say(f"sinks backward at an offset {D} {dt}")
        grads = ffa.fastest_flash_attn_backward(do, q, k, v, o, lse, causal=True, sliding_window=40, sink_tokens=6,
                                                q_offset=off)
        for name, g in zip(("dq", "dk", "dv"), grads):
            ref.check(g, r, name, "offset")


@pytest.mark.parametrize("D,dt,N", [(64, BF16, 9), (128, FP16, 9), (128, BF16, 300), (192, BF16, 140),
                                    (256, BF16, 40), (64, FP32, 40), (192, FP32, 9)])
def test_backward_without_room_for_parts(D, dt, N, monkeypatch):
    """With the workspace of the statistics alone no sweep is cut: the same gradients."""
    require_gpu()
    q, k, v = _qkv(1, 4, 1, 700, 700, D, dt)
    do = seeded((1, 4, 700, D), dt, 9).cuda()
    ours, theirs = _opt(True, 60, N, None)
    o, lse = ffa.fastest_flash_attn_forward(q, k, v, num_kv_heads=1, return_lse=True, **ours)
    lib = _lib.load()
    monkeypatch.setattr(lib, "ffa_attn_bwd_split_workspace_bytes", lambda _: 0)
    say(f"sinks backward uncut {D} {dt} {N}")
    grads = ffa.fastest_flash_attn_backward(do, q, k, v, o, lse, **ours)
    r = ref.batch(q, k, v, dout=do, **theirs)
    for name, g in zip(("dq", "dk", "dv"), grads):
        ref.check(g, r, name, "uncut")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,Hq,W", [(1, 2, 1), (31, 1, 7), (33, 1, 7), (65, 3, 40), (96, 5, 60), (450, 7, 333)])
def test_backward_with_two_halves(D, S, Hq, W):
    """Sweeps of one tile, of odd and even numbers of them, over heads of one and more tiles: two
    halves of a workgroup take them in turn, with results that do not change from run to run."""
    require_gpu()
    q, k, v = _qkv(2, Hq, 1, S, S, D, BF16)
    do = seeded((2, Hq, S, D), BF16, 9).cuda()
    ours, theirs = _opt(True, W, 3, None)
    say(f"sinks halves {D} {S} {Hq} {W}")
    o, lse = ffa.fastest_flash_attn_forward(q, k, v, num_kv_heads=1, return_lse=True, **ours)
    grads = ffa.fastest_flash_attn_backward(do, q, k, v, o, lse, **ours)
    again = ffa.fastest_flash_attn_backward(do, q, k, v, o, lse, **ours)
    r = ref.batch(q, k, v, dout=do, **theirs)
    for name, g, h in zip(("dq", "dk", "dv"), grads, again):
        ref.check(g, r, name, "halves")
        assert torch.equal(g, h)


def _paged(lens, page, Hkv, D, dt, spare=3, seed=0):
    need = [-(-n // page) for n in lens]
    P = sum(need) + spare
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(P, generator=g)
    bt = torch.zeros(len(lens), max(need + [1]), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        bt[b, :n] = order[at:at + n].to(torch.int32)
        at += n
    kp, vp = seeded((P, Hkv, page, D), dt, seed + 1).cuda(), seeded((P, Hkv, page, D), dt, seed + 2).cuda()
    return kp, vp, bt.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()


def _rows(pool, bt, b, n, page):
    ids = bt[b, :-(-n // page)].long()
    return pool[ids].transpose(0, 1).flatten(1, 2)[:, :n]


DECODE = [
    # lens, page, Hq, Hkv, D, dtype, window, sinks, softcap, tokens_per_split
    ((1, 2, 5, 17, 300), 16, 4, 2, 128, BF16, 8, 1, None, None),
    ((700, 33, 64, 65, 0), 16, 8, 2, 128, BF16, 64, 4, None, 32),
    ((700, 333, 1000), 7, 8, 1, 64, FP16, 100, 33, 20.0, 48),
    ((700, 333, 1000), 1, 8, 1, 64, FP16, 100, 64, None, 64),
    ((5000, 4200, 30), 64, 8, 8, 128, BF16, 2047, 130, None, 2048),
    ((5000, 4200, 30), 1, 8, 8, 64, BF16, 2100, 1000, None, 2048),   # splits across the gap
    ((2000, 100), 128, 20, 1, 32, BF16, 500, 200, None, None),
    ((900, 20), 16, 4, 4, 192, FP16, 50, 20, 30.0, None),
    ((900, 20), 16, 4, 4, 256, BF16, 50, 20, None, None),
    ((900, 20), 16, 4, 4, 72, BF16, 10 ** 6, 20, None, None),        # the window reaches every token
    ((900, 20), 16, 4, 4, 64, BF16, 30, 10 ** 6, None, None),        # every token a sink
    ((300, 20, 1), 16, 4, 2, 64, FP32, 30, 5, None, None),
]


@pytest.mark.parametrize("case", DECODE, ids=[str(i) for i in range(len(DECODE))])
def test_decode(case):
    require_gpu()
    lens, page, Hq, Hkv, D, dt, W, N, cap, tps = case
    kp, vp, bt, ln = _paged(lens, page, Hkv, D, dt)
    q = seeded((len(lens), Hq, D), dt, 5).cuda()
    say(f"sinks decode {case}")
    o, lse = ffa.fastest_flash_paged_decode(q, kp, vp, bt, ln, sliding_window=W, sink_tokens=N, softcap=cap,
                                            return_lse=True, tokens_per_split=tps)
    for b, n in enumerate(lens):
        if n == 0:
            assert (o[b] == 0).all() and torch.isneginf(lse[b]).all()
            continue
        r = ref.batch(q[b:b + 1, :, None], _rows(kp, bt, b, n, page)[None], _rows(vp, bt, b, n, page)[None],
                      off=n - 1, causal=True, window=W, sinks=N, softcap=cap)
        ref.check(o[b:b + 1, :, None], r, "o", f"{case} {b}")
        ref.check(lse[b:b + 1, :, None], r, "lse", f"{case} {b}")


def test_decode_reads_seen_pages_only():
    """Table entries between the sinks and the window may be anything; one among those seen takes
    its tokens out."""
    require_gpu()
    page, lens, W, N = 16, (500, 260), 100, 20
    kp, vp, bt, ln = _paged(lens, page, 2, 64, BF16)
    q = seeded((2, 4, 64), BF16, 5).cuda()
    kw = dict(sliding_window=W, sink_tokens=N, return_lse=True)
    want = ffa.fastest_flash_paged_decode(q, kp, vp, bt, ln, **kw)
    bad = bt.clone()
    bad[0, 2:25] = torch.tensor([-1, 10 ** 6] * 12, dtype=torch.int32)[:23].cuda()  # tokens 32 .. 399
    bad[1, 2:10] = -7
    say("sinks decode with foreign table entries behind the window")
    got = ffa.fastest_flash_paged_decode(q, kp, vp, bad, ln, check_block_tables=True, **kw)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    bad[0, 1] = -1  # tokens 16 .. 19 of the sinks
    got = ffa.fastest_flash_paged_decode(q, kp, vp, bad, ln, **kw)
    less = ffa.fastest_flash_paged_decode(q, kp, vp, bt, ln, sliding_window=W, sink_tokens=16, return_lse=True)
    assert torch.equal(got[0][1], want[0][1])
    assert (got[1][0] - less[1][0]).abs().max() < 1e-4 and (got[0][0] - less[0][0]).abs().max() < 2.0 ** -7
    with pytest.raises(IndexError):
        ffa.fastest_flash_paged_decode(q, kp, vp, bad, ln, check_block_tables=True, **kw)


def test_graph_replays():
    require_gpu()
    q, k, v = _qkv(1, 4, 2, 300, 300, 128, BF16)
    kw = dict(causal=True, sliding_window=64, sink_tokens=5, num_kv_heads=2, return_lse=True)
    kp, vp, bt, ln = _paged((300, 90), 16, 2, 128, BF16)
    qd = seeded((2, 4, 128), BF16, 5).cuda()
    dec = dict(sliding_window=64, sink_tokens=5, return_lse=True, max_context_len=300)

    def calls():
        return (*ffa.fastest_flash_attn_forward(q, k, v, **kw),
                *ffa.fastest_flash_paged_decode(qd, kp, vp, bt, ln, **dec))

    say("sinks capture")
    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = calls()
    for rep in range(3):
        for t, s in ((q, 50), (k, 60), (v, 70), (qd, 80), (kp, 90)):
            t.copy_(seeded(t.shape, BF16, s + rep))
        ln.copy_(torch.tensor([300 - 7 * rep, 10 + rep], dtype=torch.int32))
        for t in outs:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        assert all(torch.equal(x, y) for x, y in zip(got, calls())), f"replay {rep}"


def test_backward_in_a_graph():
    require_gpu()
    q, k, v = _qkv(1, 8, 1, 700, 700, 64, BF16)
    do = seeded((1, 8, 700, 64), BF16, 9).cuda()
    kw = dict(causal=True, sliding_window=50, sink_tokens=5)

    def calls():
        o, lse = ffa.fastest_flash_attn_forward(q, k, v, num_kv_heads=1, return_lse=True, **kw)
        return ffa.fastest_flash_attn_backward(do, q, k, v, o, lse, **kw)

    say("sinks backward capture")
    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = calls()
    for rep in range(3):
        for t, s in ((q, 50), (k, 60), (v, 70), (do, 80)):
            t.copy_(seeded(t.shape, BF16, s + rep))
        for t in outs:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        assert all(torch.equal(x, y) for x, y in zip(got, calls())), f"replay {rep}"


def test_refusals():
    require_gpu()
    q, k, v = _qkv(1, 2, 2, 64, 64, 64, BF16)
    with pytest.raises(ValueError, match="sink_tokens"):
        ffa.fastest_flash_attn_forward(q, k, v, sliding_window=8, sink_tokens=-1)
    with pytest.raises(ValueError, match="block_mask"):
        ffa.fastest_flash_attn_forward(q, k, v, sliding_window=8, sink_tokens=2, block_size=64,
                                       block_mask=torch.ones(1, 1, dtype=torch.bool))
    with pytest.raises(ValueError, match="sink_tokens"):
        ffa.fastest_flash_attn_backward(q, q, k, v, q, torch.zeros(1, 2, 64, 1).cuda(), sliding_window=8,
                                        sink_tokens=-1)
    kp, vp, bt, ln = _paged((30,), 16, 2, 64, BF16)
    with pytest.raises(ValueError, match="sink_tokens"):
        ffa.fastest_flash_paged_decode(q[:, :, 0], kp, vp, bt, ln, sliding_window=8, sink_tokens=-1)


@pytest.mark.parametrize("kind,dt", [("gqa", FP32), ("mha", FP32), ("gqa", FP16), ("gqa", BF16)])
def test_module_prompt_fork_decode_evict(kind, dt):
    """The operators together, as a serving loop uses them: prompts enter a paged cache (rotated),
    sequences fork, decode step by step over a window with sinks, pages behind the window are
    released and the pool is compacted; every step equals the module's forward of the whole
    sequence at its last position."""
    require_gpu()
    torch.manual_seed(0)
    hidden, heads, page, W, N = 256, 4, 8, 24, 5
    rot = ffa.FastestFlashRotary(32, interleaved=kind == "mha", scaling="ntk", factor=2.0)
    if kind == "gqa":
        m = ffa.FastestFlashGQA(hidden, heads, 2, causal=True, sliding_window=W, rotary=rot, sink_tokens=N)
    else:
        m = ffa.FastestFlashMHA(hidden, heads, causal=True, sliding_window=W, rotary=rot, sink_tokens=N)
    m = m.to("cuda", dt).eval()
    assert rot.inv_freq.is_cuda and rot.inv_freq.dtype == torch.float64
    x = seeded((2, 60, hidden), dt, 1).cuda()
    cache = m.new_paged_cache(max_pages=40, page_size=page)
    say(f"module over a paged cache {kind} {dt}")
    with torch.no_grad():
        y = m.prefill_with_cache(x[:, :37], cache, [0, 1])
        assert torch.equal(y, m(x[:, :37]))
        cache.fork_sequence(0, 2)
        have = [x[0, :37], x[1, :37], x[0, :37]]
        for step in range(14):
            new = torch.stack([x[0, 37 + step], x[1, 37 + step], x[1, 20 + step]])[:, None]
            got = m.decode_step(new, cache, [0, 1, 2], evict=step % 2 == 1)
            if step == 6:
                cache.compact()
            have = [torch.cat([h, n]) for h, n in zip(have, new)]
            want = torch.cat([m(h[None])[:, -1:] for h in have])
            # each of the two ways is within its type's rounding of the projections, of P and O:
            # some steps of eps / 2 of the largest output each (fp32: sums of other orders)
            lim = {FP32: 2.0 ** -18, FP16: 2.0 ** -8, BF16: 2.0 ** -5}[dt] * want.abs().max()
            off = (got - want).abs().max()
            assert off <= lim, f"step {step}: {off:.2e} over {lim:.2e}"
        assert any(-1 in cache.sequences[s]["page_table"] for s in (0, 1, 2))
        with pytest.raises(ValueError, match="evicted"):
            cache.get_kv(0)
        for s in (0, 1, 2):
            cache.free_sequence(s)
        assert cache.num_free_pages == 40


def test_module_trains():
    """Rotary and sinks under autograd in the module: gradients equal those of the float64 formula
    chained by hand through the fp32 projections."""
    require_gpu()
    torch.manual_seed(1)
    m = ffa.FastestFlashGQA(64, 4, 2, causal=True, sliding_window=9, sink_tokens=2,
                            rotary=ffa.FastestFlashRotary(16)).cuda().train()
    x = seeded((1, 40, 64), FP32, 3).cuda().requires_grad_()
    do = seeded((1, 40, 64), FP32, 4).cuda()
    say("module with rotary and sinks trains")
    names = [n for n, _ in m.named_parameters()]
    grads = torch.autograd.grad(m(x), [x, *m.parameters()], do)
    w = {n: p.detach().double().cpu().requires_grad_() for n, p in m.named_parameters()}
    x64 = x.detach().double().cpu().requires_grad_()
    q, k, v = (torch.nn.functional.linear(x64, w[f"{n}_proj.weight"]).view(1, 40, -1, 16).transpose(1, 2)
               for n in "qkv")
    ang = torch.arange(40).double()[:, None] * m.rotary.inv_freq.cpu()
    cos, sin = ang.cos(), ang.sin()

    def turn(t):
        a, b = t[..., :8], t[..., 8:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)

    q, k, v = turn(q), turn(k).repeat_interleave(2, 1), v.repeat_interleave(2, 1)
    s = (q @ k.transpose(2, 3)) / 4.0
    ok = ref.visible(torch.arange(40), torch.arange(40), True, 9, 2)
    p = torch.softmax(s.masked_fill(~ok, float("-inf")), dim=-1)
    y = torch.nn.functional.linear((p @ v).transpose(1, 2).reshape(1, 40, 64), w["o_proj.weight"])
    want = torch.autograd.grad(y, [x64, *w.values()], do.double().cpu())
    for n, g, r in zip(["x", *names], grads, want):
        assert (g.double().cpu() - r).abs().max() <= 2.0 ** -16 * r.abs().max(), n
