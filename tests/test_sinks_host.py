"""Host side of attention with sinks (CPU): argument resolution, what of a cache is joined, the C
entry points' refusals and workspace sizes, and the cuts of the backward's sweeps."""

from __future__ import annotations

import ctypes
import inspect

import pytest
import torch

import fastest_flash_attention_amd as ffa
from fastest_flash_attention_amd.kernels import _lib
from fastest_flash_attention_amd.ops import attention_forward as af
from tests import sinks_ref as ref

BAD, HEAD_DIM = -1, -3


def _resolve(S=4, Sc=0, H=2, D=8, **kw):
    q, k, v = (torch.randn(1, H, S, D, generator=torch.Generator().manual_seed(i)) for i in range(3))
    cache = None
    if Sc:
        cache = tuple(torch.randn(1, H, Sc, D, generator=torch.Generator().manual_seed(i)) for i in (8, 9))
    return af.resolve_forward_args(q, k, v, kv_cache=cache, **kw), (q, k, v), cache


def test_sinks_need_a_window():
    assert _resolve(sink_tokens=3)[0].sink_tokens == 0
    assert _resolve(sink_tokens=3, sliding_window=2)[0].sink_tokens == 3
    cfg = ffa.AttentionConfig(causal=True, sliding_window=2, sink_tokens=5)
    assert _resolve(config=cfg)[0].sink_tokens == 5
    assert ffa.AttentionConfig().sink_tokens == 0
    with pytest.raises(ValueError, match="negative"):
        _resolve(sink_tokens=-1)
    with pytest.raises(ValueError, match="block_mask"):
        _resolve(sliding_window=2, sink_tokens=1, block_mask=torch.ones(1, 1, dtype=torch.bool))
    _resolve(sliding_window=2, block_mask=torch.ones(1, 1, dtype=torch.bool))


def test_new_arguments_come_last():
    """Calls by position mean what they did."""
    last = {ffa.fastest_flash_attn_func: "sink_tokens", ffa.fastest_flash_attn_forward: "sink_tokens",
            ffa.fastest_flash_attn_backward: "sink_tokens", ffa.fastest_flash_paged_decode: "sink_tokens",
            ffa.FastestFlashGQA.__init__: "sink_tokens", ffa.FastestFlashMHA.__init__: "sink_tokens",
            ffa.AttentionConfig.__init__: "sink_tokens"}
    for fn, name in last.items():
        p = list(inspect.signature(fn).parameters.values())[-1]
        assert p.name == name and p.default == 0, fn


@pytest.mark.parametrize("S,Sc,W,N", [(4, 30, 6, 3), (1, 30, 6, 3), (4, 30, 40, 3), (4, 30, 6, 50),
                                      (4, 5, 1, 2), (9, 30, 1, 29), (9, 30, 1, 30)])
@pytest.mark.parametrize("causal", [True, False])
def test_joined_cache_leaves_unseen_rows_out(S, Sc, W, N, causal):
    """The shorter keys at the smaller offset: the same visible keys, in the same order, for every
    row, whichever way the cache is joined."""
    for in_place in (False, True):
        r, (q, k, v), (kc, vc) = _resolve(S, Sc, sliding_window=W, sink_tokens=N, causal=causal,
                                          cache_in_place=in_place)
        if in_place:
            assert r.cache is not None and r.S_kv == S + Sc
            af._join_cache(r)
        whole = torch.cat([kc, k], dim=2)
        low = Sc - W + 1
        dropped = max(0, min(low, Sc) - N)
        assert r.k.size(2) == r.v.size(2) == r.S_kv == S + Sc - dropped and r.q_offset == Sc - dropped
        ok = ref.visible(torch.arange(Sc, Sc + S), torch.arange(Sc + S), causal, W, N)
        short = ref.visible(r.q_offset + torch.arange(S), torch.arange(r.S_kv), causal, W, N)
        for i in range(S):
            assert torch.equal(whole[0, 0, ok[i]], r.k[0, 0, short[i]])


def test_without_sinks_caches_join_whole():
    r, (q, k, v), (kc, vc) = _resolve(4, 30, sliding_window=6)
    assert torch.equal(r.k, torch.cat([kc, k], dim=2)) and r.q_offset == 30


def _prefill_args(**over):
    a = _lib.PrefillArgs()
    a.q = a.k = a.v = a.o = 0x1000
    for st in (a.q_stride, a.k_stride, a.v_stride, a.o_stride):
        st[:] = [4096, 1024, 64, 1]
    a.batch, a.heads_q, a.heads_kv, a.seqlen_q, a.seqlen_kv, a.head_dim = 1, 2, 2, 16, 16, 64
    a.window, a.sinks, a.scale, a.causal = 4, 2, 0.125, 1
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,rc", [
    (dict(sinks=-1), BAD),
    (dict(block_key_mask=0x1000, block_visited=0x1000, block_key_mask_words=1, ref_block_q=64), BAD),
    (dict(head_dim=192, v_head_dim=128), HEAD_DIM),
])
def test_prefill_abi_refusals(over, rc):
    assert _lib.load().ffa_prefill_fwd(ctypes.byref(_prefill_args(**over)), None) == rc


def test_prefill_workspace_counts_the_sinks_range():
    """A split call with sinks has one range more; sinks in both segments are not split."""
    size = lambda **over: _lib.load().ffa_prefill_workspace_bytes(ctypes.byref(_prefill_args(**over)))  # noqa: E731
    call = dict(seqlen_q=1, seqlen_kv=5000, q_offset=4999, window=2048, k_cache=0x1000, v_cache=0x1000,
                cache_len=4999)
    row = 2 * 65 * 4  # two heads' partial of one range
    assert size(**call, sinks=4) == size(**call, sinks=0) + row
    assert size(**call, sinks=4999) >= size(**call, sinks=0) + row
    assert size(**call, sinks=5000) == 0
    assert size(**dict(call, window=5000), sinks=4) == size(**dict(call, window=5000), sinks=0)
    assert size(**call, sinks=-1) == 0


def test_decode_and_backward_abi_refusals():
    lib = _lib.load()
    a = _lib.PagedDecodeArgs()
    a.q = a.k_pages = a.v_pages = a.o = a.block_tables = a.context_lens = 0x1000
    a.q_stride[:] = a.o_stride[:] = a.lse_stride[:] = [128, 64]
    a.block_table_stride, a.batch, a.heads_q, a.heads_kv, a.head_dim = 64, 1, 2, 2, 64
    a.page_size, a.num_pages, a.max_context_len, a.scale = 16, 64, 1000, 0.125
    a.window, a.sinks = 100, -1
    assert lib.ffa_paged_decode_fwd(ctypes.byref(a), None) == BAD
    a.sinks = 4  # the workspace of window + sinks tokens would do; none is given
    assert lib.ffa_paged_decode_fwd(ctypes.byref(a), None) == -6
    b = _lib.AttnBwdArgs()
    for name in ("dout", "q", "k", "v", "o", "lse", "dq", "dk", "dv", "workspace"):
        setattr(b, name, 0x1000)
    for st in (b.do_stride, b.q_stride, b.k_stride, b.v_stride, b.o_stride, b.dq_stride, b.dk_stride, b.dv_stride):
        st[:] = [4096, 1024, 64, 1]
    b.batch, b.heads_q, b.heads_kv, b.seqlen_q, b.seqlen_kv, b.head_dim, b.scale = 1, 2, 2, 16, 16, 64, 0.125
    b.window, b.sinks = 4, -1
    assert lib.ffa_attn_bwd(ctypes.byref(b), None) == BAD
    assert lib.ffa_attn_bwd_split_workspace_bytes(ctypes.byref(b)) == 0
    b.sinks, b.head_dim, b.v_head_dim = 2, 192, 128
    assert lib.ffa_attn_bwd(ctypes.byref(b), None) == HEAD_DIM


def _bwd_bytes(B, Hq, Hkv, S, D, window, sinks, off=0, dtype=0):
    a = _lib.AttnBwdArgs()
    a.batch, a.heads_q, a.heads_kv, a.seqlen_q, a.seqlen_kv, a.head_dim = B, Hq, Hkv, S, S + off, D
    a.window, a.sinks, a.q_offset, a.causal, a.dtype = window, sinks, off, 1, dtype
    lib = _lib.load()
    return (lib.ffa_attn_bwd_split_workspace_bytes(ctypes.byref(a))
            - lib.ffa_attn_bwd_workspace_bytes(B, Hq, S))


@pytest.mark.parametrize("D,dtype", [(128, 0), (256, 0), (64, 2)])
def test_backward_cuts_the_sinks_rows(D, dtype):
    """The rows of 32-key blocks of sinks go over the chip: whole parts per block and KV head."""
    block = 32 * 2 * D * 4
    got = _bwd_bytes(1, 32, 8, 8192, D, 1024, 4, dtype=dtype)
    assert got == 256 * block  # 8 KV heads, one block each: 32 parts
    assert _bwd_bytes(1, 32, 8, 8192, D, 1024, 40, dtype=dtype) == 256 * block  # two blocks: 16 parts
    assert _bwd_bytes(1, 32, 8, 8192, D, 1024, 0, dtype=dtype) == 0
    assert _bwd_bytes(32, 32, 8, 8192, D, 1024, 4, dtype=dtype) == 0  # blocks enough without
    assert _bwd_bytes(1, 8, 8, 200, D, 64, 4, dtype=dtype) == 0       # seven row tiles a block


def test_backward_cuts_the_sinks_tiles():
    """Sweeps of whole 128-key tiles of sinks are cut from 1.5 parts on."""
    tile = 128 * 2 * 128 * 4
    got = _bwd_bytes(1, 16, 16, 4096, 128, 500, 1024)
    assert got == 16 * 8 * 2 * tile
    assert _bwd_bytes(1, 32, 8, 8192, 256, 1024, 128) == 32 * 8 * 32 * 2 * 256 * 4  # blocks past head_dim 192


@pytest.mark.parametrize("seed", range(40))
def test_backward_workspace_is_bounded(seed):
    """At most 180 MB over the statistics, whatever the sizes (include/ffa.h)."""
    g = torch.Generator().manual_seed(seed)
    pick = lambda lo, hi: int(torch.randint(lo, hi, (1,), generator=g))  # noqa: E731
    for _ in range(50):
        Hkv = 1 << pick(0, 6)
        S = 1 << pick(5, 18)
        got = _bwd_bytes(pick(1, 9), Hkv << pick(0, 4), Hkv, S + pick(0, 100), [64, 128, 192][pick(0, 3)],
                         1 << pick(0, 14), 1 << pick(0, 14), off=pick(0, 2) * pick(0, 1 << 15))
        assert 0 <= got <= 180 << 20, got
