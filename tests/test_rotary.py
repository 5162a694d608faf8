"""Rotary frequencies, the rotary module and the refusals of the rotary and batched append entry
points (CPU, no GPU needed)."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import fastest_flash_attention_amd as ffa
from fastest_flash_attention_amd.kernels import _lib
from tests.test_host import _c_layout


def test_plain_frequencies():
    f = ffa.rotary_frequencies(64, 10000.0)
    assert f.dtype == torch.float64 and f.shape == (32,)
    for i in range(32):
        assert math.isclose(f[i].item(), 10000.0 ** (-2 * i / 64), rel_tol=1e-14)


def test_scaled_frequencies():
    plain = ffa.rotary_frequencies(64)
    assert torch.allclose(ffa.rotary_frequencies(64, scaling="linear", factor=4.0), plain / 4, rtol=1e-15)
    ntk = ffa.rotary_frequencies(64, scaling="ntk", factor=8.0)
    assert ntk[0] == 1.0 and math.isclose(ntk[-1].item(), plain[-1].item() / 8, rel_tol=1e-12)
    assert torch.all(ntk <= plain)
    assert torch.equal(ffa.rotary_frequencies(2, scaling="ntk", factor=8.0), torch.tensor([0.125]).double())
    yarn = ffa.rotary_frequencies(64, scaling="yarn", factor=16.0, original_max_position=4096)
    turns = 4096 * plain / (2 * math.pi)
    fast, slow = turns > 40, turns < 0.8  # past the ramp's ends, rounded out by up to a pair
    assert fast.any() and slow.any()
    assert torch.equal(yarn[fast], plain[fast])
    assert torch.allclose(yarn[slow], plain[slow] / 16, rtol=1e-14)
    ratio = plain / yarn
    assert torch.all(ratio[1:] >= ratio[:-1] - 1e-12)
    assert math.isclose(ffa.yarn_magnitude(16.0), 0.1 * math.log(16.0) + 1.0)
    assert ffa.yarn_magnitude(1.0) == ffa.yarn_magnitude(0.5) == 1.0


@pytest.mark.parametrize("args,kwargs", [
    ((7,), {}), ((0,), {}), ((64, -1.0), {}), ((64,), dict(scaling="cubic", factor=2.0)),
    ((64,), dict(factor=2.0)), ((64,), dict(scaling="linear", factor=0.0)),
    ((64,), dict(scaling="yarn", factor=2.0)),
    ((64,), dict(scaling="yarn", factor=2.0, original_max_position=10, beta_fast=1.0)),
    ((64, 1.0), dict(scaling="yarn", factor=2.0, original_max_position=10)),
])
def test_frequency_refusals(args, kwargs):
    with pytest.raises(ValueError):
        ffa.rotary_frequencies(*args, **kwargs)


def test_module_keeps_64_bits():
    m = ffa.FastestFlashRotary(32, scaling="yarn", factor=4.0, original_max_position=2048)
    want = m.inv_freq.clone()
    gqa = ffa.FastestFlashGQA(64, 4, 2, head_dim=32, rotary=m).to(torch.bfloat16)
    assert gqa.rotary is m and m.inv_freq.dtype == torch.float64 and torch.equal(m.inv_freq, want)
    assert not any("rotary" in k for k in gqa.state_dict())
    assert m.magnitude == ffa.yarn_magnitude(4.0)
    m.to("meta")
    assert m.inv_freq.device.type == "meta" and m.inv_freq.dtype == torch.float64


def test_module_made_without_memory():
    """Made on the meta device, the frequencies are there once the module has memory."""
    with torch.device("meta"):
        m = ffa.FastestFlashRotary(32, scaling="linear", factor=4.0)
    assert m.inv_freq.is_meta
    m.to_empty(device="cpu")
    assert torch.equal(m.inv_freq, ffa.rotary_frequencies(32, scaling="linear", factor=4.0))


def test_entry_points_refuse_host_tensors():
    q = torch.zeros(1, 2, 3, 8)
    f = ffa.rotary_frequencies(8)
    with pytest.raises(RuntimeError, match="ROCm"):
        ffa.fastest_flash_rotary(q, q, f)
    with pytest.raises(ValueError):
        ffa.fastest_flash_rotary(q, q[:, :, :2], f)
    with pytest.raises(ValueError):
        ffa.fastest_flash_rotary(q[0], q, f)
    with pytest.raises(TypeError):
        ffa.fastest_flash_rotary(q, q.half(), f)
    pool = torch.zeros(4, 2, 4, 8)
    bt, at = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="ROCm"):
        ffa.fastest_flash_paged_append(q, q, pool, pool, bt, at)
    with pytest.raises(ValueError, match="inv_freq"):
        ffa.fastest_flash_paged_append(q, q, pool, pool, bt, at, q=q)
    with pytest.raises(TypeError, match="int32"):
        ffa.fastest_flash_paged_append(q, q, pool, pool, bt.long(), at)
    with pytest.raises(ValueError, match="pools"):
        ffa.fastest_flash_paged_append(q[:, :1], q[:, :1], pool, pool, bt, at)


@pytest.mark.parametrize("cls,cname", [
    (_lib.RotaryArgs, "ffa_rotary_args"),
    (_lib.PagedAppendBatchArgs, "ffa_paged_append_batch_args"),
    (_lib.PagedCopyArgs, "ffa_paged_copy_args"),
])
def test_ctypes_struct_matches_header(cls, cname):
    fields = [f for f, _ in cls._fields_]
    c = _c_layout(cname, fields)
    assert c["sizeof"] == ctypes.sizeof(cls)
    for f in fields:
        assert c[f] == getattr(cls, f).offset, f


# ---------------------------------------------------------------------------------
# Refusals of the C entry points: before any HIP call, so they run here
# ---------------------------------------------------------------------------------

BAD, DTYPE, ALIGN = -1, -2, -4


def _rotary_args(**over):
    a = _lib.RotaryArgs()
    a.q = a.k = a.q_out = a.k_out = a.inv_freq = 0x1000
    for st in (a.q_stride, a.k_stride, a.q_out_stride, a.k_out_stride):
        st[:] = [64, 32, 8]
    a.batch, a.heads_q, a.heads_k, a.seqlen, a.head_dim, a.rotary_dim = 1, 2, 2, 4, 8, 8
    a.magnitude = 1.0
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,rc", [
    (dict(dtype=3), DTYPE), (dict(batch=-1), BAD), (dict(heads_q=-1), BAD), (dict(seqlen=-1), BAD),
    (dict(rotary_dim=7), BAD), (dict(rotary_dim=10), BAD), (dict(rotary_dim=0), BAD),
    (dict(magnitude=math.inf), BAD), (dict(q=None), BAD), (dict(k_out=None), BAD),
    (dict(inv_freq=None), BAD), (dict(inv_freq=0x1004), ALIGN), (dict(q=0x1001), ALIGN),
    (dict(k=0x1002, dtype=2), ALIGN), (dict(positions=0x1000, position_bytes=2), BAD),
    (dict(positions=0x1004, position_bytes=8), ALIGN), (dict(batch=0, q=None), 0),
])
def test_rotary_abi_refusals(over, rc):
    assert _lib.load().ffa_rotary(ctypes.byref(_rotary_args(**over)), None) == rc


def _append_args(**over):
    a = _lib.PagedAppendBatchArgs()
    a.k_pages = a.v_pages = a.k_new = a.v_new = a.q = a.q_out = 0x1000
    a.inv_freq = a.block_tables = a.positions = 0x1000
    for st in (a.k_new_stride, a.v_new_stride, a.q_stride, a.q_out_stride):
        st[:] = [64, 32, 8]
    a.block_table_stride, a.batch, a.heads_q, a.heads_kv, a.n_tokens = 4, 1, 2, 2, 1
    a.head_dim, a.rotary_dim, a.page_size, a.num_pages, a.magnitude = 8, 8, 4, 4, 1.0
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,rc", [
    (dict(dtype=5), DTYPE), (dict(heads_kv=0), BAD), (dict(n_tokens=-1), BAD), (dict(page_size=0), BAD),
    (dict(rotary_dim=3), BAD), (dict(k_pages=None), BAD), (dict(v_new=None), BAD),
    (dict(block_tables=None), BAD), (dict(positions=None), BAD), (dict(inv_freq=None), BAD),
    (dict(q_out=None), BAD), (dict(positions=0x1002), ALIGN), (dict(counts=0x1001), ALIGN),
    (dict(v_pages=0x1001), ALIGN), (dict(magnitude=math.nan), BAD), (dict(n_tokens=0, k_new=None), 0),
])
def test_append_abi_refusals(over, rc):
    assert _lib.load().ffa_paged_append_batch(ctypes.byref(_append_args(**over)), None) == rc


@pytest.mark.parametrize("over,rc", [
    (dict(n_pairs=-1), BAD), (dict(k_pages=None), BAD), (dict(src=None), BAD), (dict(page_bytes=33), ALIGN),
    (dict(dst=0x1002), ALIGN), (dict(n_pairs=0, k_pages=None), 0), (dict(page_bytes=0), 0),
])
def test_copy_abi_refusals(over, rc):
    a = _lib.PagedCopyArgs()
    a.k_pages = a.v_pages = a.src = a.dst = 0x1000
    a.page_bytes, a.n_pairs, a.num_pages = 64, 2, 8
    for k, v in over.items():
        setattr(a, k, v)
    assert _lib.load().ffa_paged_copy(ctypes.byref(a), None) == rc
