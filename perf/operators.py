"""Long-context operators, each in a plain form and through its public entry point.

A case is a dict of plain values; its ``kind`` names the operator:

- ``forward``  attention over a sliding window and a few first tokens that stay visible (sinks);
               with ``Sc`` the queries are a chunk over ``Sc`` cached tokens
- ``train``    the same with its gradients
- ``decode``   the same for one token per sequence over a paged cache
- ``rotary``   rotary positions of queries and keys; with ``grad`` also their gradients
- ``append``   new tokens' keys rotated and written with the values into a paged cache, their
               queries rotated on the way
- ``copy``     pages of a paged cache copied onto others (forked sequences, compaction)

``listed`` holds the fixed cases, ``draw`` makes more of the same ranges. ``run`` computes the
operators from elementary operations, or, with ``own`` set, calls the framework.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # One short chat prompt on a small GQA model: launch and latency bound.
        dict(name="sinks_prompt_short", kind="forward", B=1, Hq=8, Hkv=2, S=197, Sc=0, D=64,
             dtype="fp16", causal=True, window=64, sinks=4, softcap=0.0),
        # A long document read by a GQA model whose layers see a window and four sinks.
        dict(name="sinks_prompt_long", kind="forward", B=1, Hq=32, Hkv=8, S=8192, Sc=0, D=128,
             dtype="bf16", causal=True, window=4096, sinks=4, softcap=0.0),
        # A training step's attention on a GQA model, ragged length.
        dict(name="sinks_train_gqa", kind="train", B=2, Hq=32, Hkv=8, S=2011, D=128, dtype="bf16",
             causal=True, window=512, sinks=4, softcap=0.0),
        # Training a small model in fp32.
        dict(name="sinks_train_fp32", kind="train", B=2, Hq=8, Hkv=8, S=1024, D=64, dtype="fp32",
             causal=True, window=200, sinks=16, softcap=0.0),
        # Serving: a decode step of a large batch with mixed context lengths.
        dict(name="sinks_decode_batch", kind="decode", B=64, Hq=32, Hkv=8, D=128, page=16, lo=512,
             hi=32768, dtype="bf16", window=4096, sinks=4, softcap=0.0),
        # Serving a few users with long contexts: few sequences, latency bound.
        dict(name="sinks_decode_few", kind="decode", B=4, Hq=32, Hkv=8, D=128, page=64, lo=3000,
             hi=20000, dtype="fp16", window=1024, sinks=16, softcap=30.0),
        # The queries and keys of a batch of prompts, out of their projections.
        dict(name="rotary_prompts", kind="rotary", B=2, Hq=32, Hkv=8, S=4096, D=128, R=128,
             dtype="bf16", interleaved=False, factor=1.0, offset=0, packed=False, grad=False),
        # Training with half of each head rotated, pairs interleaved, documents packed into rows.
        dict(name="rotary_train_partial", kind="rotary", B=4, Hq=16, Hkv=16, S=1023, D=96, R=48,
             dtype="fp16", interleaved=True, factor=4.0, offset=0, packed=True, grad=True),
        # Serving: the new tokens of a large batch enter the cache.
        dict(name="append_batch", kind="append", B=64, Hq=32, Hkv=8, n=1, D=128, R=128, page=16,
             hi=1024, dtype="bf16", interleaved=False, factor=8.0),
        # Two requests of equal length are admitted: their prompts enter the cache.
        dict(name="append_prompts", kind="append", B=2, Hq=32, Hkv=8, n=777, D=128, R=64, page=64,
             hi=1, dtype="fp16", interleaved=True, factor=1.0),
        # Beam search: each of sixteen beams gets a last page of its own.
        dict(name="copy_beams", kind="copy", pages=512, n=16, Hkv=8, page=16, D=128, dtype="bf16"),
        # Compaction of a large pool: a fifth of its pages move.
        dict(name="copy_compaction", kind="copy", pages=5003, n=1009, Hkv=8, page=64, D=128,
             dtype="bf16"),
    ]


# ---------------------------------------------------------------------------------
# Drawn cases
# ---------------------------------------------------------------------------------

# The most work of a drawn case: head-dim multiplies of all (query, key) pairs of the plain
# forms, half of sinks_prompt_long's, and all of sinks_train_gqa's; tokens of the largest pool;
# elements of q and k in rotary_prompts.
_MAX_FORWARD = 32 * 8192 * 8192 * 128 // 2
_MAX_TRAIN = 2 * 32 * 2011 * 2011 * 128
_MAX_POOL = 64 * 32768 * 8 * 128 // 2
_MAX_ROTARY = 2 * 40 * 4096 * 128


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    """(Hq, Hkv) of multi-head, grouped-query and multi-query models."""
    return rng.choice([(8, 8), (12, 12), (16, 16), (32, 32), (8, 2), (32, 8), (24, 8), (28, 4),
                       (40, 8), (8, 1)])


def _options(rng):
    return dict(window=_log(rng, 16, 4096), sinks=rng.choice([1, 4, 4, 4, 8, 16, 33, 64, 128, 200]),
                softcap=rng.choice([20.0, 30.0, 50.0]) if rng.random() < 0.2 else 0.0)


def _draw_forward(rng):
    Hq, Hkv = _heads(rng)
    D = rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256])
    cached = rng.random() < 0.4
    S = rng.choice([1, 1, 2, 7, _log(rng, 16, 1024)]) if cached else _log(rng, 32, 8192)
    Sc = _log(rng, 64, 16384) if cached else 0
    while Hq * S * (S + Sc) * D > _MAX_FORWARD:
        S -= max(1, S // 8)
    room = _MAX_FORWARD // (Hq * S * (S + Sc) * D)
    return dict(kind="forward", B=rng.randint(1, max(1, min(8, room))), Hq=Hq, Hkv=Hkv, S=S, Sc=Sc,
                D=D, dtype=rng.choice(["bf16", "bf16", "fp16"]), causal=cached or rng.random() < 0.85,
                **_options(rng))


def _draw_train(rng):
    Hq, Hkv = _heads(rng)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    S = _log(rng, 64, 1024 if dtype == "fp32" else 4096)
    D = rng.choice([64, 128]) if dtype == "fp32" else rng.choice([64, 96, 128, 128, 192, 256])
    most = _MAX_TRAIN // (8 if dtype == "fp32" else 1)
    while Hq * S * S * D > most:
        S -= S // 8
    room = most // (Hq * S * S * D)
    return dict(kind="train", B=rng.randint(1, max(1, min(6, room))), Hq=Hq, Hkv=Hkv, S=S, D=D,
                dtype=dtype, causal=rng.random() < 0.85, **_options(rng))


def _draw_decode(rng):
    Hq, Hkv = _heads(rng)
    D = rng.choice([64, 128, 128, 256])
    hi = _log(rng, 64, 32768)
    room = _MAX_POOL // (hi * Hkv * D)
    return dict(kind="decode", B=_log(rng, 1, max(1, min(96, room))), Hq=Hq, Hkv=Hkv, D=D,
                page=rng.choice([16, 16, 32, 64, 128]), lo=max(1, hi // rng.choice([1, 4, 64])), hi=hi,
                dtype=rng.choice(["bf16", "bf16", "fp16"]), **_options(rng))


def _draw_rotary(rng):
    Hq, Hkv = _heads(rng)
    D = rng.choice([64, 80, 96, 128, 128, 128, 192, 256])
    S = _log(rng, 1, 8192)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    room = _MAX_ROTARY // ((Hq + Hkv) * S * D * (2 if dtype == "fp32" else 1))
    return dict(kind="rotary", B=_log(rng, 1, max(1, min(64, room))), Hq=Hq, Hkv=Hkv, S=S, D=D,
                R=rng.choice([D, D, D // 2, D // 4]), dtype=dtype, interleaved=rng.random() < 0.4,
                factor=rng.choice([1.0, 1.0, 4.0, 16.0]), offset=rng.choice([0, 0, 17, 131071]),
                packed=rng.random() < 0.3, grad=rng.random() < 0.5)


def _draw_append(rng):
    Hq, Hkv = _heads(rng)
    D = rng.choice([64, 96, 128, 128, 256])
    n = rng.choice([1, 1, 1, 2, 5, _log(rng, 8, 1024)])
    hi = _log(rng, 1, 2048)
    B = _log(rng, 1, max(1, min(128, _MAX_POOL // (16 * (hi + n) * Hkv * D), 4096 // n)))
    return dict(kind="append", B=B, Hq=Hq, Hkv=Hkv, n=n, D=D, R=rng.choice([D, D, D // 2]),
                page=rng.choice([16, 16, 64, 100]), hi=hi, dtype=rng.choice(["bf16", "bf16", "fp16"]),
                interleaved=rng.random() < 0.4, factor=rng.choice([1.0, 1.0, 8.0]))


def _draw_copy(rng):
    Hkv, page, D = rng.choice([1, 2, 8, 8, 32]), rng.choice([16, 16, 64, 128]), rng.choice([64, 96, 128, 256])
    n = _log(rng, 1, max(1, min(1009, 1009 * 8 * 64 * 128 // (Hkv * page * D))))
    return dict(kind="copy", pages=2 * n + _log(rng, 1, 64), n=n, Hkv=Hkv, page=page, D=D,
                dtype=rng.choice(["bf16", "fp16", "fp32"]))


def draw(rng):
    return rng.choice([_draw_forward, _draw_forward, _draw_train, _draw_train, _draw_decode,
                       _draw_decode, _draw_rotary, _draw_rotary, _draw_append, _draw_copy])(rng)


# ---------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------


def _rand(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _heads_view(gen, B, H, S, D, dtype):
    """[B, H, S, D] as a projection's output gives it: a view of [B, S, H D]."""
    return _rand(gen, (B, S, H, D), dtype).transpose(1, 2)


def _tables(rng, lens, page, pages=0):
    """Block tables over a pool in random page order: (int32 [B, width], pages of the pool:
    those used, or as many as given)."""
    need = [-(-n // page) for n in lens]
    pages = pages or sum(need)
    order = rng.permutation(pages)
    bt = np.zeros((len(lens), max(need)), dtype=np.int32)
    at = 0
    for b, n in enumerate(need):
        bt[b, :n] = order[at:at + n]
        at += n
    return torch.from_numpy(bt).cuda(), pages


def _frequencies(R, factor):
    """base^(-2i / R) in 64 bits; a longer context by a larger base, the highest frequency kept
    and the lowest divided by the factor."""
    base = 10000.0 * factor ** (R / (R - 2)) if factor != 1.0 else 10000.0
    return torch.tensor([base ** (-2.0 * i / R) for i in range(R // 2)], dtype=torch.float64,
                        device="cuda")


def prepare(case, seed):
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    st = {"case": case}
    if kind == "copy":
        shape = (case["pages"], case["Hkv"], case["page"], case["D"])
        st["k_pages"], st["v_pages"] = _rand(gen, shape, dt), _rand(gen, shape, dt)
        ids = rng.permutation(case["pages"]).astype(np.int32)
        st["src"] = torch.from_numpy(ids[:case["n"]].copy()).cuda()
        st["dst"] = torch.from_numpy(ids[case["n"]:2 * case["n"]].copy()).cuda()
        return st
    B, Hq, Hkv, D = (case[x] for x in ("B", "Hq", "Hkv", "D"))
    if kind in ("forward", "train"):
        S = case["S"]
        st["q"] = _heads_view(gen, B, Hq, S, D, dt)
        st["k"] = _heads_view(gen, B, Hkv, S, D, dt)
        st["v"] = _heads_view(gen, B, Hkv, S, D, dt)
        if kind == "train":
            st["do"] = _heads_view(gen, B, Hq, S, D, dt)
            for x in "qkv":
                st[x].requires_grad_()
        elif case["Sc"]:
            st["kv_cache"] = tuple(_rand(gen, (B, Hkv, case["Sc"], D), dt) for _ in "kv")
    elif kind == "decode":
        lens = [int(x) for x in rng.integers(case["lo"], case["hi"] + 1, size=B)]
        st["bt"], pages = _tables(rng, lens, case["page"])
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["max_len"] = max(lens)
        shape = (pages, Hkv, case["page"], D)
        st["k_pages"], st["v_pages"] = _rand(gen, shape, dt), _rand(gen, shape, dt)
        st["q"] = _rand(gen, (B, Hq, D), dt)
    elif kind == "rotary":
        S = case["S"]
        for x, H in (("q", Hq), ("k", Hkv), ("dq", Hq), ("dk", Hkv)):
            if x in ("q", "k") or case["grad"]:
                st[x] = _heads_view(gen, B, H, S, D, dt)
        if case["grad"]:
            st["q"].requires_grad_()
            st["k"].requires_grad_()
        st["inv_freq"] = _frequencies(case["R"], case["factor"])
        st["positions"] = None
        if case["packed"]:  # documents one after another in each row, positions from 0 in each
            cut = torch.from_numpy(rng.integers(0, S, size=(B, 1))).cuda()
            pos = torch.arange(S, device="cuda")[None, :].expand(B, S)
            st["positions"] = torch.where(pos < cut, pos, pos - cut) + case["offset"]
    else:  # append
        n = case["n"]
        at = [int(x) for x in rng.integers(0, case["hi"], size=B)]
        st["bt"], pages = _tables(rng, [x + n for x in at], case["page"],
                                  B * -(-(case["hi"] + n) // case["page"]))
        st["at"] = torch.tensor(at, dtype=torch.int32, device="cuda")
        shape = (pages, Hkv, case["page"], D)
        st["k_pages"], st["v_pages"] = _rand(gen, shape, dt), _rand(gen, shape, dt)
        st["q"] = _heads_view(gen, B, Hq, n, D, dt)
        st["k"] = _heads_view(gen, B, Hkv, n, D, dt)
        st["v"] = _heads_view(gen, B, Hkv, n, D, dt)
        st["inv_freq"] = _frequencies(case["R"], case["factor"])
    return st


# ---------------------------------------------------------------------------------
# One pass: plain forms
# ---------------------------------------------------------------------------------


def _visible(rows, keys, case):
    """Keys that rows see: not after the row, and inside its window or among the sinks."""
    gap = rows[:, None] - keys[None, :]
    seen = (gap < case["window"]) | (keys < case["sinks"])[None, :]
    return seen & (gap >= 0) if case["causal"] else seen


def _scores(q, k, case):
    s = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(case["D"]))
    return case["softcap"] * torch.tanh(s / case["softcap"]) if case["softcap"] else s


def _spread(x, case):
    """A KV head for each query head, in 32 bits."""
    return x.detach().float().repeat_interleave(case["Hq"] // case["Hkv"], dim=1)


def _gathered(x, case):
    """The sum over the query heads of each KV head."""
    return x.unflatten(1, (case["Hkv"], -1)).sum(dim=2)


def _plain_forward(st, case):
    k, v = st["k"], st["v"]
    if case["Sc"]:
        k, v = torch.cat([st["kv_cache"][0], k], dim=2), torch.cat([st["kv_cache"][1], v], dim=2)
    keys = torch.arange(k.size(2), device="cuda")
    seen = _visible(keys[case["Sc"]:], keys, case)
    s = _scores(st["q"].float(), _spread(k, case), case).masked_fill(~seen, float("-inf"))
    m = s.amax(dim=-1, keepdim=True)
    e = torch.exp(s - m)
    total = e.sum(dim=-1, keepdim=True)
    o = (e @ _spread(v, case)) / total
    return o.to(st["q"].dtype), m + torch.log(total)


def _plain_train(st, case):
    q, do = st["q"].detach().float(), st["do"].float()
    k, v = _spread(st["k"], case), _spread(st["v"], case)
    keys = torch.arange(case["S"], device="cuda")
    s = _scores(q, k, case)
    kept = s.masked_fill(~_visible(keys, keys, case), float("-inf"))
    p = torch.exp(kept - kept.amax(dim=-1, keepdim=True))
    p = p / p.sum(dim=-1, keepdim=True)
    o = p @ v
    ds = p * (do @ v.transpose(-1, -2) - (do * o).sum(dim=-1, keepdim=True)) * (1.0 / math.sqrt(case["D"]))
    if case["softcap"]:
        ds = ds * (1.0 - (s / case["softcap"]) ** 2)
    dt = st["q"].dtype
    return (o.to(dt), (ds @ k).to(dt), _gathered(ds.transpose(-1, -2) @ q, case).to(dt),
            _gathered(p.transpose(-1, -2) @ do, case).to(dt))


def _plain_decode(st, case):
    """The sinks and the window of each sequence gathered from the pages, the rest left out."""
    W, N, page = case["window"], case["sinks"], case["page"]
    last = st["lens"].long()[:, None] - 1
    token = torch.cat([torch.arange(N, device="cuda").expand(len(last), N),
                       last - W + 1 + torch.arange(W, device="cuda")], dim=1)
    first = last - W + 1  # a sink inside the window counts once
    seen = torch.cat([(token[:, :N] < first), (token[:, N:] >= 0)], dim=1)
    token = token.clamp(min=0).minimum(last)
    at, slot = st["bt"].long().gather(1, token // page), token % page
    k = st["k_pages"][at, :, slot].float().permute(0, 2, 1, 3)  # [B, Hkv, tokens, D]
    v = st["v_pages"][at, :, slot].float().permute(0, 2, 1, 3)
    q = st["q"].float().unflatten(1, (case["Hkv"], -1))         # [B, Hkv, group, D]
    s = _scores(q, k, case).masked_fill(~seen[:, None, None, :], float("-inf"))
    m = s.amax(dim=-1, keepdim=True)
    e = torch.exp(s - m)
    total = e.sum(dim=-1, keepdim=True)
    return ((e @ v) / total).flatten(1, 2).to(st["q"].dtype), (m + torch.log(total)).flatten(1)


def _turn(x, cos, sin, case):
    """x [B, H, S, D] with its first R dims rotated by the angles of cos and sin [B, 1, S, R / 2]."""
    R = case["R"]
    y = x.detach().float()
    if case["interleaved"]:
        a, b = y[..., 0:R:2], y[..., 1:R:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = y[..., :R // 2], y[..., R // 2:R]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, y[..., R:]], dim=-1).to(x.dtype)


def _angles(positions, inv_freq):
    """cos and sin of far positions: the angles in 64 bits."""
    angle = positions.double()[:, None, :, None] * inv_freq
    return torch.cos(angle).float(), torch.sin(angle).float()


def _plain_rotary(st, case):
    pos = st["positions"]
    if pos is None:
        pos = (case["offset"] + torch.arange(case["S"], device="cuda"))[None, :]
    cos, sin = _angles(pos, st["inv_freq"])
    out = (_turn(st["q"], cos, sin, case), _turn(st["k"], cos, sin, case))
    if case["grad"]:
        out += (_turn(st["dq"], cos, -sin, case), _turn(st["dk"], cos, -sin, case))
    return out


def _plain_append(st, case):
    pos = st["at"].long()[:, None] + torch.arange(case["n"], device="cuda")
    cos, sin = _angles(pos, st["inv_freq"])
    at, slot = st["bt"].long().gather(1, pos // case["page"]), pos % case["page"]
    st["k_pages"][at, :, slot] = _turn(st["k"], cos, sin, case).transpose(1, 2)
    st["v_pages"][at, :, slot] = st["v"].transpose(1, 2)
    return _turn(st["q"], cos, sin, case), st["k_pages"], st["v_pages"]


def _plain_copy(st, case):
    src, dst = st["src"].long(), st["dst"].long()
    st["k_pages"][dst] = st["k_pages"][src]
    st["v_pages"][dst] = st["v_pages"][src]
    return st["k_pages"], st["v_pages"]


# ---------------------------------------------------------------------------------
# One pass: the framework's operators
# ---------------------------------------------------------------------------------


def _own_pass(st, case):
    import fastest_flash_attention_amd as ffa

    kind = case["kind"]
    if kind in ("forward", "train", "decode"):
        opt = dict(sliding_window=case["window"], sink_tokens=case["sinks"],
                   softcap=case["softcap"] or None)
    if kind == "forward":
        return ffa.fastest_flash_attn_forward(
            st["q"], st["k"], st["v"], causal=case["causal"], num_kv_heads=case["Hkv"],
            kv_cache=st.get("kv_cache"), return_lse=True, **opt)
    if kind == "train":
        out = ffa.fastest_flash_attn_func(st["q"], st["k"], st["v"], causal=case["causal"],
                                          num_kv_heads=case["Hkv"], **opt)
        return (out.detach(), *torch.autograd.grad(out, (st["q"], st["k"], st["v"]), st["do"]))
    if kind == "decode":
        return ffa.fastest_flash_paged_decode(
            st["q"], st["k_pages"], st["v_pages"], st["bt"], st["lens"], return_lse=True,
            max_context_len=st["max_len"], **opt)
    if kind == "rotary":
        out = ffa.fastest_flash_rotary(st["q"], st["k"], st["inv_freq"], positions=st["positions"],
                                       q_offset=0 if case["packed"] else case["offset"],
                                       interleaved=case["interleaved"])
        if not case["grad"]:
            return out
        grads = torch.autograd.grad(out, (st["q"], st["k"]), (st["dq"], st["dk"]))
        return (*(x.detach() for x in out), *grads)
    if kind == "append":
        q = ffa.fastest_flash_paged_append(st["k"], st["v"], st["k_pages"], st["v_pages"], st["bt"],
                                           st["at"], q=st["q"], inv_freq=st["inv_freq"],
                                           interleaved=case["interleaved"])
        return q, st["k_pages"], st["v_pages"]
    ffa.fastest_flash_copy_pages(st["k_pages"], st["v_pages"], st["src"], st["dst"])
    return st["k_pages"], st["v_pages"]


_PLAIN = {"forward": _plain_forward, "train": _plain_train, "decode": _plain_decode,
          "rotary": _plain_rotary, "append": _plain_append, "copy": _plain_copy}


def run(state):
    case = state["case"]
    if own:
        return _own_pass(state, case)
    with torch.no_grad():
        return _PLAIN[case["kind"]](state, case)


# ---------------------------------------------------------------------------------
# Work
# ---------------------------------------------------------------------------------


def _pairs(case):
    """Visible (query, key) pairs per head, and the keys that any query sees."""
    S, off = case["S"], case.get("Sc", 0)
    total = S + off
    row = off + np.arange(S, dtype=np.int64)
    last = row if case["causal"] else np.full(S, total - 1)
    first = np.maximum(row - case["window"] + 1, 0)
    sinks = np.minimum(np.minimum(first, case["sinks"]), last + 1)
    low = int(first[0])
    return int((last - first + 1 + sinks).sum()), total - low + min(low, case["sinks"])


def work(case):
    kind = case["kind"]
    e = 4 if case["dtype"] == "fp32" else 2
    if kind == "copy":  # K and V of each page read and written
        return {"bytes": 4 * case["n"] * case["Hkv"] * case["page"] * case["D"] * e, "flops": 0}
    B, Hq, Hkv, D = (case[x] for x in ("B", "Hq", "Hkv", "D"))
    if kind in ("forward", "train"):
        pairs, keys = _pairs(case)
        qo = B * Hq * case["S"] * D * e  # q, or O
        kv = B * Hkv * keys * D * e      # K, or V
        if kind == "train":  # q, dO, O, dQ; K, V, dK, dV; the forward's and five products
            return {"bytes": 4 * qo + 4 * kv, "flops": 14 * D * pairs * B * Hq}
        return {"bytes": 2 * qo + 2 * kv + B * Hq * case["S"] * 4, "flops": 4 * D * pairs * B * Hq}
    if kind == "decode":
        most = case["window"] + case["sinks"]
        tokens = min((case["lo"] + case["hi"]) // 2, most)
        return {"bytes": B * (2 * tokens * Hkv + 2 * Hq) * D * e, "flops": 4 * B * tokens * Hq * D}
    if kind == "rotary":
        x = B * case["S"] * (Hq + Hkv)
        times = 2 if case["grad"] else 1
        return {"bytes": 2 * x * D * e * times, "flops": 3 * x * case["R"] * times}
    x = B * case["n"]
    return {"bytes": 2 * x * (Hq + 2 * Hkv) * D * e, "flops": 3 * x * (Hq + Hkv) * case["R"]}


# ---------------------------------------------------------------------------------
# Results in 64 bits
# ---------------------------------------------------------------------------------


def _head64(q, k, v, off, case, do=None):
    """One head in float64, rows in blocks: q [S, D] at positions off .., k and v [N, D].
    (O, lse), or with the output's gradient (O, dq, dk, dv)."""
    q, k, v = q.double(), k.double(), v.double()
    scale, cap = 1.0 / math.sqrt(case["D"]), case["softcap"]
    key = torch.arange(k.size(0), device=k.device)
    kt, vt = k.t().contiguous(), v.t().contiguous()
    outs, dk, dv = [], torch.zeros_like(k), torch.zeros_like(v)
    for a in range(0, q.size(0), 4096):
        qa = q[a:a + 4096]
        row = (off + a + torch.arange(qa.size(0), device=k.device))[:, None]
        hidden = (key <= row - case["window"]) & (key >= case["sinks"])
        if case["causal"]:
            hidden |= key > row
        s = torch.matmul(qa, kt).mul_(scale)
        t = torch.tanh(s / cap) if cap else None
        s = (cap * t if cap else s).masked_fill(hidden, -math.inf)
        lse = torch.logsumexp(s, dim=1)
        p = torch.exp(s - lse[:, None])
        o = torch.matmul(p, v)
        if do is None:
            outs.append((o, lse))
            continue
        da = do[a:a + 4096].double()
        ds = p * (torch.matmul(da, vt) - torch.sum(da * o, dim=1, keepdim=True)) * scale
        ds = ds * (1 - t * t) if cap else ds
        dk += torch.matmul(ds.t().contiguous(), qa)
        dv += torch.matmul(p.t().contiguous(), da)
        outs.append((o, torch.matmul(ds, k)))
    first, second = (torch.cat(x) for x in zip(*outs))
    return (first, second) if do is None else (first, second, dk, dv)


def _turn64(x, pos, case, freq, sign=1.0):
    """Pair i of x as a complex number, times e^(i angle)."""
    R = case["R"]
    y = x.detach().double().clone()
    head = y[..., :R]
    pair = (head.unflatten(-1, (R // 2, 2)) if case["interleaved"]
            else head.unflatten(-1, (2, R // 2)).transpose(-1, -2)).contiguous()
    angle = pos.double()[..., None] * freq * sign
    z = torch.view_as_complex(pair) * torch.polar(torch.ones_like(angle), angle)
    back = torch.view_as_real(z)
    y[..., :R] = (back if case["interleaved"] else back.transpose(-1, -2)).flatten(-2)
    return y


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "copy":
        k, v = st["k_pages"].double(), st["v_pages"].double()
        for s, d in zip(st["src"].tolist(), st["dst"].tolist()):
            k[d], v[d] = st["k_pages"][s], st["v_pages"][s]
        return k, v
    B, Hq, Hkv, D = (case[x] for x in ("B", "Hq", "Hkv", "D"))
    G = Hq // Hkv
    if kind == "rotary":
        pos = st["positions"]
        if pos is None:
            pos = torch.arange(case["offset"], case["offset"] + case["S"], device="cuda").expand(B, -1)
        out = tuple(_turn64(st[x], pos[:, None], case, st["inv_freq"]) for x in ("q", "k"))
        if case["grad"]:
            out += tuple(_turn64(st[x], pos[:, None], case, st["inv_freq"], -1.0) for x in ("dq", "dk"))
        return out
    if kind == "append":
        k_pages, v_pages = st["k_pages"].double(), st["v_pages"].double()
        at = st["at"].tolist()
        pos = torch.stack([torch.arange(p, p + case["n"], device="cuda") for p in at])
        q, k = (_turn64(st[x], pos[:, None], case, st["inv_freq"]) for x in ("q", "k"))
        table = st["bt"].tolist()
        for b, start in enumerate(at):
            for j in range(case["n"]):
                page, slot = table[b][(start + j) // case["page"]], (start + j) % case["page"]
                k_pages[page, :, slot], v_pages[page, :, slot] = k[b, :, j], st["v"][b, :, j].double()
        return q, k_pages, v_pages
    if kind == "decode":
        o = torch.empty(B, Hq, D, dtype=torch.float64, device="cuda")
        lse = torch.empty(B, Hq, dtype=torch.float64, device="cuda")
        for b, n in enumerate(st["lens"].tolist()):
            # every query head at the last position, over the tokens that it sees
            seen = torch.tensor([t for t in range(n) if t >= n - case["window"] or t < case["sinks"]],
                                device="cuda")
            ids, slot = st["bt"][b].long()[seen // case["page"]], seen % case["page"]
            all_seen = dict(case, window=1, sinks=n, causal=False)
            for h in range(Hkv):
                k, v = st["k_pages"][ids, h, slot], st["v_pages"][ids, h, slot]
                o[b, h * G:(h + 1) * G], lse[b, h * G:(h + 1) * G] = _head64(
                    st["q"][b, h * G:(h + 1) * G], k, v, 0, all_seen)
        return o, lse
    q, k, v = (st[x].detach() for x in "qkv")
    S, off = case["S"], case.get("Sc", 0)
    if off:
        k, v = torch.cat([st["kv_cache"][0], k], dim=2), torch.cat([st["kv_cache"][1], v], dim=2)
    if kind == "train":
        o, dq = (torch.empty(B, Hq, S, D, dtype=torch.float64, device="cuda") for _ in range(2))
        dk, dv = (torch.zeros(B, Hkv, S, D, dtype=torch.float64, device="cuda") for _ in range(2))
        for b in range(B):
            for h in range(Hq):
                o[b, h], dq[b, h], gk, gv = _head64(q[b, h], k[b, h // G], v[b, h // G], 0, case,
                                                    do=st["do"][b, h])
                dk[b, h // G] += gk
                dv[b, h // G] += gv
        return o, dq, dk, dv
    o = torch.empty(B, Hq, S, D, dtype=torch.float64, device="cuda")
    lse = torch.empty(B, Hq, S, 1, dtype=torch.float64, device="cuda")
    for b in range(B):
        for h in range(Hq):
            o[b, h], lse[b, h, :, 0] = _head64(q[b, h], k[b, h // G], v[b, h // G], off, case)
    return o, lse
