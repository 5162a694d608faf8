"""Attention over a sliding window with sinks in float64 on the CPU, with error bounds (not a test
module).

Bounds, e = half a step of the type relative to a value (torch.finfo(t).eps / 2), u = 2^-12 the
fp32 part: a score is off by at most D 2^-24 sum |q_i k_i| scale (below 2^-13 for the inputs here)
and the exponential, softcap and sums by less than 2^-13 more, relative to p.
  O   p is rounded to the type for P V, O once:      (e + u) sum p |v| + e |O|
  dV  p rounded, dV once:                            (e + u) sum p |dO| + e |dV|
  dS  = p (dO.v - D_i), D_i = rowsum(dO O) from the rounded O: off by e sum |dO O| there, by u in
      p and by e for its own rounding:               p e sum |dO O| + (e + u) |dS| + u p |dO.v - D_i|
      and the difference of two fp32 sums of D products, each off by at most D 2^-24 times the
      sum of its products' sizes (they cancel where a row sees one key: dS is 0 there, the sums
      are not):                                      p D 2^-24 (sum |dO v| + sum |dO O|)
  dQ, dK sum those times |k|, |q|, and round once. fp32 has no rounding of p, dS: e = 2^-24 then.
"""

from __future__ import annotations

import math

import torch

U = 2.0 ** -12


def visible(rows, keys, causal, window, sinks):
    ok = torch.ones(len(rows), len(keys), dtype=torch.bool)
    if causal:
        ok &= keys[None] <= rows[:, None]
    if window is not None:
        ok &= (keys[None] > rows[:, None] - window) | (keys[None] < sinks)
    return ok


def attend(q, k, v, *, causal, window, sinks, off=0, scale=None, softcap=None, dout=None):
    """One head: q [S, D] at positions off .., k, v [N, D]. A dict of results and ``*_tol`` bounds;
    with ``dout`` the gradients too."""
    e = torch.finfo(q.dtype).eps / 2
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    scale = 1.0 / math.sqrt(q.size(1)) if scale is None else scale
    s = (q @ k.T) * scale
    t = torch.tanh(s / softcap) if softcap else None
    s = softcap * t if softcap else s
    ok = visible(off + torch.arange(q.size(0)), torch.arange(k.size(0)), causal, window, sinks)
    s = s.masked_fill(~ok, float("-inf"))
    lse = torch.logsumexp(s, dim=1)
    p = torch.where(ok, torch.exp(s - lse[:, None]), torch.zeros_like(s))
    p = torch.nan_to_num(p, nan=0.0)  # rows that see nothing
    o = p @ v
    r = {"o": o, "lse": lse, "o_tol": (e + U) * (p @ v.abs()) + e * o.abs()}
    if dout is None:
        return r
    do = dout.double().cpu()
    dp = do @ v.T - (do * o).sum(1, keepdim=True)
    size = (do * o).abs().sum(1, keepdim=True)
    cap = (1 - t * t) if softcap else 1.0
    ds = p * dp * cap
    sums = q.size(1) * 2.0 ** -24 * (do.abs() @ v.abs().T + size)
    ds_tol = (p * (e * size + sums) + (e + U) * ds.abs() + U * p * dp.abs()) * abs(scale)
    ds = ds * scale
    r["dq"], r["dk"], r["dv"] = ds @ k, ds.T @ q, p.T @ do
    r["dq_tol"] = ds_tol @ k.abs() + e * r["dq"].abs()
    r["dk_tol"] = ds_tol.T @ q.abs()
    r["dv_tol"] = (e + U) * (p.T @ do.abs())
    return r


def batch(q, k, v, *, dout=None, **kw):
    """[B, H, S, D] with k, v of fewer heads: results stacked, dK / dV summed over groups (their
    own rounding added after the sum)."""
    e = torch.finfo(q.dtype).eps / 2
    B, Hq = q.shape[:2]
    G = Hq // k.size(1)
    out = {}
    for b in range(B):
        for h in range(Hq):
            r = attend(q[b, h], k[b, h // G], v[b, h // G], dout=None if dout is None else dout[b, h], **kw)
            for name, x in r.items():
                heads = k.size(1) if name[:2] in ("dk", "dv") else Hq
                t = out.setdefault(name, torch.zeros(B, heads, *x.shape, dtype=torch.float64))
                if heads == Hq and name[:2] not in ("dk", "dv"):
                    t[b, h] = x
                else:
                    t[b, h // G] += x
    for name in ("dk", "dv"):
        if name in out:
            out[name + "_tol"] += e * out[name].abs()
    return out


def check(got, ref, name, what, lse_abs=1e-3):
    got = got.detach().double().cpu()
    want = ref[name]
    if name == "lse":
        got = got.reshape(want.shape)
        assert torch.equal(torch.isneginf(got), torch.isneginf(want)), f"{what}: lse -inf at other rows"
        fin = torch.isfinite(want)
        off = (got - want)[fin].abs().max().item() if fin.any() else 0.0
        assert off <= lse_abs, f"{what}: lse off by {off:.3e}"
        return
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{what}: {name} not finite"
    over = (got - want).abs() - ref[name + "_tol"]
    worst = over.max().item() if over.numel() else -1.0
    # (products of values near fp16's lowest normal step by 2^-24)
    assert worst <= 2.0 ** -24, f"{what}: {name} {worst:.3e} over its bound, off by {(got - want).abs().max():.3e}"
