"""Inputs and 64-bit references of the prompt-attention, shared-prefix and append tests."""
import math

import torch

D = 128


def pages_for(lens, page, gen, spare=2):
    need = [-(-n // page) for n in lens]
    total = sum(need) + spare
    ids = torch.randperm(total, generator=gen).to(torch.int32)
    table = torch.full((len(lens), max(1, max(need, default=1))), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    return table, total


def fill_pool(lens, page, hkv, dt, gen, make=None):
    """(k, v, table, k_rows, v_rows): pools that hold NaN wherever no token lies."""
    table, total = pages_for(lens, page, gen)
    k = torch.full((total, page, hkv, D), float("nan")).to(dt)
    v = k.clone()
    ks, vs = [], []
    for i, n in enumerate(lens):
        kr, vr = torch.randn(n, hkv, D, generator=gen).to(dt), torch.randn(n, hkv, D, generator=gen).to(dt)
        if make is not None:
            kr, vr = make(i, kr, vr)
        at = torch.arange(n)
        k[table[i, at // page].long(), at % page] = kr
        v[table[i, at // page].long(), at % page] = vr
        ks.append(kr)
        vs.append(vr)
    return k, v, table, ks, vs


def attend64(q, k, v, scale, first):
    """q [n, Hq, D], k / v [L, Hkv, D]; row i sees keys < first[i].  In 64 bits: out, lse, and per
    row sum_j w_j |v_j| and the largest sum_d |q_d k_jd| scale, which the tolerances need."""
    n, hq = q.shape[:2]
    L, hkv = k.shape[:2]
    out, mag = torch.zeros(n, hq, D, dtype=torch.float64), torch.zeros(n, hq, D, dtype=torch.float64)
    lse, big = torch.full((n, hq), -math.inf, dtype=torch.float64), torch.zeros(n, hq, dtype=torch.float64)
    if L == 0 or n == 0:
        return out, lse, mag, big
    hidden = torch.arange(L)[None] >= first[:, None]
    for h in range(hq):
        kk, vv = k[:, h // (hq // hkv)].double(), v[:, h // (hq // hkv)].double()
        s = (q[:, h].double() @ kk.T) * scale
        s[hidden] = -math.inf
        m = s.max(-1, keepdim=True).values
        w = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
        l = w.sum(-1, keepdim=True)
        w = w / torch.where(l > 0, l, torch.ones_like(l))
        out[:, h], mag[:, h] = w @ vv, w @ vv.abs()
        lse[:, h] = torch.where(l > 0, m + l.log(), torch.full_like(l, -math.inf))[:, 0]
        big[:, h] = ((q[:, h].double().abs() @ kk.abs().T) * scale).masked_fill(hidden, 0).max(-1).values
    return out, lse, mag, big


def tolerances(ref, lse, mag, big, dt, n_keys):
    """Bounds that hold for every element.  eps/2 is half a step of the 16-bit type.
    Scores: 128 fp32 products and sums, 130 half steps of fp32 on sum |q k| scale (the scaling
    and the subtraction of the maximum included): e_s.  A weight is off by 2 e_s (its own and the
    sum's), by the exponential's 2^-21, and by eps/2 where P is rounded; the sums over n keys by
    n 2^-24; the result is rounded once more."""
    half = torch.finfo(dt).eps / 2
    e_s = 130 * 2.0 ** -24 * big
    o_tol = half * ref.abs() + (half + 2 * e_s + 2 * n_keys * 2.0 ** -24 + 2.0 ** -20)[..., None] * mag * (1 + half) + 1e-30
    l_tol = e_s + n_keys * 2.0 ** -24 + 2.0 ** -20 + 4 * 2.0 ** -24 * torch.where(torch.isfinite(lse), lse.abs(), torch.zeros_like(lse))
    return o_tol, l_tol


def assert_close(out, lse, ref, ref_lse, mag, big, dt, n_keys):
    out = out.double().cpu()
    o_tol, l_tol = tolerances(ref, ref_lse, mag, big, dt, n_keys)
    worst = ((out - ref).abs() / o_tol).max().item() if out.numel() else 0.0
    assert torch.isfinite(out).all() and worst <= 1.0, f"output off by {worst:.3g} of its bound"
    if lse is not None:
        lse = lse.double().cpu()
        seen = torch.isfinite(ref_lse)
        assert torch.equal(torch.isfinite(lse), seen) and (lse[~seen] == -math.inf).all()
        if seen.any():
            worst = ((lse - ref_lse).abs() / l_tol)[seen].max().item()
            assert worst <= 1.0, f"lse off by {worst:.3g} of its bound"
