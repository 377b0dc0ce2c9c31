"""Plain 64-bit forms of the attention operators (CPU torch, loops): what the tests compare with.

Rotation, the append into the paged 8-bit cache (one power-of-two scale for each 16 tokens and head, older codes
rescaled when it grows), and causal attention over the cache, each written from its definition.
"""
import math

import torch

PAGE, BLOCK = 64, 16
E4M3 = torch.float8_e4m3fn


def rotate(x, positions, inv_freq, mscale=1.0, layout="half", offset=0, inverse=False):
    """x [tokens, heads, dim] -> float64; the angles in 64 bits (positions below 2^53)."""
    y = x.double().clone()
    half = len(inv_freq)
    for i, f in enumerate(inv_freq):
        t = positions.double() * f * (-1.0 if inverse else 1.0)
        c, s = (t.cos() * mscale)[:, None], (t.sin() * mscale)[:, None]
        a, b = (offset + i, offset + i + half) if layout == "half" else (offset + 2 * i, offset + 2 * i + 1)
        xa, xb = x[..., a].double(), x[..., b].double()
        y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
    return y


def scale_exponent(amax):
    """Smallest e with amax <= 448 * 2^e, at least -126."""
    if amax == 0:
        return -126
    e = math.ceil(math.log2(amax / 448.0))
    while amax > 448.0 * 2.0**e:
        e += 1
    while amax <= 448.0 * 2.0 ** (e - 1):
        e -= 1
    return max(e, -126)


def append(cache, k, v, q_start, seq_lens, table):
    """cache: dict of CPU tensors k, v (float8), ks, vs (exponents, int) updated in place; k already rotated (float64).
    Returns {(page, head, slot): exact key row} and the same of values, for the rounding's own bound."""
    exact_k, exact_v = {}, {}
    for b, n in enumerate(seq_lens):
        m = q_start[b + 1] - q_start[b]
        ctx = n - m
        for base in range(max(ctx, 0) // BLOCK * BLOCK, n, BLOCK):
            page, at = table[b][base // PAGE], base % PAGE
            lo, hi = max(max(ctx, 0) - base, 0), min(n - base, BLOCK)
            if lo >= hi:
                continue
            rows = slice(q_start[b] + base + lo - ctx, q_start[b] + base + hi - ctx)
            for h in range(k.shape[1]):
                kr, vr = k[rows, h].double().clone(), v[rows, h].double().clone()
                bad = ~(torch.isfinite(kr).all(1) & torch.isfinite(vr).all(1))
                kr[bad] = math.nan
                vr[~torch.isfinite(vr)] = 0.0
                for name, r, sn in (("k", kr, "ks"), ("v", vr, "vs")):
                    fin = r[torch.isfinite(r)].abs()
                    e = scale_exponent(float(fin.max()) if fin.numel() else 0.0)
                    old = int(cache[sn][page, h, at // BLOCK])
                    if lo > 0:
                        e = max(e, old)
                    codes = cache[name][page, h]
                    view = codes if name == "k" else codes.T          # [64, dim]
                    if lo > 0 and e > old:
                        was = view[at:at + lo].float() * 2.0 ** (old - e)
                        view.view(torch.uint8)[at:at + lo] = was.to(E4M3).view(torch.uint8)
                    view.view(torch.uint8)[at + lo:at + hi] = (r * 2.0 ** -e).float().to(E4M3).view(torch.uint8)
                    cache[sn][page, h, at // BLOCK] = e
                for t in range(hi - lo):
                    exact_k[page, h, at + lo + t], exact_v[page, h, at + lo + t] = kr[t], vr[t]
    return exact_k, exact_v


def attend(cache, q, q_start, seq_lens, table, scale, window=0):
    """(out, weighted mean of |v|, bound of |scale q.k|, scale * max|q| * max sum|k|), float64; rows of no sequence stay NaN in out."""
    T, H, _ = q.shape
    kvh, dv = cache["k"].shape[1], cache["v"].shape[2]
    g = H // kvh
    out = torch.full((T, H, dv), math.nan, dtype=torch.float64)
    mean_abs = torch.zeros(T, H, dv, dtype=torch.float64)
    size = torch.zeros(T, H, 1, dtype=torch.float64)
    loud = torch.zeros(T, H, 1, dtype=torch.float64)
    for b, n in enumerate(seq_lens):
        r0, r1 = q_start[b], q_start[b + 1]
        out[r0:r1] = 0.0
        if n == 0 or r1 == r0:
            continue
        pages = torch.tensor([table[b][i] for i in range(-(-n // PAGE))])
        for h in range(kvh):
            two = lambda e: torch.exp2(e.double()).repeat_interleave(BLOCK, -1)   # noqa: E731
            K = (cache["k"][pages, h].double() * two(cache["ks"][pages, h])[..., None]).reshape(-1, q.shape[2])[:n]
            V = (cache["v"][pages, h].double() * two(cache["vs"][pages, h])[:, None, :]).transpose(1, 2).reshape(-1, dv)[:n]
            for i in range(r1 - r0):
                pos = n - (r1 - r0) + i
                lo = max(0, pos + 1 - window) if window else 0
                if pos < 0:
                    continue
                Q = q[r0 + i, h * g:(h + 1) * g].double()
                Ks, Vs = K[lo:pos + 1], V[lo:pos + 1]
                w = torch.softmax(Q @ Ks.T * scale, -1)
                out[r0 + i, h * g:(h + 1) * g] = w @ Vs
                mean_abs[r0 + i, h * g:(h + 1) * g] = w @ Vs.abs()
                size[r0 + i, h * g:(h + 1) * g, 0] = (Q.abs() @ Ks.abs().T * scale).max(-1).values
                loud[r0 + i, h * g:(h + 1) * g, 0] = Q.abs().max(-1).values * Ks.abs().sum(-1).max() * scale
    return out, mean_abs, size, loud
