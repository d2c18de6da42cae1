"""The paged 8-bit cache restated in 64 bits on the host: planning, appending, attention, and the error a
correct kernel may have."""
from __future__ import annotations

import math

import torch

E4M3 = torch.float8_e4m3fn


def plan(cached, new, table, free_pages, free_count, page, max_tokens):
    """Plain lists in and out; `table` is a list of rows and is updated."""
    lengths, cu, slots = [], [0], [-1] * max_tokens
    wanted, taken = 0, 0
    for i, (c, n) in enumerate(zip(cached, new)):
        start, stop = cu[-1], cu[-1] + max(n, 0)
        ok = c >= 0 and n >= 0 and c + n <= len(table[i]) * page
        have, need = -(-c // page), 0
        if ok:
            need = -(-(c + n) // page) - have
        wanted += need
        served = ok and stop <= max_tokens and (need == 0 or wanted <= free_count)
        lengths.append(c + n if served else c)
        if served:
            for k in range(need):
                table[i][have + k] = free_pages[free_count - 1 - (wanted - need) - k]
            taken = max(taken, wanted if need else 0)
            for t in range(n):
                pos = c + t
                slots[start + t] = table[i][pos // page] * page + pos % page
        cu.append(stop)
    return lengths, [min(v, max_tokens) for v in cu], slots, free_count - taken


def round_e4m3(y: torch.Tensor) -> torch.Tensor:
    """float64, |y| <= 448 (or NaN), to the nearest e4m3 value, ties to even."""
    _, e = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), (e - 1).clamp_min(-6) - 3)
    return torch.round(y / step) * step


def append(x, slots, code, scale, page):
    """code: float64 [pages, Hkv, page, D] of code values, scale: float64 [pages, Hkv]; both updated.  x: [T, Hkv, D]."""
    x = x.double()
    by_page: dict = {}
    for t, s in enumerate(slots):
        if 0 <= s < code.shape[0] * page:
            by_page.setdefault(s // page, []).append((s % page, t))
    for p, rows in by_page.items():
        begin = min(r for r, _ in rows)
        ts = [t for _, t in rows]
        for h in range(x.shape[1]):
            v = x[ts, h]
            finite = v[torch.isfinite(v)].abs()
            amax = float(finite.max()) if finite.numel() else 0.0
            k = -110
            if amax > 0:
                m, e = math.frexp(amax)              # 448 = 0.875 * 2^9
                k = max(k, e - 9 if m <= 0.875 else e - 8)
            s = 2.0 ** k
            if begin:
                s = max(s, float(scale[p, h]))
                code[p, h, :begin] = round_e4m3(code[p, h, :begin] * (float(scale[p, h]) / s))
            scale[p, h] = s
            for r, t in rows:
                y = torch.where(torch.isfinite(x[t, h]), x[t, h] / s, math.nan)
                code[p, h, r] = round_e4m3(y)


def attend(Q, code, kscale, vcode, vscale, table, lengths, cu, page, scale, causal, many=False):
    """(O, allowed error) in float64 for Q [T, Hq, D]; rows outside cu are NaN.

    What a kernel with fp32 sums and P rounded to fp16 may be off by, with A = sum p |v| / sum p (per element):
      P to fp16 (half a step, relative 2^-11; below 2^-14 absolute 2^-25)    -> 2^-11 A + 2^-25 sum |v| / sum p,
      a score's fp32 dot product of D terms and its scaling, d = (D + 8) 2^-24 scale sum |q k|, shifts p by a
      factor e^d in numerator and denominator                                 -> 2 d A,
      exp2 (2^-22) and the fp32 sums over keys (sequential at worst per lane:
      keys / 8 terms, and the merges)                                         -> (2^-21 + 2 keys/8 2^-24) A,
      the result's own rounding                                               -> eps / 2 |o|.
    `many`, the kernel for many rows, widens codes to f16 times a power of two, relative to the largest scale: half of
    f16's smallest step, 2^-25, times that scale per element of K (a score: 2^-25 kmax scale sum |q|, added to d)
    and V (2^-25 vmax); and it rounds V times what its scale is beside a power of two to f16 -> 2^-11 A.
    """
    T, Hq, D = Q.shape
    Hkv = code.shape[1]
    G = Hq // Hkv
    out = torch.full((T, Hq, D), math.nan, dtype=torch.float64)
    tol = torch.zeros((T, Hq, D), dtype=torch.float64)
    half_step = torch.finfo(Q.dtype).eps / 2
    for i in range(len(lengths)):
        a, b, L = cu[i], cu[i + 1], lengths[i]
        n = b - a
        if n == 0:
            continue
        ids = table[i][: -(-L // page)]
        for h in range(Hkv):
            K = (code[ids, h] * kscale[ids, h, None, None]).reshape(-1, D)[:L]
            V = (vcode[ids, h] * vscale[ids, h, None, None]).reshape(-1, D)[:L]
            q = Q[a:b, h * G:(h + 1) * G].double()                            # [n, G, D]
            z = torch.einsum("ngd,kd->ngk", q, K) * scale
            size = torch.einsum("ngd,kd->ngk", q.abs(), K.abs()) * abs(scale)
            if causal:
                blind = torch.arange(L) > (torch.arange(n)[:, None] + L - n)
                z = z.masked_fill(blind[:, None], -math.inf)
            if L == 0:
                out[a:b, h * G:(h + 1) * G] = 0
                continue
            top = z.amax(dim=2, keepdim=True)
            p = torch.exp(z - top.clamp_min(-1e300))
            l = p.sum(dim=2, keepdim=True)
            o = torch.where(l > 0, (p @ V) / l.clamp_min(1e-300), torch.zeros(()).double())
            A = torch.where(l > 0, (p @ V.abs()) / l.clamp_min(1e-300), torch.zeros(()).double())
            rest = torch.where(l > 0, ((p > 0).double() @ V.abs()) / l.clamp_min(1e-300), torch.zeros(()).double())
            d = (D + 8) * 2.0 ** -24 * torch.where(p > 0, size, 0).amax(dim=2, keepdim=True)
            small = 0.0
            if many:
                d = d + 2.0 ** -25 * float(kscale[ids, h].max()) * abs(scale) * q.abs().sum(dim=2, keepdim=True)
                small = 2.0 ** -11 * A + 2.0 ** -25 * float(vscale[ids, h].max())
            err = small + (2.0 ** -11 + 2 * d + 2.0 ** -21 + 2 * (L / 8) * 2.0 ** -24) * A + 2.0 ** -25 * rest
            out[a:b, h * G:(h + 1) * G] = o
            # subnormal results of a 16-bit type are off by half of their smallest step instead
            tiny = torch.finfo(Q.dtype).smallest_normal * half_step
            tol[a:b, h * G:(h + 1) * G] = err + half_step * (o.abs() + err) + tiny
    return out, tol
