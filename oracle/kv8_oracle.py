"""64-bit restatement of the 8-bit paged cache: append, block scores, attention (CPU, torch float64).

Test infrastructure only.  A cache is a dict of float64 tensors: k, v [P, H, page, D] code values, exps
int64 [P, H, 2], bounds [P, H, 2, D].
"""
from __future__ import annotations

import math

import torch

F8 = {torch.float8_e4m3fn: (3, -6, 448.0), torch.float8_e5m2: (2, -14, 57344.0)}   # mantissa bits, least exponent, largest
EXP_MIN, EXP_MAX = -60, 60


def nearest_code(y: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """y (float64) rounded to the nearest code of the type, ties to even, saturating; NaN stays NaN."""
    bits, least, largest = F8[dtype]
    _, x = torch.frexp(torch.where(torch.isfinite(y), y, torch.ones_like(y)))
    step = torch.ldexp(torch.ones_like(y), (x - 1).clamp(min=least) - bits)
    r = torch.round(y / step) * step
    r = torch.where(torch.isinf(y), torch.sign(y) * largest, r)
    return torch.where(torch.isnan(y), y, r.clamp(-largest, largest))


def page_exponent(x: torch.Tensor, dtype: torch.dtype) -> int:
    """Smallest e in range with max finite |x| <= largest * 2^e."""
    a = x.abs()
    a = a[torch.isfinite(a)]
    top = float(a.max()) if a.numel() else 0.0
    for e in range(EXP_MIN, EXP_MAX + 1):
        if top <= F8[dtype][2] * 2.0 ** e:
            return e
    return EXP_MAX


def append(cache: dict, table, k_new, v_new, tok0, counts, dtype) -> dict:
    """The cache after the append (a new dict); k_new/v_new float64 [B, H, n, D]."""
    c = {n: t.clone() for n, t in cache.items()}
    page = c["k"].shape[2]
    for b in range(k_new.shape[0]):
        n0, n = int(tok0[b]), int(counts[b])
        if n == 0:
            continue
        for p in range(n0 // page, (n0 + n - 1) // page + 1):
            pid, t0 = int(table[b, p]), p * page
            first, rows = max(n0 - t0, 0), min(n0 + n - t0, page)
            for h in range(c["k"].shape[1]):
                for i, (name, new) in enumerate((("k", k_new), ("v", v_new))):
                    x = c[name][pid, h, :rows] * 2.0 ** int(c["exps"][pid, h, i])
                    x[first:rows] = new[b, h, t0 + first - n0:t0 + rows - n0]
                    e = page_exponent(x, dtype)
                    code = nearest_code(x * 2.0 ** -e, dtype)
                    c[name][pid, h, :rows] = code
                    c["exps"][pid, h, i] = e
                    if i == 0:
                        c["bounds"][pid, h, 0], c["bounds"][pid, h, 1] = code.amin(dim=0), code.amax(dim=0)
    return c


def block_scores(q, cache, table, lens):
    """(scores, magnitudes) [B, H, max_pages] float64: the sum over the group of the largest q.k of every
    block, and the same sum of magnitudes; -inf and 0 where there is no block.  q [B, Hq, D]."""
    B, Hq, D = q.shape
    H, page = cache["k"].shape[1], cache["k"].shape[2]
    G = Hq // H
    out = torch.full((B, H, table.shape[1]), -math.inf, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for b in range(B):
        for j in range(min(-(-int(lens[b]) // page), table.shape[1])):
            pid = int(table[b, j])
            for h in range(H):
                lo, hi = cache["bounds"][pid, h]
                qq = q[b, h * G:(h + 1) * G]
                s = 2.0 ** int(cache["exps"][pid, h, 0])
                out[b, h, j] = torch.maximum(qq * lo, qq * hi).sum() * s
                mag[b, h, j] = (qq.abs() * torch.maximum(lo.abs(), hi.abs())).sum() * s
    return out, mag


def attention(q, cache, table, lens, *, blocks=None, counts=None, scale=None, weight_bits=11):
    """(out, bound) [B, Hq, Q, D] float64.  `bound`: how far fp32 sums, fp32 base-2 softmax arithmetic and
    weights rounded to fp16 (weight_bits: 11, or 21 for two terms) can put a result off, before the
    rounding of the output:
      scores: D products summed in fp32, D/16 + 4 roundings of the running sum, each at most 2^-22
        of the sum of magnitudes (a tensor core may truncate), and the query's scaled fp16
        form, 2^-25 of its largest element per element;
      exponent: t = s*f + e and t - m, three roundings of at most 2^-23 of |t| + 64;  exp2: 2^-22;
      weights: 2^-weight_bits each, and 2^-25 of the largest weight where fp16 is subnormal;
      sums over T weights: (T/16 + 16) roundings of 2^-22, for the numerator and for the denominator.
    """
    B, Hq, Q, D = q.shape
    H, page = cache["k"].shape[1], cache["k"].shape[2]
    G = Hq // H
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros_like(q)
    bound = torch.zeros_like(q)
    for b in range(B):
        for h in range(H):
            n = int(lens[b])
            if blocks is None:
                blk = list(range(-(-n // page)))
            else:
                blk = [int(x) for x in blocks[b, h, :int(counts[b, h]) if counts is not None else None]]
            if not blk:
                continue
            pid = torch.tensor([int(table[b, j]) for j in blk])
            t = (torch.tensor(blk)[:, None] * page + torch.arange(page)).reshape(-1)
            ek, ev = cache["exps"][pid, h, 0], cache["exps"][pid, h, 1]
            k = (cache["k"][pid, h] * torch.pow(2.0, ek.double())[:, None, None]).reshape(-1, D)
            v = (cache["v"][pid, h] * torch.pow(2.0, ev.double())[:, None, None]).reshape(-1, D)
            v8 = cache["v"][pid, h].reshape(-1, D)
            evt = ev.double().repeat_interleave(page)
            for i in range(Q):
                see = t < n - Q + 1 + i
                if not bool(see.any()):
                    continue
                qq = q[b, h * G:(h + 1) * G, i]
                s = qq @ k[see].T * scale
                mag = qq.abs() @ k[see].abs().T * abs(scale)
                # per element 2^-25 of the query row's largest, against |k|
                mag_q = qq.abs().amax(dim=-1, keepdim=True) * k[see].abs().sum(dim=-1)[None] * abs(scale)
                p = torch.softmax(s, dim=-1)
                out[b, h * G:(h + 1) * G, i] = p @ v[see]
                err = (mag * (D / 16 + 4) * 2.0 ** -22 + mag_q * 2.0 ** -25
                       + (s.abs().amax(dim=-1, keepdim=True) * 1.4427 + 64) * 3 * 2.0 ** -23 + 2.0 ** -22)
                rel = 2 * err.amax(dim=-1, keepdim=True) + 2.0 ** -weight_bits + (int(see.sum()) / 16 + 16) * 2 * 2.0 ** -22
                big = (p * torch.pow(2.0, evt[see])[None]).amax(dim=-1, keepdim=True)
                bound[b, h * G:(h + 1) * G, i] = (rel * (p @ v[see].abs())
                                                  + 2.0 ** -25 * big * v8[see].abs().sum(dim=0)[None])
    return out, bound
