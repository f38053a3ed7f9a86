"""64-bit oracle of the paged 8-bit key/value cache -- TEST INFRASTRUCTURE ONLY (see ``oracle``).

Token by token and page by page in Python, on the CPU, from the definition: nothing here shares code
with ``fused_attn``.  ``append`` works on float64 copies of the stored e4m3 values; ``attention``
also returns how far a result may be off, from the roundings that the kernels are allowed.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

E4M3_MAX = 448.0
MIN_EXP, MAX_EXP = -64, 120

# The 127 finite magnitudes, from the format: 4 exponent bits (bias 7), 3 significand bits.
MAGNITUDES = torch.tensor([(m / 8) * 2.0**-6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
                           for e in range(16) for m in range(8)][:127], dtype=torch.float64)


def round_e4m3(x: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 value, ties to an even significand; NaN where x is not finite."""
    x = x.double()
    a = x.abs().contiguous()
    hi = torch.searchsorted(MAGNITUDES, a).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = MAGNITUDES[hi] - a, a - MAGNITUDES[lo]
    at = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    y = torch.copysign(MAGNITUDES[at], x)
    return torch.where(torch.isfinite(x), y, torch.full_like(y, math.nan))


def needed_exp(amax: float) -> int:
    if amax == 0:
        return MIN_EXP
    m, e = math.frexp(amax)
    return min(MAX_EXP, max(MIN_EXP, e - 9 if m <= 0.875 else e - 8))


def rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool):
    """x [heads, D] in float64 at one position, cos / sin [rot / 2]."""
    y = x.clone()
    half = cos.numel()
    for j in range(half):
        a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
        y[:, a] = x[:, a] * cos[j] - x[:, b] * sin[j]
        y[:, b] = x[:, b] * cos[j] + x[:, a] * sin[j]
    return y


class Pages(NamedTuple):
    """float64 copies of a cache: k, v [P, Hkv, page, D] (unscaled), k_scale, v_scale [P, Hkv]."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def pages_of(k, v, k_scale, v_scale) -> Pages:
    return Pages(*(t.detach().cpu().float().double().contiguous().clone() for t in (k, v)),
                 *(t.detach().cpu().double().clone() for t in (k_scale, v_scale)))


def _offsets(T: int, S: int, cu) -> list[int]:
    return [int(x) for x in cu] if cu is not None else [T // S * i for i in range(S + 1)]


def append(c: Pages, k, v, table, lens, cu=None, q=None, cos=None, sin=None, interleaved=False):
    """Appends to `c` in place; returns q rotated (float64, zeros behind the last sequence).  A
    token without a page, a position in cos / sin or a place in front of the cache is left out."""
    P, Hkv, size, D = c.k.shape
    k, v = k.detach().cpu().double(), v.detach().cpu().double()
    out = None
    if q is not None:
        q = q.detach().cpu().double()
        out = torch.zeros_like(q)
    cu = _offsets(k.shape[0], len(lens), cu)
    if cos is not None:
        cos, sin = cos.cpu().double(), sin.cpu().double()
    for s, held in enumerate(int(x) for x in lens):
        n = cu[s + 1] - cu[s]
        by_page: dict[int, list] = {}
        for i in range(n):
            pos = held - n + i
            if pos < 0:
                continue
            row_k, row_v = k[cu[s] + i], v[cu[s] + i]
            if cos is not None and pos >= cos.shape[0]:
                continue
            if cos is not None:
                row_k = rotate(row_k, cos[pos], sin[pos], interleaved)
                if q is not None:
                    out[cu[s] + i] = rotate(q[cu[s] + i], cos[pos], sin[pos], interleaved)
            at = pos // size
            page = int(table[s][at]) if at < len(table[s]) else -1
            if 0 <= page < P:
                by_page.setdefault(page, []).append((pos % size, row_k, row_v))
        for page, rows in by_page.items():
            first = rows[0][0]
            for which, (cache, scale) in enumerate(((c.k, c.k_scale), (c.v, c.v_scale))):
                use = [(slot, both[which]) for slot, *both in rows]
                for h in range(Hkv):
                    new = torch.stack([r[h] for _, r in use])
                    fin = new[torch.isfinite(new)].abs()
                    e = needed_exp(float(fin.max()) if fin.numel() else 0.0)
                    if first > 0:
                        old = float(scale[page, h])
                        e = max(e, min(MAX_EXP, max(MIN_EXP, math.ceil(math.log2(old)))))
                        if old != 2.0**e:
                            cache[page, h, :first] = round_e4m3(cache[page, h, :first] * old
                                                                / 2.0**e)
                    scale[page, h] = 2.0**e
                    for slot, r in use:
                        cache[page, h, slot] = round_e4m3(r[h] / 2.0**e)
    return out


class Answer(NamedTuple):
    o: torch.Tensor
    lse: torch.Tensor
    o_room: torch.Tensor    # how far o may be off in absolute value, before its own rounding
    lse_room: torch.Tensor


def attention(c: Pages, q, table, lens, cu=None, causal=True, scale=None) -> Answer:
    """Attention over the cache in 64 bits, and the room for the kernels' roundings:

    * scores: fp32 sums of D exact products, so |ds| <= D 2^-24 scale sum |q k| and some 2^-24 of
      the score, relative error of P the same;
    * P in fp16: half a step, 2^-11 relative (2^-12 of the binade's top), or 2^-25 where the largest
      P of a row is 1 or more;
    * exponentials and sums in fp32: 2^-18 relative covers 2^-22 each and chains of additions.
    """
    P, Hkv, size, D = c.k.shape
    T, H, _ = q.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    q = q.detach().cpu().double()
    group = H // Hkv
    o, o_room = torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, D, dtype=torch.float64)
    lse, lse_room = torch.zeros(T, H, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    cu = _offsets(T, len(lens), cu)
    for s, held in enumerate(int(x) for x in lens):
        n = cu[s + 1] - cu[s]
        held = max(0, min(held, len(table[s]) * size))
        ids = [int(p) for p in table[s][: -(-held // size)]]
        key = torch.arange(held)
        here = torch.tensor([0 <= ids[j // size] < P for j in range(held)], dtype=torch.bool)
        slots = [(max(0, ids[j // size]) if here[j] else 0, j % size) for j in range(held)]
        for h in range(Hkv):
            def rows(cache, sc):
                if not held:
                    return torch.zeros(0, D, dtype=torch.float64), torch.ones(0, dtype=torch.float64)
                return (torch.stack([cache[p, h, x] for p, x in slots]),
                        torch.stack([sc[p, h] for p, _ in slots]))

            kq, ks = rows(c.k, c.k_scale)
            vq, vs = rows(c.v, c.v_scale)
            kk, vv = kq * ks[:, None], vq * vs[:, None]
            for i in range(n):
                sees = here & (key <= held - n + i) if causal else here
                for g in range(group):
                    x = h * group + g
                    t = cu[s] + i
                    if not bool(sees.any()):
                        lse[t, x] = math.inf
                        continue
                    qq, k1, v1, vs1 = q[t, x], kk[sees], vv[sees], vs[sees]
                    a = (k1 @ qq) * scale
                    ds = D * 2.0**-24 * scale * (k1.abs() @ qq.abs()) + 2.0**-22 * a.abs()
                    m = a.max()
                    p = torch.exp(a - m)
                    total = p.sum()
                    o[t, x] = (p @ v1) / total
                    lse[t, x] = m + torch.log(total)
                    worst = float(ds.max())
                    w = (p @ v1.abs()) / total
                    # 2^-25 of the largest t = a + ln vs, for every key, in units of its V
                    u = a + torch.log(vs1)
                    floor = torch.exp(u.max() - lse[t, x]) * (v1 / vs1[:, None]).abs().sum(0)
                    o_room[t, x] = w * (2.0**-11 + 2 * worst + 2.0**-18) + 2.0**-25 * floor
                    lse_room[t, x] = worst + 2.0**-18 + 2.0**-22 * abs(float(lse[t, x]))
    return Answer(o, lse, o_room, lse_room)
