"""What is measured of the paged 8-bit key/value cache: ``cache_append`` and ``cache_attention``.

A case is one call as a serving step makes it.  ``run`` computes it with elementary torch operations where ``own``
is false and through ``fused_attn`` where it is true; ``exact`` gives the definition in 64 bits.

The cache: e4m3 pages [P, Hkv, page, D] for K and for V, one fp32 power-of-two scale for each (page, kv head), a block
table [S, max_pages], and the lengths after the step.  Each sequence's new tokens are its last ones.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_E4M3 = torch.float8_e4m3fn
_E4M3_MAX = 448.0
_MIN_EXP, _MAX_EXP = -64, 120


def _fused_attn():
    package = str(Path(__file__).resolve().parents[1] / "fused-attention-cuda_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import fused_attn

    return fused_attn


# --------------------------------------------------------------------------------------------------------------
# cases


def _attention(name, dtype, S, H, Hkv, D, page, lens, new, causal=True, token_major=False):
    return {"name": name, "op": "attention", "dtype": dtype, "S": S, "H": H, "Hkv": Hkv, "D": D, "page": page,
            "len_lo": lens[0], "len_hi": lens[1], "new_lo": new[0], "new_hi": new[1], "causal": causal,
            "token_major": token_major, "tail": 0}


def _append(name, dtype, S, H, Hkv, D, page, lens, new, rot, interleaved=False, token_major=False, tail=0):
    return {"name": name, "op": "append", "dtype": dtype, "S": S, "H": H, "Hkv": Hkv, "D": D, "page": page,
            "len_lo": lens[0], "len_hi": lens[1], "new_lo": new[0], "new_hi": new[1], "rot": rot,
            "interleaved": interleaved, "token_major": token_major, "tail": tail}


def listed():
    return [
        # One user, one token, a short conversation: latency is all there is.
        _attention("decode_one", "bf16", 1, 32, 8, 128, 64, (777, 777), (1, 1)),
        # A full decoding batch, lengths from a fresh prompt to a long one: the cache's bytes bound it.
        _attention("decode_batch", "bf16", 64, 32, 8, 128, 16, (97, 8191), (1, 1)),
        # GPT-2 heads (12 of 64, one key head for each), a batch of 16 inside the 1024 window.
        _attention("decode_gpt2", "fp16", 16, 12, 12, 64, 32, (1, 1024), (1, 1), token_major=True),
        # One long context: the work has to be split along the keys.
        _attention("decode_long", "fp16", 1, 32, 8, 128, 64, (131071, 131071), (1, 1)),
        # A draft of a few tokens checked against the cache.
        _attention("draft_check", "bf16", 32, 32, 8, 128, 64, (500, 4003), (5, 5)),
        # A chunk of a long prompt behind what is cached: products bound it.
        _attention("prompt_chunk", "bf16", 1, 32, 8, 128, 64, (16384, 16384), (2048, 2048)),
        # A mixed step: ragged chunks from one token up, on 128-token pages.
        _attention("mixed_step", "fp16", 8, 16, 4, 128, 128, (300, 6001), (1, 801)),
        # The step of one user: one token into the cache.
        _append("append_one", "bf16", 1, 32, 8, 128, 64, (778, 778), (1, 1), 128),
        # The step of a full decoding batch, in a batch padded to 72 rows.
        _append("append_batch", "bf16", 64, 32, 8, 128, 16, (97, 2047), (1, 1), 128, tail=8),
        # Prompts of a prefill step, ragged.
        _append("append_prompts", "bf16", 6, 32, 8, 128, 64, (1500, 4001), (700, 4000), 128),
        # GPT-2 heads: learned positions, so no rotation; a batch of 16 whole windows.
        _append("append_gpt2", "fp16", 16, 12, 12, 64, 32, (1024, 1024), (1024, 1024), 0, token_major=True),
        # Half of each head rotated, in neighbouring pairs, one key head, behind a cached prefix.
        _append("append_pairs", "fp16", 3, 16, 1, 128, 128, (2500, 9000), (333, 2222), 64, interleaved=True),
    ]


def _spread(lo, hi, n, turn):
    """n whole numbers over [lo, hi], evenly spread in a mixed order, a function of the case alone."""
    return [lo + int((hi - lo + 1) * ((i + 1) * turn % 1.0)) for i in range(n)]


def _lengths(case):
    """(keys held, new tokens) of each sequence."""
    new = _spread(case["new_lo"], case["new_hi"], case["S"], 0.7548776662466927)
    held = _spread(case["len_lo"], case["len_hi"], case["S"], 0.6180339887498949)
    return [max(a, b) for a, b in zip(held, new)], new


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        D = rng.choice([64, 128])
        Hkv = rng.choice([1, 2, 4, 8, 12])
        H = Hkv * rng.choice([1, 2, 3, 4, 7, 8])
        S = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, 131071 if S == 1 else 16000)
        lo = rng.randint(1, hi)
        case = {"op": rng.choice(["attention", "append"]), "dtype": rng.choice(["fp16", "bf16"]), "S": S, "H": H,
                "Hkv": Hkv, "D": D, "page": rng.choice([16, 32, 64, 128]), "len_lo": lo, "len_hi": hi,
                "token_major": rng.random() < 0.3, "tail": rng.choice([0, 0, 3])}
        if rng.random() < 0.5:
            case["new_lo"] = case["new_hi"] = rng.choice([1, 1, 2, 5, 8])
        else:
            case["new_hi"] = _log_int(rng, 1, min(hi, 4000))
            case["new_lo"] = rng.randint(1, case["new_hi"])
        if case["op"] == "attention":
            case["causal"] = rng.random() < 0.8
        else:
            case["rot"] = rng.choice([0, D // 2, D, D])
            case["interleaved"] = case["rot"] > 0 and rng.random() < 0.3
        held, new = _lengths(case)
        # no dearer than the largest listed case of the kind, in work and in the padded plain form's memory
        if case["op"] == "attention":
            w = work(case)
            padded = S * max(held)
            if (w["flops"] <= 5.2e11 and w["bytes"] <= 6e8 and padded * H * max(new) <= 1.1e9
                    and padded * Hkv * D <= 5.5e8):
                return case
        elif sum(new) * (H + 2 * Hkv) * D <= 1.0e8 and sum(held) * Hkv * D <= 1.4e8:
            return case


# --------------------------------------------------------------------------------------------------------------
# inputs


def _pow2(e):
    """2.0**e in float64 for a tensor of whole numbers, exactly."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _need_exp(amax):
    """The least e in [-64, 120] with amax <= 448 * 2**e (int64), amax in float64."""
    m, x = torch.frexp(amax)
    e = torch.where(m <= 0.875, x - 9, x - 8)
    return torch.where(amax > 0, e, torch.full_like(e, _MIN_EXP)).clamp(_MIN_EXP, _MAX_EXP).to(torch.int64)


def _round_e4m3(x):
    """float64 -> the nearest e4m3 value (ties to even), still in float64; not finite -> NaN."""
    _, e = torch.frexp(x)
    step = _pow2((e - 1).clamp(min=-6) - 3)
    y = (torch.round(x / step) * step).clamp(-_E4M3_MAX, _E4M3_MAX)
    return torch.where(torch.isfinite(x), y, torch.full_like(y, float("nan")))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 17)
    dev, dtype = torch.device("cuda"), _DTYPES[case["dtype"]]
    S, H, Hkv, D, page = (case[x] for x in ("S", "H", "Hkv", "D", "page"))
    held, new = _lengths(case)
    T = sum(new) + case["tail"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32)

    # pages in the order a pool hands them out after a while: any; entries past a sequence's last page are -1
    pages = [-(-n // page) for n in held]
    P = sum(pages) + 5
    order = torch.randperm(P, generator=g, device=dev).to(torch.int32)
    table = torch.full((S, max(pages)), -1, dtype=torch.int32)
    at = torch.arange(sum(pages))
    row = torch.repeat_interleave(torch.arange(S), torch.tensor(pages))
    first = torch.cumsum(torch.tensor([0, *pages[:-1]]), 0)
    table[row, at - first[row]] = at.to(torch.int32)
    table = table.to(dev)
    table = torch.where(table >= 0, order[table.clamp(min=0).long()], table)

    state = {"case": case, "block_table": table, "seq_lens": torch.tensor(held, dtype=torch.int32, device=dev),
             "scale": 1.0 / math.sqrt(D)}
    uniform = min(new) == max(new) and case["tail"] == 0
    cu = torch.cumsum(torch.tensor([0, *new]), 0).to(torch.int32).to(dev)
    state["cu_seqlens"] = None if uniform else cu

    # the pages' contents: normal values whose size differs from page to page and from channel to channel
    def pool(spread):
        shape = (P, page, Hkv, D) if case["token_major"] else (P, Hkv, page, D)
        cache = torch.empty(shape, dtype=_E4M3, device=dev)
        view = cache.transpose(1, 2) if case["token_major"] else cache
        scale = torch.empty(P, Hkv, dtype=torch.float32, device=dev)
        channel = torch.exp(spread * randn(Hkv, 1, D))
        step = max(1, (1 << 26) // (Hkv * page * D))
        for i in range(0, P, step):
            x = randn(min(step, P - i), Hkv, page, D) * channel * torch.exp(0.5 * randn(min(step, P - i), Hkv, 1, 1))
            s = _pow2(_need_exp(x.abs().amax((2, 3)).double())).float()
            scale[i:i + step] = s
            view[i:i + step] = (x / s[:, :, None, None]).to(_E4M3)
        return view, scale

    state["k_cache"], state["k_scale"] = pool(0.3)
    state["v_cache"], state["v_scale"] = pool(0.0)
    if case["op"] == "attention":
        state["q"] = randn(T, H, D).to(dtype)
        return state

    # q, k, v as a fused projection leaves them: one [T, (H + 2 Hkv) D] tensor, split into views
    qkv = randn(T, H + 2 * Hkv, D)
    qkv[:, H:H + Hkv] *= torch.exp(0.3 * randn(1, Hkv, D))
    state["q"], state["k"], state["v"] = qkv.to(dtype).split([H, Hkv, Hkv], dim=1)
    state["cos"] = state["sin"] = None
    if case["rot"]:
        half = case["rot"] // 2
        freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)
        angle = torch.arange(max(held) + 64, dtype=torch.float64, device=dev)[:, None] * freq
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    return state


# --------------------------------------------------------------------------------------------------------------
# one pass


def _cu(state):
    if state["cu_seqlens"] is not None:
        return state["cu_seqlens"].long()
    S = state["seq_lens"].numel()
    return torch.arange(S + 1, device=state["q"].device) * (state["q"].shape[0] // S)


def _rotate(x, cos, sin, pos, rot, interleaved):
    """The rotation of x [T, heads, D] at positions pos in 64 bits."""
    x = x.double()
    if not rot:
        return x
    c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    ya, yb = a * c - b * s, b * c + a * s
    y = torch.stack([ya, yb], -1).flatten(-2) if interleaved else torch.cat([ya, yb], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _narrow(x, dtype):
    """float64 -> fp16 / bf16 with one rounding: to odd in 32 bits first, so that the second rounding cannot tie."""
    y = x.float()
    back = y.double()
    bits = y.view(torch.int32)
    down = torch.where((back.abs() > x.abs()) & torch.isfinite(y), bits - 1, bits)  # toward zero
    odd = torch.where((back != x) & torch.isfinite(x), down | 1, bits)
    return odd.view(torch.float32).to(dtype)


def _store(x, page, slot, cache, scale):
    """Quantises x [n, Hkv, D] (64 bits) into its pages' slots; earlier tokens of a page follow its scale."""
    P, Hkv, size, D = cache.shape
    ax = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1)
    amax = torch.zeros(P, Hkv, dtype=torch.float64, device=x.device)
    amax.scatter_reduce_(0, page[:, None].expand(-1, Hkv), ax, "amax")
    begin = torch.full((P,), size, dtype=torch.int64, device=x.device).scatter_reduce_(0, page, slot, "amin")
    used = torch.unique(page)
    old = torch.frexp(scale[used])[1].to(torch.int64) - 1
    exp = _need_exp(amax[used])
    kept = begin[used] > 0
    exp = torch.where(kept[:, None], torch.maximum(exp, old), exp)
    scale[used] = _pow2(exp).float()
    # the earlier tokens of a page that was begun
    part, bytes_ = used[kept], cache.view(torch.uint8)
    shift = _pow2((old - exp)[kept])[:, :, None, None]
    was = bytes_[part]
    moved = _round_e4m3(was.view(_E4M3).double() * shift).to(_E4M3).view(torch.uint8)
    before = torch.arange(size, device=x.device)[None, :] < begin[part][:, None]
    bytes_[part] = torch.where(before[:, None, :, None], moved, was)
    # the new ones
    e = torch.zeros(P, Hkv, dtype=torch.int64, device=x.device)
    e[used] = exp
    y = _round_e4m3(x * _pow2(-e)[page][..., None])
    bytes_[page, :, slot] = y.to(_E4M3).view(torch.uint8)


def _append_plain(state):
    case, table = state["case"], state["block_table"]
    cu, lens = _cu(state), state["seq_lens"].long()
    n = int(cu[-1])
    t = torch.arange(n, device=table.device)
    seq = torch.bucketize(t, cu[1:], right=True)
    pos = lens[seq] - (cu[1:] - cu[:-1])[seq] + t - cu[seq]
    page = table[seq, pos // case["page"]].long()
    slot = pos % case["page"]
    turn = (state["cos"], state["sin"], pos, case["rot"], case["interleaved"])
    q = None
    if case["rot"]:
        q = torch.zeros(state["q"].shape, dtype=state["q"].dtype, device=table.device)
        q[:n] = _narrow(_rotate(state["q"][:n], *turn), q.dtype)
    _store(_rotate(state["k"][:n], *turn), page, slot, state["k_cache"], state["k_scale"])
    _store(state["v"][:n].double(), page, slot, state["v_cache"], state["v_scale"])
    return q


def _gathered(cache, scale, table, valid):
    """[S, Hkv, L, D] in 32 bits: the table's pages in order, zero where no key is held."""
    S, M = table.shape
    _, Hkv, size, D = cache.shape
    at = table.clamp(min=0).long()
    x = cache.view(torch.uint8)[at].view(_E4M3).float() * scale[at][..., None, None]
    x = x.transpose(1, 2).reshape(S, Hkv, M * size, D)
    return torch.where(valid[:, None, :, None], x, torch.zeros((), device=x.device))


def _attention_plain(state):
    case, table, q = state["case"], state["block_table"], state["q"]
    cu, lens = _cu(state), state["seq_lens"].long()
    S, H, Hkv, D = case["S"], case["H"], case["Hkv"], case["D"]
    G, T, dev = H // Hkv, q.shape[0], q.device
    n = cu[1:] - cu[:-1]
    N, L = max(_lengths(case)[1]), table.shape[1] * case["page"]
    key = torch.arange(L, device=dev)
    valid = key[None, :] < lens[:, None]
    i = torch.arange(N, device=dev)
    row = (cu[:-1, None] + i).clamp(max=T - 1)
    qp = q[row].float().reshape(S, N, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(S, Hkv, G * N, D)
    k = _gathered(state["k_cache"], state["k_scale"], table, valid)
    s = torch.matmul(qp, k.transpose(2, 3)).mul_(state["scale"]).view(S, Hkv, G, N, L)
    del k
    last = lens[:, None] - n[:, None] + i if case["causal"] else (lens - 1)[:, None].expand(S, N)
    sees = valid[:, None, :] & (key[None, None, :] <= last[:, :, None])
    s.masked_fill_(~sees[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(torch.isfinite(m), m, torch.zeros_like(m))).exp_()
    total = p.sum(-1, keepdim=True)
    v = _gathered(state["v_cache"], state["v_scale"], table, valid)
    o = torch.matmul(p.view(S, Hkv, G * N, L), v).view(S, Hkv, G, N, D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = torch.where(total > 0, m + total.log(), torch.full_like(m, float("inf")))[..., 0]
    # back to the packed rows; the rows behind the last sequence are zero
    out = torch.zeros(T, H, D, dtype=q.dtype, device=dev)
    out_lse = torch.zeros(T, H, dtype=torch.float32, device=dev)
    live = i[None, :] < n[:, None]
    out[row[live]] = o.permute(0, 3, 1, 2, 4).reshape(S, N, H, D)[live].to(q.dtype)
    out_lse[row[live]] = lse.permute(0, 3, 1, 2).reshape(S, N, H)[live]
    return out, out_lse


def run(state):
    s, case = state, state["case"]
    if case["op"] == "attention":
        if own:
            o, lse = _fused_attn().cache_attention(
                s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["block_table"], s["seq_lens"],
                cu_seqlens=s["cu_seqlens"], is_causal=case["causal"], scale=s["scale"], return_lse=True)
        else:
            o, lse = _attention_plain(s)
        return {"o": o, "lse": lse}
    if own:
        q = _fused_attn().cache_append(
            s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["block_table"], s["seq_lens"],
            cu_seqlens=s["cu_seqlens"], q=s["q"] if case["rot"] else None, cos=s["cos"], sin=s["sin"], interleaved=case["interleaved"])
    else:
        q = _append_plain(s)
    out = {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    return {"q": q, **out} if case["rot"] else out


def work(case):
    held, new = _lengths(case)
    H, Hkv, D, page = (case[x] for x in ("H", "Hkv", "D", "page"))
    T = sum(new)
    if case["op"] == "attention":
        pages = sum(-(-n // page) for n in held)
        if case["causal"]:
            pairs = sum(n * h - n * (n - 1) // 2 for h, n in zip(held, new))
        else:
            pairs = sum(n * h for h, n in zip(held, new))
        nbytes = 4 * T * H * D + 4 * T * H + 2 * sum(held) * Hkv * D + pages * (8 * Hkv + 4)
        return {"bytes": nbytes, "flops": 4 * D * H * pairs}
    touched = sum((h - 1) // page - (h - n) // page + 1 for h, n in zip(held, new))
    # cos and sin are read once for each position that any sequence has
    spans, positions, end = sorted((h - n, h) for h, n in zip(held, new)), 0, 0
    for a, b in spans:
        positions += max(0, b - max(a, end))
        end = max(end, b)
    turned = T * H * D if case["rot"] else 0  # without a rotation the queries stay where they are
    nbytes = 4 * turned + 6 * T * Hkv * D + 4 * positions * case["rot"] + touched * (8 * Hkv + 4)
    return {"bytes": nbytes, "flops": 3 * T * (H + Hkv) * case["rot"] + 4 * T * Hkv * D}


# --------------------------------------------------------------------------------------------------------------
# the definition in 64 bits


def _exact_attention(case, st):
    held, new = _lengths(case)
    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    G, T = H // Hkv, st["q"].shape[0]
    o = torch.zeros(T, H, D, dtype=torch.float64, device="cuda")
    lse = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    t0 = 0
    for s, (L, n) in enumerate(zip(held, new)):
        ids = st["block_table"][s, : -(-L // case["page"])].tolist()
        last = torch.arange(n, device="cuda") + (L - n) if case["causal"] else torch.full((n,), L - 1, device="cuda")
        hidden = torch.arange(L, device="cuda")[None, :] > last[:, None]
        for h in range(Hkv):
            k = torch.cat([st["k_cache"][p, h].double() * st["k_scale"][p, h].double() for p in ids])[:L]
            v = torch.cat([st["v_cache"][p, h].double() * st["v_scale"][p, h].double() for p in ids])[:L]
            for x in range(h * G, h * G + G):
                a = st["q"][t0:t0 + n, x].double() @ k.T * st["scale"]
                a = a.masked_fill(hidden, -math.inf)
                lse[t0:t0 + n, x] = torch.logsumexp(a, -1)
                o[t0:t0 + n, x] = torch.softmax(a, -1) @ v
        t0 += n
    return {"o": o, "lse": lse}


def _nearest(x, values):
    """The nearest of the e4m3 magnitudes `values` (ascending; an even place wins a tie) with x's sign."""
    a = x.abs().contiguous()
    hi = torch.searchsorted(values, a).clamp(max=values.numel() - 1)
    lo = (hi - 1).clamp(min=0)
    up, down = values[hi] - a, a - values[lo]
    take = torch.where(up == down, torch.where(hi % 2 == 0, hi, lo), torch.where(up < down, hi, lo))
    return torch.copysign(values[take], x)


def _exact_append(case, st):
    held, new = _lengths(case)
    H, page, rot = case["H"], case["page"], case["rot"]
    values = torch.arange(127, dtype=torch.uint8).view(_E4M3).double().cuda()
    q = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    caches = {x: st[x + "_cache"].double() for x in "kv"}
    scales = {x: st[x + "_scale"].double() for x in "kv"}
    if rot:
        idx = torch.arange(rot // 2, device="cuda")
        ia, ib = (2 * idx, 2 * idx + 1) if case["interleaved"] else (idx, idx + rot // 2)
    t0 = 0
    for s, (L, n) in enumerate(zip(held, new)):
        rows = {"q": st["q"][t0:t0 + n].double(), "k": st["k"][t0:t0 + n].double(), "v": st["v"][t0:t0 + n].double()}
        if rot:
            c, sn = st["cos"][L - n:L].double()[:, None], st["sin"][L - n:L].double()[:, None]
            for x in "qk":
                a, b = rows[x][..., ia], rows[x][..., ib]
                turned = rows[x].clone()
                turned[..., ia] = a * c - b * sn
                turned[..., ib] = a * sn + b * c
                rows[x] = turned
        q[t0:t0 + n] = rows["q"]
        for j in range((L - n) // page, (L - 1) // page + 1):
            p = int(st["block_table"][s, j])
            a, b = max(L - n, j * page), min(L, (j + 1) * page)
            had = a - j * page
            for x in "kv":
                y = rows[x][a - (L - n):b - (L - n)].transpose(0, 1)
                e = torch.ceil(torch.log2(y.abs().amax((1, 2)) / _E4M3_MAX)).clamp(_MIN_EXP, _MAX_EXP)
                size = torch.exp2(e)
                if had:
                    size = torch.maximum(size, scales[x][p])
                    caches[x][p, :, :had] = _nearest(
                        caches[x][p, :, :had] * (scales[x][p] / size)[:, None, None], values)
                scales[x][p] = size
                caches[x][p, :, had:had + b - a] = _nearest(y / size[:, None, None], values)
        t0 += n
    out = {"k_cache": caches["k"], "v_cache": caches["v"], "k_scale": scales["k"], "v_scale": scales["v"]}
    return {"q": q, **out} if rot else out


def exact(case, seed):
    held, new = _lengths(case)
    if case["op"] == "attention":
        w = work(case)
        if w["flops"] > 6e11 or sum(-(-n // case["page"]) for n in held) * case["Hkv"] > 200000:
            return None
    elif sum(n // case["page"] + 2 for n in new) > 4000:
        return None
    state = prepare(case, seed)
    return (_exact_attention if case["op"] == "attention" else _exact_append)(case, state)
